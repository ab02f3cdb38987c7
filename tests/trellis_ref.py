"""The operators on trellis weights in 64 bits, from their definitions, on the CPU: what the GPU
tests compare with.  Weights are decoded by the C oracle."""
import math

import numpy as np
import torch

CODES = {"exl3_mul1", "exl3_3inst", "exl3_mcg"}


def random_weight(k, n, K, seed, device="cuda"):
    """(trellis, suh, svh): any bits are a tail-biting stream; signed channel scales."""
    g = torch.Generator().manual_seed(seed)
    tr = torch.randint(-32768, 32768, (k // 16, n // 16, 16 * K), generator=g, dtype=torch.int16)
    sign = lambda m: torch.where(torch.rand(m, generator=g) < 0.5, -1.0, 1.0)  # noqa: E731
    suh = (sign(k) * (0.5 + torch.rand(k, generator=g)) / math.sqrt(k)).half()
    svh = (sign(n) * (0.5 + torch.rand(n, generator=g))).half()
    return tr.to(device), suh.to(device), svh.to(device)


def inner(O, tr, K, code):
    """Decoded weight [k, n], 64 bits."""
    return torch.from_numpy(np.asarray(O.decode(tr.cpu().numpy(), O.code_lut(code), K))).double()


def had(v):
    """Normalised block-128 transform of the last dimension."""
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < 128:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    s = v.shape
    return (v.reshape(-1, 128) @ (h / math.sqrt(128.0))).reshape(s)


def dense(O, tr, suh, svh, K, code, scale=1.0):
    """W [k, n], 64 bits."""
    w = had(inner(O, tr, K, code))
    w = had(w.t().contiguous()).t()
    return w * suh.cpu().double()[:, None] * svh.cpu().double()[None, :] * scale


def act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def roundoff(dtype):
    """Largest relative error of one rounding to dtype."""
    return {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[dtype]


def row_errors(got, want):
    """2-norm of the difference over the 2-norm of the result, by rows."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape
    norm = want.norm(dim=-1)
    off = (got - want).norm(dim=-1)
    return torch.where(norm > 0, off / norm.clamp(min=1e-300), (off > 0).double())
