"""The operators of a block's feed-forward half beside its linear layers: the gated projection on two EXL3
weights (forward, and with its gradients), the norm of rows, and the residual sum with the norms before and
after it, its gate and its scale (forward, and with their gradients).

`run` computes each in its plain form with elementary torch operations in 32 bits, or, where `own` is set,
through the package's public functions.  Shapes are the layer shapes of this repository's own workloads
(1024, 4096, 5120, 6144, 17408) or generic ones.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "exl3xpu-mixedk_amd", "quantize")
CODES = ("exl3_mul1", "exl3_mcg", "exl3_3inst")
ACTS = ("none", "relu", "silu", "gelu")
GATES = ("none", "sigmoid", "silu")
KINDS = ("rms", "layer")
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gated(name, m, k, n, K1, K2, typ, act, bias, train=False, code="exl3_mul1"):
    c = {"kind": "gated", "m": m, "k": k, "n": n, "K1": K1, "K2": K2, "code": code, "type": typ, "act": act,
         "bias": bias, "train": train}
    return dict(c, name=name) if name else c


def _norm(name, m, d, typ, kind, params="fp32", bias=False, train=False):
    c = {"kind": "norm", "m": m, "d": d, "type": typ, "norm": kind, "params": params, "bias": bias,
         "train": train}
    return dict(c, name=name) if name else c


def _residual(name, m, d, typ, kind, post, gate, scale, params="fp32", bias=False, train=False):
    """kind, post: "rms", "layer" or ""; gate: one of GATES or ""; scale: "", "number" or "channel"."""
    c = {"kind": "residual", "m": m, "d": d, "type": typ, "norm": kind, "post": post, "gate": gate,
         "scale": scale, "params": params, "bias": bias, "train": train}
    return dict(c, name=name) if name else c


def listed():
    """The twelve cases."""
    return [
        # One token of a decoding loop through gate and up.
        _gated("gated_1x5120x17408_k4", 1, 5120, 17408, 4, 4, "bf16", "silu", False),
        # A few drafted tokens, gate and up quantized to different widths.
        _gated("gated_6x5120x17408_k3k5", 6, 5120, 17408, 3, 5, "fp16", "gelu", True),
        # A batch of 48 sequences, one token each.
        _gated("gated_48x5120x17408_k4", 48, 5120, 17408, 4, 4, "bf16", "silu", False),
        # A short prompt of odd length through a narrower layer.
        _gated("gated_333x4096x6144_k5", 333, 4096, 6144, 5, 5, "fp16", "silu", False, code="exl3_3inst"),
        # A long prompt, or a batch that calibrates the down projection: the largest call.
        _gated("gated_4096x5120x17408_k4", 4096, 5120, 17408, 4, 4, "bf16", "silu", False),
        # Forward and backward of a small layer over a short sequence.
        _gated("train_gated_100x1024x4096_k6k4", 100, 1024, 4096, 6, 4, "fp16", "silu", True, True, "exl3_mcg"),
        # Forward and backward over a whole sequence of odd length.
        _gated("train_gated_2047x5120x17408_k4", 2047, 5120, 17408, 4, 4, "bf16", "silu", True, True),
        # One token's norm before a block: the smallest call of a decoding loop.
        _norm("norm_1x5120", 1, 5120, "bf16", "rms", "bf16"),
        # Forward and backward of the norm of each head's 128 channels: 4096 tokens of 8 heads.
        _norm("train_norm_32768x128", 32768, 128, "bf16", "rms", train=True),
        # One token between two blocks of a decoding loop, normed before it is added and after.
        _residual("residual_1x5120", 1, 5120, "fp16", "rms", "rms", "", "", "fp16"),
        # A prompt of odd length, an odd width, with centred norms, biases and the channels' scales.
        _residual("residual_333x1023", 333, 1023, "fp16", "layer", "", "", "channel", "fp32", True),
        # Forward and backward between two blocks over a long batch, everything there is.
        _residual("train_residual_8191x5120", 8191, 5120, "bf16", "rms", "rms", "sigmoid", "channel", "fp32",
                  False, True),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], uniform over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(["gated", "gated", "gated", "norm", "residual", "residual"])
    typ = rng.choice(["bf16", "fp16"])
    if kind == "gated":
        train = rng.random() < 0.4
        return _gated("", _log(rng, 1, 2047 if train else 4096), 128 * _log(rng, 1, 40), 128 * _log(rng, 1, 136),
                      rng.randint(2, 7), rng.randint(2, 7), typ, rng.choice(ACTS), rng.random() < 0.5, train,
                      rng.choice(CODES))
    d = _log(rng, 16, 17408)
    m = _log(rng, 1, min(65536, 8191 * 5120 // d))
    params = rng.choice(["fp32", typ])
    if kind == "norm":
        return _norm("", m, d, typ, rng.choice(KINDS), params, rng.random() < 0.5, rng.random() < 0.5)
    return _residual("", m, d, typ, rng.choice(KINDS + ("",)), rng.choice(KINDS + ("",)), rng.choice(GATES + ("",)),
                     rng.choice(["", "number", "channel"]), params, rng.random() < 0.5, rng.random() < 0.5)


# ------------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _acts(gen, rows, k, dtype):
    """Activations: unit Gaussians, one channel in 128 twenty times as large, rows of different size."""
    x = _randn(gen, rows, k)
    x[:, ::128] *= 20.0
    return (x * torch.exp(_randn(gen, rows, 1) * 0.5)).to(dtype)


def _signs(gen, *shape):
    return torch.where(torch.rand(*shape, generator=gen, device="cuda") < 0.5, -1.0, 1.0)


def _trellis(gen, tk, tn, K):
    """Trellis words (any bits are a tail-biting stream) and channel scales as quantize_linear leaves them."""
    tr = torch.randint(-32768, 32768, (tk, tn, 16 * K), generator=gen, device="cuda", dtype=torch.int16)
    suh = (_signs(gen, 16 * tk) * (0.5 + torch.rand(16 * tk, generator=gen, device="cuda"))
           / math.sqrt(16 * tk)).half()
    svh = (_signs(gen, 16 * tn) * (0.5 + torch.rand(16 * tn, generator=gen, device="cuda"))).half()
    return tr, suh, svh


NUMBER = 0.22                  # a residual scale that is one number
EPS = 1e-6


def prepare(case, seed):
    """What a user's program holds before the call."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, train = TYPES[case["type"]], case["train"]
    s = {"case": case}
    if case["kind"] == "gated":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = _acts(gen, m, k, dt)
        s["gate"] = _trellis(gen, k // 16, n // 16, case["K1"])
        s["up"] = _trellis(gen, k // 16, n // 16, case["K2"])
        for name in ("gate_bias", "up_bias"):
            s[name] = _randn(gen, n).to(dt) if case["bias"] else None
        if train:
            s["dy"] = _randn(gen, m, n).to(dt)
            s["leaves"] = [s[v].requires_grad_() for v in ("x", "gate_bias", "up_bias") if s[v] is not None]
        if own:
            xt = _package()
            s["layers"] = [xt.TrellisLinear(*s[w], case[K], code=case["code"])
                           for w, K in (("gate", "K1"), ("up", "K2"))]
        return s
    m, d, pt = case["m"], case["d"], TYPES[case["params"]]
    s["x"] = _acts(gen, m, d, dt)
    names = ["x"]

    def parameter(name, there, mean, dev):
        s[name] = (mean + dev * _randn(gen, d)).to(pt) if there else None
        names.append(name)

    parameter("weight", bool(case["norm"]), 1.0, 0.2)
    parameter("bias", bool(case["norm"]) and case["bias"], 0.0, 0.2)
    if case["kind"] == "residual":
        s["residual"] = _acts(gen, m, d, dt)
        s["gate"] = _randn(gen, m, d).to(dt) if case["gate"] else None
        names += ["residual", "gate"]
        parameter("scale", case["scale"] == "channel", 0.5, 0.2)
        parameter("post_weight", bool(case["post"]), 1.0, 0.2)
        parameter("post_bias", bool(case["post"]) and case["bias"], 0.0, 0.2)
        s["dy"] = _randn(gen, m, d).to(dt) if train else None
    s["dh"] = _randn(gen, m, d).to(dt) if train and case["norm"] else None
    s["names"] = [v for v in names if s[v] is not None]
    if train:
        s["leaves"] = [s[v].requires_grad_() for v in s["names"]]
    return s


def _package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import trellis_ops
    return trellis_ops


# --------------------------------------------------------------------- pass
def run(state):
    """One pass."""
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_gated(state) if state["case"]["kind"] == "gated" else _plain_norm(state)


def _run_own(s):
    xt, c = _package(), s["case"]
    if c["kind"] == "gated":
        y = xt.gated(s["x"], *s["layers"], gate_bias=s["gate_bias"], up_bias=s["up_bias"], act=c["act"])
        if not c["train"]:
            return {"y": y}
        g = torch.autograd.grad(y, s["leaves"], s["dy"])
        return {"y": y.detach(), "dx": g[0], "dgate_bias": g[1] if c["bias"] else None,
                "dup_bias": g[2] if c["bias"] else None}
    if c["kind"] == "norm":
        h = xt.norm(s["x"], s["weight"], s["bias"], kind=c["norm"], eps=EPS)
        if not c["train"]:
            return {"h": h}
        return dict(zip(["d" + v for v in s["names"]], torch.autograd.grad(h, s["leaves"], s["dh"])), h=h.detach())
    y, h = xt.residual_norm(
        s["x"], s["residual"], s["weight"], s["bias"], kind=c["norm"] or None, eps=EPS, gate=s["gate"],
        gate_act=c["gate"] or "none",
        scale={"": None, "number": NUMBER, "channel": s["scale"]}[c["scale"]],
        post=c["post"] or None, post_weight=s["post_weight"], post_bias=s["post_bias"], post_eps=EPS)
    if not c["train"]:
        return {"y": y, "h": h}
    outs, douts = ((y, h), (s["dy"], s["dh"])) if c["norm"] else ((y,), (s["dy"],))
    grads = torch.autograd.grad(outs, s["leaves"], douts)
    return dict(zip(["d" + v for v in s["names"]], grads), y=y.detach(), h=h.detach() if c["norm"] else None)


def _hadamard(dtype=torch.float32):
    """The normalised 128x128 Sylvester matrix: entry (i, j) has the sign of the parity of i & j."""
    i = torch.arange(128, device="cuda")
    p = i[:, None] & i[None, :]
    p = p ^ (p >> 4)
    p = p ^ (p >> 2)
    p = (p ^ (p >> 1)) & 1
    return (1 - 2 * p).to(dtype) / math.sqrt(128.0)


def _values(states, code):
    """Codebook values of trellis states (int64), fp32."""
    if code == "exl3_mul1":
        h = (states * 0x83DCD12D) & 0xFFFFFFFF
        total = (h & 255) + ((h >> 8) & 255) + ((h >> 16) & 255) + (h >> 24)
        return ((1024 + total).float() * (1774.0 / 262144.0) - 1329.0 / 128.0).half().float()
    h = states * 89226354 + 64248484 if code == "exl3_3inst" else states * 0xCBAC1FED
    h = (h & 0x8FFF8FFF) ^ 0x3B603B60
    lo = (h & 0xFFFF).to(torch.int16).view(torch.float16)
    hi = (h >> 16).to(torch.int16).view(torch.float16)
    return (lo.float() + hi.float()).half().float()


def _weight(w, K, code):
    """Dense [k, n] fp32 weight of a trellis [k/16, n/16, 16K] and its scales."""
    tr, suh, svh = w
    tk, tn = tr.shape[:2]
    words = tr.contiguous().view(torch.int32).to(torch.int64) & 0xFFFFFFFF
    last = torch.arange(256, device="cuda") * K + K - 1       # a window's last bit
    lo = last >> 5
    both = (words[..., (lo - 1) % (8 * K)] << 32) | words[..., lo]
    states = (both >> (31 - (last & 31))) & 0xFFFF
    vals = _values(states, code)
    r, c = torch.arange(16, device="cuda")[:, None], torch.arange(16, device="cuda")[None, :]
    t = 32 * (c % 8) + 8 * ((r % 8) // 2) + 4 * (c // 8) + 2 * (r // 8) + r % 2
    inner = vals[..., t.reshape(-1)].view(tk, tn, 16, 16).transpose(1, 2)
    h = _hadamard()
    inner = inner.reshape(tk * 16, tn // 8, 128) @ h
    inner = inner.reshape(tk // 8, 128, tn * 16).transpose(1, 2) @ h
    dense = inner.transpose(1, 2).reshape(tk * 16, tn * 16)
    return dense * suh.float()[:, None] * svh.float()[None, :]


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 + z * (1 - sig))
    if act == "gelu":
        return (0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    if act == "sigmoid":
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 - sig)
    return torch.ones_like(z)


def _plain_gated(s):
    c = s["case"]
    dt = TYPES[c["type"]]
    x = s["x"].float()
    wg, wu = _weight(s["gate"], c["K1"], c["code"]), _weight(s["up"], c["K2"], c["code"])
    zg, zu = x @ wg, x @ wu
    if c["bias"]:
        zg, zu = zg + s["gate_bias"].float(), zu + s["up_bias"].float()
    a = _act(zg, c["act"])
    y = (a * zu).to(dt)
    if not c["train"]:
        return {"y": y}
    dy = s["dy"].float()
    dg, du = dy * zu * _act_grad(zg, c["act"]), dy * a
    return {"y": y, "dx": (dg @ wg.t() + du @ wu.t()).to(dt), "dgate_bias": dg.sum(0).to(dt) if c["bias"] else None,
            "dup_bias": du.sum(0).to(dt) if c["bias"] else None}


def _float(t):
    return None if t is None else t.float()


def _normed(x, kind):
    """Rows without weight, and the factor of their deviations."""
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    return x * rstd, rstd


def _norm_grad(g, xhat, rstd, kind):
    """Gradient of a row from its normed row's."""
    dx = g - xhat * (g * xhat).mean(1, keepdim=True)
    if kind == "layer":
        dx = dx - g.mean(1, keepdim=True)
    return dx * rstd


def _affine(xhat, w, b):
    n = xhat if w is None else xhat * w
    return n if b is None else n + b


def _plain_norm(s):
    c = s["case"]
    dt = TYPES[c["type"]]
    x, w, b = s["x"].float(), _float(s["weight"]), _float(s["bias"])
    out, grads = {}, {}
    y = x
    if c["kind"] == "residual":
        pw, pb, gate = _float(s["post_weight"]), _float(s["post_bias"]), _float(s["gate"])
        scale = s["scale"].float() if c["scale"] == "channel" else NUMBER if c["scale"] == "number" else 1.0
        p = x
        if c["post"]:
            phat, prstd = _normed(x, c["post"])
            p = _affine(phat, pw, pb)
        q = p if gate is None else p * _act(gate, c["gate"])
        y = s["residual"].float() + scale * q
        out["y"] = y.to(dt)
    dtotal = s["dy"].float() if c["train"] and c["kind"] == "residual" else 0.0
    if c["norm"]:
        yhat, rstd = _normed(y, c["norm"])
        out["h"] = _affine(yhat, w, b).to(dt)
        if c["train"]:
            dh = s["dh"].float()
            grads["weight"] = (dh * yhat).sum(0)
            grads["bias"] = dh.sum(0) if b is not None else None
            dtotal = dtotal + _norm_grad(dh * w, yhat, rstd, c["norm"])
    elif c["kind"] == "residual":
        out["h"] = None
    if not c["train"]:
        return out
    if c["kind"] == "norm":
        grads["x"] = dtotal
    else:
        grads["residual"] = dtotal
        if c["scale"] == "channel":
            grads["scale"] = (dtotal * q).sum(0)
        dq = dtotal * scale
        dp = dq
        if gate is not None:
            grads["gate"] = dq * p * _act_grad(gate, c["gate"])
            dp = dq * _act(gate, c["gate"])
        grads["x"] = dp
        if c["post"]:
            grads["post_weight"] = (dp * phat).sum(0)
            grads["post_bias"] = dp.sum(0) if pb is not None else None
            grads["x"] = _norm_grad(dp * pw, phat, prstd, c["post"])
    return dict({"d" + v: grads[v].to(s[v].dtype) for v in s["names"]}, **out)


# --------------------------------------------------------------------- work
def work(case):
    """Each input read and each output written once; two operations per product and sum."""
    if case["kind"] == "gated":
        m, k, n = case["m"], case["k"], case["n"]
        bias = 4 * n if case["bias"] else 0
        fwd = k * n * (case["K1"] + case["K2"]) / 8 + 4 * (k + n) + 2.0 * m * (k + n) + bias
        if not case["train"]:
            return {"bytes": fwd, "flops": 4.0 * m * k * n}
        return {"bytes": fwd + 2.0 * m * (k + n) + bias, "flops": 8.0 * m * k * n}
    m, d = case["m"], case["d"]
    norm, each = bool(case["norm"]), 4 if case["params"] == "fp32" else 2
    tensors, params, ops = 1 + norm, norm * (1 + case["bias"]), 6 * norm        # x, h
    if case["kind"] == "residual":
        post, gate = bool(case["post"]), bool(case["gate"])
        tensors += 2 + gate                                                     # residual, y
        params += (case["scale"] == "channel") + post * (1 + case["bias"])
        ops += 3 + 6 * post + 4 * gate
    if case["train"]:
        # gradients of every input and every output
        tensors, params, ops = 2 * tensors, 2 * params, 3 * ops
    return {"bytes": 2.0 * tensors * m * d + each * params * d, "flops": float(ops) * m * d}


# -------------------------------------------------------------------- exact
def _butterfly(v):
    """The block-128 transform of the last dimension, by sums and differences."""
    shape = v.shape
    v = v.reshape(-1, 128)
    for b in range(7):
        u = v.reshape(-1, 128 >> (b + 1), 2, 1 << b)
        v = torch.stack([u[:, :, 0] + u[:, :, 1], u[:, :, 0] - u[:, :, 1]], 2).reshape(-1, 128)
    return v.reshape(shape) / math.sqrt(128.0)


def _codebook(code):
    """The 65,536 codebook values, from their definition."""
    half = lambda bits: torch.tensor(bits, dtype=torch.int64).to(torch.int16).view(torch.float16).double()  # noqa: E731
    st = torch.arange(1 << 16)
    if code == "exl3_mul1":
        h = (st * 0x83DCD12D) & 0xFFFFFFFF
        total = sum((h >> b) & 255 for b in (0, 8, 16, 24))
        return ((1024 + total).double() * half([0x1EEE]) + half([0xC931 - 0x10000])).half().double().cuda()
    h = st * 89226354 + 64248484 if code == "exl3_3inst" else st * 0xCBAC1FED
    h = (h & 0x8FFF8FFF) ^ 0x3B603B60
    return (half((h & 0xFFFF).tolist()) + half((h >> 16).tolist())).half().double().cuda()


def _inner(tr, K, code):
    """Inner weight [k, n] in 64 bits: each state gathered bit by bit from its circular stream."""
    tk, tn = tr.shape[:2]
    sh = torch.arange(15, -1, -1, device="cuda")
    order = torch.arange(16 * K, device="cuda").view(-1, 2).flip(1).reshape(-1)  # words: high half first
    bits = ((tr[:, :, order].to(torch.int32)[..., None] >> sh) & 1).to(torch.uint8).reshape(tk, tn, 256 * K)
    t = torch.arange(256, device="cuda")
    st = torch.zeros(tk, tn, 256, dtype=torch.int32, device="cuda")
    for b in range(16):
        st = 2 * st + bits[:, :, (t * K + K - 16 + b) % (256 * K)]
    book = _codebook(code)
    out = torch.empty(tk, 16, tn, 16, dtype=torch.float64, device="cuda")
    for e in range(8):      # elements 8g + e: rows 2 (g % 4) + .., columns g // 4 + ..
        for q in range(4):
            out[:, 2 * q + e % 2 + 8 * (e // 2 % 2), :, 8 * (e // 4):8 * (e // 4) + 8] = \
                book[st[:, :, 8 * q + e::32].long()]
    return out.reshape(16 * tk, 16 * tn)


def exact(case, seed):
    """What run returns, from the operators' definitions in 64 bits."""
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_gated(case, s) if case["kind"] == "gated" else _exact_norm(case, s)


def _exact_act(z, act):
    """An activation and its slope."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act in ("silu", "sigmoid"):
        sig = torch.sigmoid(z)
        return (z * sig, sig + z * sig * (1 - sig)) if act == "silu" else (sig, sig * (1 - sig))
    if act == "gelu":
        cdf = torch.erfc(-z / math.sqrt(2.0)) / 2
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def _exact_gated(case, s):
    x, z, inner = s["x"].double(), [], []
    for name, K, bias in (("gate", "K1", "gate_bias"), ("up", "K2", "up_bias")):
        tr, suh, svh = s[name]
        inner.append(_inner(tr, case[K], case["code"]))
        v = _butterfly(_butterfly(x * suh.double()) @ inner[-1]) * svh.double()
        z.append(v if s[bias] is None else v + s[bias].double())
    a, slope = _exact_act(z[0], case["act"])
    if not case["train"]:
        return {"y": a * z[1]}
    dy = s["dy"].double()
    dz = [dy * z[1] * slope, dy * a]
    dx = 0.0
    for name, g, w in zip(("gate", "up"), dz, inner):
        _, suh, svh = s[name]
        dx = dx + _butterfly(_butterfly(g * svh.double()) @ w.t().contiguous()) * suh.double()
    sums = [g.sum(0) if case["bias"] else None for g in dz]
    return {"y": a * z[1], "dx": dx, "dgate_bias": sums[0], "dup_bias": sums[1]}


def _exact_norm(case, s):
    """Gradients by reverse differentiation of the definition, in 64 bits."""
    v = {n: s[n].detach().double().requires_grad_(case["train"]) for n in s["names"]}

    def normed(t, kind, weight, bias):
        mean = t.mean(-1, keepdim=True) if kind == "layer" else 0.0
        t = (t - mean) * torch.rsqrt(((t - mean) ** 2).mean(-1, keepdim=True) + EPS) * v[weight]
        return t + v[bias] if bias in v else t

    with torch.enable_grad():
        t, outs, douts = v["x"], {}, []
        if case["kind"] == "residual":
            if case["post"]:
                t = normed(t, case["post"], "post_weight", "post_bias")
            if case["gate"]:
                t = t * _exact_act(v["gate"], case["gate"])[0]
            t = v["residual"] + t * (v["scale"] if "scale" in v else NUMBER if case["scale"] == "number" else 1.0)
            outs["y"] = t
            douts.append(s["dy"])
        if case["norm"]:
            outs["h"] = normed(t, case["norm"], "weight", "bias")
            douts.append(s["dh"])
        grads = {}
        if case["train"]:
            grads = dict(zip(["d" + n for n in v], torch.autograd.grad(
                list(outs.values()), list(v.values()), [g.double() for g in douts])))
    outs = {n: t.detach() for n, t in outs.items()}
    if case["kind"] == "residual" and not case["norm"]:
        outs["h"] = None
    return dict(grads, **outs)
