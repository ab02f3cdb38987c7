"""trellis_ops.py -- products with weights in the EXL3 trellis format, on the GPU.

What quantize_linear returns is multiplied with as it is: the weight stays in
its trellis, the kernels decode it on the way to the matrix cores.

    import quantize as xq, trellis_ops as xt
    r = xq.quantize_linear(W, H, K=4, device="cuda", channel_scales=True)
    w = xt.TrellisLinear.from_result(r)
    y = xt.linear(x, w, bias=b, act="silu", residual=res)     # differentiable in x, bias, residual
    G = xt.input_gram(x)                                      # the H of the next quantize_linear

Activations are bfloat16 or float16 and results have their type; sums are fp32
and every result is rounded once.  Calls are ordered on the current stream,
never wait for the GPU, and can be captured in a HIP graph.  There is no
fallback: tensors that are not on a HIP device raise.

The reference multiplies with its weights in a serving stack of its own
(serve/patches/0001-exl3-ops-mixed-k.patch); there is no counterpart here to
cite for these functions.
"""
from __future__ import annotations

import contextlib
import ctypes
import os
import sys

import torch
import torch.autograd.forward_ad as _fad

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import hip_backend as _hb  # noqa: E402

ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_FAST = 16
_COUNTERS = 16384
_counters: dict = {}
_HERE = contextlib.nullcontext()


def _stream(dev: torch.device) -> int:
    """The current stream of dev.  The raw handle comes without a Stream object
    around it: 0.1 us instead of 2, of the 10 that a call of one token takes."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _on(dev: torch.device):
    """dev as the current device, where it is not that already."""
    return _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _counter_words(dev: torch.device, stream: int) -> torch.Tensor:
    """The zeroed words a call counts its finished parts in: one set per stream,
    since calls on one stream never overlap (every call leaves them zero).  A
    captured call gets a set of its own, cleared inside the graph, because the
    graph may be replayed on any stream; the caller keeps it until its kernels
    are recorded."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(_COUNTERS, dtype=torch.int32, device=dev)
    key = (dev.index, stream)
    t = _counters.get(key)
    if t is None:                       # (of two threads that come here at once, one's set stays)
        t = _counters.setdefault(key, torch.zeros(_COUNTERS, dtype=torch.int32, device=dev))
    return t


class TrellisLinear:
    """A trellis weight W [k in, n out] to multiply with: trellis int16
    [k/16, n/16, 16K], suh [k] and svh [n] fp16 on one HIP device, their K and
    code, and the weight's scale (quantize_linear's Wscale where the channel
    scales do not hold it).  Nothing is laid out anew; the tensors are kept."""

    def __init__(self, trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor, K: int,
                 code: str = "exl3_mul1", scale: float = 1.0):
        K = int(K)
        if not 2 <= K <= 7:
            raise ValueError(f"K must be 2..7, got {K}")
        if _hb.code_name(code) == "1mad":
            raise NotImplementedError("the products take the EXL3 codes (mul1, 3inst, mcg): "
                                      "1mad's values are not fp16 numbers")
        if trellis.dim() != 3 or trellis.shape[2] != 16 * K:
            raise ValueError(f"trellis must be [k/16, n/16, {16 * K}], got {tuple(trellis.shape)}")
        k, n = 16 * trellis.shape[0], 16 * trellis.shape[1]
        if not k or not n or k % 128 or n % 128:
            raise ValueError(f"k and n must be multiples of 128, got {k}, {n}")
        if suh.shape != (k,) or svh.shape != (n,):
            raise ValueError(f"suh must be [{k}] and svh [{n}], got {tuple(suh.shape)}, "
                             f"{tuple(svh.shape)}")
        self.trellis = _hb._dev_tensor(trellis, torch.int16, "trellis")
        self.suh = _hb._dev_tensor(suh, torch.float16, "suh")
        self.svh = _hb._dev_tensor(svh, torch.float16, "svh")
        self.device = self.trellis.device
        if self.suh.device != self.device or self.svh.device != self.device:
            raise ValueError("trellis, suh and svh must be on one device")
        self.k, self.n, self.K, self.code, self.scale = k, n, K, code, float(scale)
        self._w = _hb.TrellisWeight(self.trellis.data_ptr(), self.suh.data_ptr(),
                                    self.svh.data_ptr(), self.scale, k, n, K,
                                    _hb.code_name(code).encode())
        self._p = ctypes.byref(self._w)

    @classmethod
    def from_result(cls, r: dict, device="cuda") -> "TrellisLinear":
        """From a quantize_linear result."""
        return cls(r["trellis"].to(device), r["suh"].to(device).half(), r["svh"].to(device).half(),
                   r["K"], code=r["code"], scale=1.0 if r["channel_scales"] else r["Wscale"])

    def __call__(self, x, bias=None, act="none", residual=None, fast=False):
        return linear(x, self, bias=bias, act=act, residual=residual, fast=fast)


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """t [.., cols] as rows whose elements are consecutive (a copy if need be)."""
    t = t.reshape(-1, cols) if t.dim() != 2 else t
    if t.shape[0] > 1 and (t.stride(1) != 1 or t.stride(0) < cols):
        return t.contiguous()
    return t if t.shape[0] != 1 or t.stride(1) == 1 else t.contiguous()


def _stride(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _check_act(act: str) -> int:
    try:
        return ACTS[act]
    except KeyError:
        raise ValueError(f"act {act!r} not in {tuple(ACTS)}") from None


def _like(t: torch.Tensor, x: torch.Tensor, shape, name: str, dtypes) -> None:
    if t.device != x.device or t.dtype not in dtypes or t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)} of {' or '.join(map(str, dtypes))} on "
                         f"{x.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")


def _no_tangents(name: str, *tensors) -> None:
    """Raises for tensors that carry a forward-mode derivative: a kernel reads their
    values alone, and the result's missing tangent would read as zero."""
    if _fad._current_level >= 0 and any(t is not None and _fad.unpack_dual(t).tangent is not None
                                        for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def _forward(x, w, bias, act, residual, fast, keep_z):
    rows = _rows(x, w.k)
    m = rows.shape[0]
    y = torch.empty(*x.shape[:-1], w.n, dtype=x.dtype, device=x.device)
    z = torch.empty(m, w.n, dtype=x.dtype, device=x.device) if keep_z else None
    if m == 0:
        return y, z
    res = None if residual is None else _rows(residual, w.n)
    bias = None if bias is None else bias.contiguous()
    L = _hb.lib()
    with _on(x.device):
        stream = _stream(x.device)
        need = L.xtq_linear_ws_bytes(w._p, m, 2 if keep_z else 0)
        words = _counter_words(x.device, stream)
        ws = torch.empty(max(need, 0), dtype=torch.uint8, device=x.device)
        rc = L.xtq_linear_dev(
            w._p, _TYPES[x.dtype] | fast, rows.data_ptr(), _stride(rows), m,
            None if bias is None else bias.data_ptr(), int(bias is not None and
                                                           bias.dtype == torch.float32), act,
            None if res is None else res.data_ptr(), 0 if res is None else _stride(res),
            None if z is None else z.data_ptr(), y.data_ptr(), w.n, ws.data_ptr(), ws.numel(),
            words.data_ptr(), stream)
    _hb._check("xtq_linear_dev", rc)
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, residual, w, act, fast):
        need = ctx.needs_input_grad[0] or (bias is not None and ctx.needs_input_grad[1])
        y, z = _forward(x, w, bias, act, residual, fast, need and act != 0)
        ctx.w, ctx.act, ctx.fast, ctx.shape = w, act, fast, x.shape
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(z)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        z, = ctx.saved_tensors
        _no_tangents("linear's gradient", dy)
        w = ctx.w
        want_x, want_b, want_r = ctx.needs_input_grad[:3]
        dx = dbias = None
        if want_x or want_b:
            rows = _rows(dy, w.n)
            m = rows.shape[0]
            if want_x:
                dx = torch.empty(ctx.shape, dtype=dy.dtype, device=dy.device)
            if want_b:
                dbias = torch.empty(w.n, dtype=ctx.bias_dtype, device=dy.device)
            if m == 0:
                return dx, None if dbias is None else dbias.zero_(), dy if want_r else None, None, None, None
            L = _hb.lib()
            with _on(dy.device):
                stream = _stream(dy.device)
                need = L.xtq_linear_ws_bytes(w._p, m, 1)
                words = _counter_words(dy.device, stream)
                ws = torch.empty(max(need, 0), dtype=torch.uint8, device=dy.device)
                rc = L.xtq_linear_bwd_dev(
                    w._p, _TYPES[dy.dtype] | ctx.fast, rows.data_ptr(), _stride(rows),
                    None if z is None else z.data_ptr(), ctx.act, m,
                    None if dx is None else dx.data_ptr(), w.k,
                    None if dbias is None else dbias.data_ptr(),
                    int(ctx.bias_dtype == torch.float32), ws.data_ptr(), ws.numel(),
                    words.data_ptr(), stream)
            _hb._check("xtq_linear_bwd_dev", rc)
        return dx, dbias, dy if want_r else None, None, None, None


def linear(x: torch.Tensor, w: TrellisLinear, bias: torch.Tensor | None = None,
           act: str = "none", residual: torch.Tensor | None = None,
           fast: bool = False) -> torch.Tensor:
    """act(x W + bias) + residual for x [.., k] (bfloat16 or float16) -> [.., n]
    in x's type.  act: none, relu, silu or gelu (erf).  bias [n] has x's type or
    fp32, residual y's shape and x's type.  Differentiable in x, bias and
    residual (once, in reverse mode; the weight is frozen); the same result with a gradient and
    without.  x enters the product with 22 bits for float16 and for relu, and with
    11 otherwise, which a bfloat16 result's 8 hide; the gradient's product likewise
    (float16: 22).  fast: with 11 bits always, at half the matrix work: float16
    results and gradients are then off by 1.4 times their own rounding, and relu's
    gradient takes some slopes on the wrong side of zero."""
    if x.dtype not in _TYPES:
        raise ValueError(f"x must be bfloat16 or float16, got {x.dtype}")
    if x.device != w.device:
        raise ValueError(f"x must be on {w.device}, got {x.device}")
    if x.dim() < 1 or x.shape[-1] != w.k:
        raise ValueError(f"x must be [.., {w.k}], got {tuple(x.shape)}")
    a, fast = _check_act(act), _FAST if fast else 0
    _no_tangents("linear", x, bias, residual)
    if bias is not None:
        _like(bias, x, (w.n,), "bias", (x.dtype, torch.float32))
    if residual is not None:
        _like(residual, x, (*x.shape[:-1], w.n), "residual", (x.dtype,))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, bias, residual)):
        return _Linear.apply(x, bias, residual, w, a, fast)
    return _forward(x, w, bias, a, residual, fast, False)[0]


_MOE_ROWS = 64


class TrellisExperts:
    """The experts of a mixture layer: lists of TrellisLinear, gate and up [d, f],
    down [f, d], one code, each with its own K.  Keeps them and a table of their
    addresses on the device."""

    def __init__(self, gate, up, down):
        gate, up, down = list(gate), list(up), list(down)
        if not gate or len(up) != len(gate) or len(down) != len(gate):
            raise ValueError(f"one gate, up and down per expert, got {len(gate)}, {len(up)}, {len(down)}")
        self.weights = [w for ws in zip(gate, up, down) for w in ws]
        first = gate[0]
        self.device, self.code, self.d, self.f = first.device, first.code, first.k, first.n
        for i, w in enumerate(self.weights):
            want = (self.f, self.d) if i % 3 == 2 else (self.d, self.f)
            if (w.k, w.n) != want or w.device != self.device or \
                    _hb.code_name(w.code) != _hb.code_name(self.code):
                raise ValueError(f"expert {i // 3}'s {('gate', 'up', 'down')[i % 3]} must be "
                                 f"[{want[0]}, {want[1]}] {self.code} on {self.device}, got "
                                 f"[{w.k}, {w.n}] {w.code} on {w.device}")
        n = len(gate)
        host = (_hb.TrellisWeight * (3 * n))(*[w._w for w in self.weights])
        words = torch.empty(3 * n, 4, dtype=torch.int64)
        _hb._check("xtq_moe_table", _hb.lib().xtq_moe_table(host, n, words.data_ptr()))
        self.n, self.table = n, words.to(self.device)
        self._code = _hb.code_name(self.code).encode()
        self._rows: dict = {}               # by top_k: tokens that one call takes


def _moe_rows(experts: int, top_k: int, d: int, f: int) -> int:
    """The most tokens that a call of xtq_moe_dev takes: its workgroups count
    themselves in XTQ_OP_COUNTERS words, which many experts' wide layers use up
    before 64 tokens.  0: not even one."""
    need = _hb.lib().xtq_moe_ws_bytes
    return next((r for r in range(_MOE_ROWS, 0, -1) if need(r, experts, top_k, d, f) >= 0), 0)


def moe(x: torch.Tensor, router: torch.Tensor, experts: TrellisExperts, top_k: int,
        act: str = "silu", renorm: bool = True, residual: torch.Tensor | None = None,
        valid: torch.Tensor | None = None, return_routing: bool = False):
    """A mixture-of-experts layer for a few tokens x [.., d]: softmax(x router^T),
    the top_k experts (ties: the lowest), and residual + sum of their
    weight * down(act(gate(x)) * up(x)), in x's type.  router [experts, d] has x's
    type or fp32; renorm divides the weights by their sum.  Tokens that valid [..]
    (bool) leaves out are not looked at: their result is the residual or 0.
    return_routing: also the expert numbers int32 [.., top_k] (-1 where left out)
    and weights fp32.  More than 64 tokens run 64 at a time, fewer where many
    experts' wide layers take more counters than there are.  No gradient."""
    if x.dtype not in _TYPES:
        raise ValueError(f"x must be bfloat16 or float16, got {x.dtype}")
    if x.device != experts.device:
        raise ValueError(f"x must be on {experts.device}, got {x.device}")
    if x.dim() < 1 or x.shape[-1] != experts.d:
        raise ValueError(f"x must be [.., {experts.d}], got {tuple(x.shape)}")
    a, top_k, d = _check_act(act), int(top_k), experts.d
    if not 1 <= top_k <= min(16, experts.n):
        raise ValueError(f"top_k must be 1..{min(16, experts.n)}, got {top_k}")
    _like(router, x, (experts.n, d), "router", (x.dtype, torch.float32))
    if residual is not None:
        _like(residual, x, x.shape, "residual", (x.dtype,))
    if valid is not None:
        _like(valid, x, x.shape[:-1], "valid", (torch.bool,))
        valid = valid.contiguous()
    _no_tangents("moe", x, router, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, router, residual)):
        raise NotImplementedError("moe has no gradient: call it under torch.no_grad()")
    most = experts._rows.get(top_k)
    if most is None:
        most = experts._rows[top_k] = _moe_rows(experts.n, top_k, d, experts.f)
    if not most:
        raise ValueError(f"{top_k} experts of {d} by {experts.f} a token are more than a call can count")
    rows, router = _rows(x, d), router.contiguous()
    res = None if residual is None else _rows(residual, d)
    m = rows.shape[0]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    ids = torch.empty(*x.shape[:-1], top_k, dtype=torch.int32, device=x.device)
    weights = torch.empty(*x.shape[:-1], top_k, dtype=torch.float32, device=x.device)
    L = _hb.lib()
    with _on(x.device):
        stream = _stream(x.device)
        words = _counter_words(x.device, stream)        # (of all batches: they follow each other)
        for r in range(0, m, most):
            n = min(most, m - r)
            need = L.xtq_moe_ws_bytes(n, experts.n, top_k, d, experts.f)
            ws = torch.empty(max(need, 0), dtype=torch.uint8, device=x.device)
            rc = L.xtq_moe_dev(
                experts.table.data_ptr(), experts.n, d, experts.f, experts._code, _TYPES[x.dtype],
                rows.data_ptr() + 2 * r * _stride(rows), _stride(rows), n, router.data_ptr(),
                int(router.dtype == torch.float32), top_k, a, int(bool(renorm)),
                None if valid is None else valid.data_ptr() + r,
                None if res is None else res.data_ptr() + 2 * r * _stride(res),
                0 if res is None else _stride(res), y.data_ptr() + 2 * r * d, d,
                ids.data_ptr() + 4 * r * top_k, weights.data_ptr() + 4 * r * top_k, ws.data_ptr(),
                ws.numel(), words.data_ptr(), stream)
            _hb._check("xtq_moe_dev", rc)
    return (y, ids, weights) if return_routing else y


def input_gram(x: torch.Tensor, valid: torch.Tensor | None = None,
               prev: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """prev + sum of x_t x_t^T over the tokens t of x [.., k] (bfloat16 or
    float16) that valid [..] (bool) keeps, as fp32 [k, k]: the input Gram that
    quantize_linear takes as H_x.  Tokens left out may hold anything.  prev: the
    Gram so far (None: zero); out: where to write (prev itself accumulates in
    place).  No gradient."""
    if x.dtype not in _TYPES:
        raise ValueError(f"x must be bfloat16 or float16, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"x must be a HIP device tensor, got {x.device}")
    if x.dim() < 1 or not x.shape[-1] or x.shape[-1] % 128:
        raise ValueError(f"x must be [.., k] with k a multiple of 128, got {tuple(x.shape)}")
    k = x.shape[-1]
    _no_tangents("input_gram", x, prev, out)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, prev, out)):
        raise NotImplementedError("input_gram has no gradient: call it under torch.no_grad()")
    if valid is not None:
        _like(valid, x, x.shape[:-1], "valid", (torch.bool,))
        valid = valid.contiguous()
    for t, name in ((prev, "prev"), (out, "out")):
        if t is not None:
            _like(t, x, (k, k), name, (torch.float32,))
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
    if prev is not None and out is not None and 0 < abs(prev.data_ptr() - out.data_ptr()) < 4 * k * k:
        raise ValueError("prev and out must be one tensor's memory or apart")
    rows = _rows(x, k)
    m = rows.shape[0]
    given = out is not None
    if not given:
        out = torch.empty(k, k, dtype=torch.float32, device=x.device)
    L = _hb.lib()
    with _on(x.device):
        need = L.xtq_gram_ws_bytes(m, k)
        ws = torch.empty(max(need, 0), dtype=torch.uint8, device=x.device)
        rc = L.xtq_gram_dev(_TYPES[x.dtype], rows.data_ptr() if m else None,
                            _stride(rows) if m else k, m, k,
                            None if valid is None else valid.data_ptr(),
                            None if prev is None else prev.data_ptr(), out.data_ptr(),
                            ws.data_ptr() if need else None, ws.numel(), _stream(x.device))
    _hb._check("xtq_gram_dev", rc)
    if given and not out.is_inference():        # written behind autograd's back: whoever kept it has to know
        torch.autograd.graph.increment_version(out)
    return out
