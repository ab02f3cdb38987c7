"""trellis_block.py -- a block of a language model from calibration to serving on
trellis weights.

    python exl3xpu-mixedk_amd/examples/trellis_block.py [--dim 512] [--hidden 1024] [--experts 8]

A dense layer pair (up with silu, down with bias and residual) and a mixture of
experts, random weights and activations:

1. calibrate  trellis_ops.input_gram sums the inputs' Gram over padded batches
2. quantize   quantize.quantize_linear with that Gram, K by weight
3. run        trellis_ops.linear and trellis_ops.moe on the trellis weights
4. tune       the biases, by gradients through the frozen trellis weights
5. serve      one token at a time, from a captured HIP graph

Prints what each step gives; main() returns it.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "quantize"))
import quantize as xq  # noqa: E402
import trellis_ops as xt  # noqa: E402


def _activations(gen, batch, tokens, dim, mix):
    """Correlated activations of padded sequences, and which tokens are real."""
    x = (torch.randn(batch, tokens, dim, generator=gen) @ mix).to(torch.bfloat16).cuda()
    lengths = torch.randint(tokens // 2, tokens + 1, (batch, 1), generator=gen)
    valid = (torch.arange(tokens)[None] < lengths).cuda()
    x[~valid] = float("nan")                # padding may hold anything
    return x, valid


def _quantize(W, gram, count, K):
    return xt.TrellisLinear.from_result(
        xq.quantize_linear(W, gram.cpu() / count, K=K, device="cuda", channel_scales=True))


def _error(got, want):
    return float((got.float() - want.float()).norm() / want.float().norm())


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--dim", type=int, default=512)
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--experts", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=256)
    a = ap.parse_args(argv)
    gen = torch.Generator().manual_seed(0)
    d, f, e = a.dim, a.hidden, a.experts

    def weight(n, k):
        return torch.randn(n, k, generator=gen) / k ** 0.5

    mix = torch.randn(d, d, generator=gen) / d ** 0.5 * torch.logspace(-1, 0.5, d)[:, None]
    up, down = weight(f, d), weight(d, f)
    experts = [(weight(f, d), weight(f, d), weight(d, f)) for _ in range(e)]
    router = weight(e, d).to(torch.bfloat16).cuda()
    out = {}

    # 1. calibrate: the Gram of the dense layers' inputs, over the real tokens alone
    grams = {k: torch.zeros(k, k, device="cuda") for k in (d, f)}
    count = 0
    for _ in range(4):
        x, valid = _activations(gen, 4, a.tokens, d, mix)
        h = torch.nn.functional.silu(x.float() @ up.t().cuda()).to(torch.bfloat16)
        xt.input_gram(x, valid=valid, prev=grams[d], out=grams[d])
        xt.input_gram(h, valid=valid, prev=grams[f], out=grams[f])
        count += int(valid.sum())

    # 2. quantize
    q_up, q_down = _quantize(up, grams[d], count, 4), _quantize(down, grams[f], count, 3)
    plain = torch.eye(f)
    layers = [[xt.TrellisLinear.from_result(xq.quantize_linear(
        W, plain[:W.shape[1], :W.shape[1]], K=K, device="cuda", channel_scales=True))
        for W, K in zip(ws, (4, 4, 5))] for ws in experts]
    mixture = xt.TrellisExperts(*zip(*layers))

    # 3. run, against the full-precision block
    x, valid = _activations(gen, 2, 32, d, mix)
    rows = x[valid]
    dense = torch.nn.functional.silu(rows.float() @ up.t().cuda()) @ down.t().cuda() + rows.float()
    bias = torch.zeros(d, device="cuda", requires_grad=True)
    inner = torch.zeros(f, device="cuda", requires_grad=True)

    def block(t):
        return xt.linear(xt.linear(t, q_up, bias=inner, act="silu"), q_down, bias=bias, residual=t)

    with torch.no_grad():
        out["dense error"] = _error(block(rows), dense)
        y, ids, weights = xt.moe(x.view(-1, d), router, mixture, 2, residual=x.view(-1, d).nan_to_num(),
                                 valid=valid.view(-1), return_routing=True)
    out["mixture finite"] = bool(y.isfinite().all())
    out["padding without experts"] = bool((ids[~valid.view(-1)] == -1).all())
    used = ids[valid.view(-1)].long()
    want = torch.zeros_like(rows, dtype=torch.float32)
    for i, (wg, wu, wd) in enumerate(experts):
        part = weights[valid.view(-1)] * (used == i)
        t = rows.float()
        o = (torch.nn.functional.silu(t @ wg.t().cuda()) * (t @ wu.t().cuda())) @ wd.t().cuda()
        want += part.sum(1, keepdim=True) * o
    out["mixture error"] = _error(y[valid.view(-1)].float() - rows.float(), want)

    # 4. tune the biases towards the full-precision block
    losses = []
    for _ in range(8):
        loss = (block(rows).float() - dense).square().mean()
        losses.append(float(loss.detach()))
        g_bias, g_inner = torch.autograd.grad(loss, (bias, inner))
        with torch.no_grad():
            scale = d * 0.2
            bias -= scale * g_bias
            inner -= scale * g_inner
    out["loss before, after"] = (losses[0], losses[-1])

    # 5. serve: one token through the dense layers and the mixture, captured once
    token = rows[:1].clone()

    def step():
        t = block(token)
        return xt.moe(t, router, mixture, 2, residual=t)

    with torch.no_grad():
        eager = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            step()
            with torch.cuda.graph(graph, stream=side):
                captured = step()
        torch.cuda.current_stream().wait_stream(side)
        same = True
        for row in (0, 1, len(rows) - 1):
            token.copy_(rows[row:row + 1])
            graph.replay()
            same &= bool(torch.equal(captured, step()))
        token.copy_(rows[:1])
        graph.replay()
        same &= bool(torch.equal(captured, eager))
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(100):
            graph.replay()
        end.record()
        end.synchronize()
    out["replays equal eager"] = same
    out["us a token"] = begin.elapsed_time(end) * 10.0
    for k, v in out.items():
        print(f"{k}: {v}", flush=True)
    return out


if __name__ == "__main__":
    main()
