"""An attention sublayer over packed sequences out of the framework's calls, forward and
backward: norm, projections (torch's products), the heads' norm with rotation, attention,
projection, dropped update; and its steps of one token against a cache."""

from __future__ import annotations

import pytest
import torch

from foldjax_amd import kernels
from tests import packed_oracle as O
from tests import rotary_oracle as R
from tests.gpu_util import say

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32
H, KV, D, C, PAIRS = 6, 2, 32, 96, 12
SCALE, LENS = D**-0.5, [45, 1, 80, 19]
DROP = {"p": 0.25, "seed": 77, "offset": 3}


def setup(dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s, by=1.0: (by * torch.randn(*s, generator=g, device="cuda")).to(dtype)  # noqa: E731
    n = sum(LENS)
    w = {"norm": 1 + rand(C, by=0.1), "qkv": rand(C, (H + 2 * KV) * D, by=C**-0.5), "q": 1 + rand(D, by=0.1),
         "k": 1 + rand(D, by=0.1), "out": rand(H * D, C, by=(H * D)**-0.5)}
    x, dy = rand(n, C), rand(n, C)
    starts = torch.tensor([0, *LENS], device="cuda").cumsum(0).to(torch.int32)
    pos = torch.cat([torch.arange(m) for m in LENS])[None].to("cuda", torch.int32)
    fr = 10000.0 ** (-torch.arange(PAIRS, dtype=torch.float64, device="cuda") / PAIRS)
    return x, dy, w, starts, pos, fr


def split(qkv):
    """q, k and v as views of the projection's rows"""
    return (t.unflatten(-1, (-1, D)).transpose(0, 1) for t in qkv.split([H * D, KV * D, KV * D], -1))


def joined(*heads):
    return torch.cat([t.transpose(0, 1).flatten(1) for t in heads], -1)


def sublayer(x, w, starts, pos, fr):
    n = kernels.rms_norm(x, w["norm"])
    qkv = n @ w["qkv"]
    q, k, v = split(qkv)
    qr, kr = kernels.head_norm_rotary(q, k, pos, fr, q_weight=w["q"], k_weight=w["k"])
    o, lse, rest = kernels.packed_attention(qr, kr, v, starts, scale=SCALE, causal=True, return_lse=True)
    rows = o.transpose(0, 1).reshape(-1, H * D)
    assert rows.data_ptr() == o.data_ptr()
    y = kernels.dropout_add(rows @ w["out"], residual=x, **DROP)
    return y, (n, q, k, v, qr, kr, o, lse, rest)


def backward(dy, x, w, starts, pos, fr, kept):
    n, q, k, v, qr, kr, o, lse, rest = kept
    du = kernels.dropout_backward(dy, **DROP)
    do = (du @ w["out"].T).unflatten(-1, (H, D)).transpose(0, 1)
    dqr, dkr, dv = kernels.packed_attention_backward(do, qr, kr, v, o, lse, rest, starts, scale=SCALE, causal=True)
    dq, dk, dwq, dwk = kernels.head_norm_rotary_backward(dqr, dkr, q, k, pos, fr, q_weight=w["q"], k_weight=w["k"])
    dqkv = joined(dq, dk, dv)
    dx, dnorm = kernels.rms_norm_backward(dqkv @ w["qkv"].T, x, w["norm"], dh=dy)
    grads = {"x": dx, "norm": dnorm, "qkv": n.T @ dqkv, "q": dwq, "k": dwk, "out": o.transpose(0, 1).flatten(1).T @ du}
    return grads, (do, dqr, dkr, dv, dq, dk)


def plain(x, w, pos, fr, kept):
    """The same in 64 bits, by autograd's operations; kept: dropout's factors."""
    rms = lambda t, g: t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * g  # noqa: E731
    q, k, v = split(rms(x, w["norm"]) @ w["qkv"])
    q, k = (R.turn(rms(t, g), pos, fr, (PAIRS,), False) for t, g in ((q, w["q"]), (k, w["k"])))
    parts, at = [], 0
    for n in LENS:
        rows = slice(at, at + n)
        kk, vv = (t[:, rows].repeat_interleave(H // KV, 0) for t in (k, v))
        s = SCALE * q[:, rows] @ kk.transpose(1, 2).contiguous()
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=s.device).triu(1), -torch.inf)
        parts.append(s.softmax(-1) @ vv)
        at += n
    return x + kept * (torch.cat(parts, 1).transpose(0, 1).flatten(1) @ w["out"])


def test_sublayer_against_64_bits():
    """float32: forward and backward together are 12 steps, each off by at most 256 terms' w
    (1.5e-5) of its terms' absolute sums, and those are within 5 of the results' own size:
    1e-3 of each result's norm."""
    say("packed sublayer float32")
    x, dy, w, starts, pos, fr = setup(FP32)
    y, kept = sublayer(x, w, starts, pos, fr)
    grads, _ = backward(dy, x, w, starts, pos, fr, kept)
    drop = kernels.dropout_add(torch.ones_like(x), **DROP).double()
    x64 = x.double().requires_grad_()
    w64 = {n: t.double().requires_grad_() for n, t in w.items()}
    with torch.enable_grad():
        want = plain(x64, w64, pos, fr, drop)
        want.backward(dy.double())
    for name, got, value in [("y", y, want.detach()), ("x", grads["x"], x64.grad), *((n, grads[n], w64[n].grad) for n in w)]:
        off = ((got.double() - value).norm() / value.norm()).item()
        assert off <= 1e-3, f"{name}: off by {off:.2g}"


def test_sublayer_step_by_step():
    """bfloat16: each call's results at what the call before it gave, views of wider rows
    among them, within that call's own bounds."""
    say("packed sublayer bfloat16")
    x, dy, w, starts, pos, fr = setup(BF16, 1)
    _, kept = sublayer(x, w, starts, pos, fr)
    _, (do, dqr, dkr, dv, dq, dk) = backward(dy, x, w, starts, pos, fr, kept)
    _, q, k, v, qr, kr, o, _, _ = kept
    for t, weight, dyt, y, dx in ((q, w["q"], dqr, qr, dq), (k, w["k"], dkr, kr, dk)):
        wy, wdx, _ = R.norm_rotary(t, weight, pos, fr, (PAIRS,), dy=dyt)
        O.check(y, wy, "rotated")
        O.check(dx, wdx, "its gradient")
    want = O.attention(qr, kr, v, starts.tolist(), scale=SCALE, causal=True, dout=do)
    for name, got in (("out", o), ("dq", dqr), ("dk", dkr), ("dv", dv)):
        O.check(got, want[name], name)


def test_sublayer_captured():
    """Both directions in one graph; each replay gives what the calls give at its inputs."""
    say("packed sublayer captured")
    x, dy, w, starts, pos, fr = setup(BF16, 2)

    def step():
        y, kept = sublayer(x, w, starts, pos, fr)
        grads, _ = backward(dy, x, w, starts, pos, fr, kept)
        return [y, *grads.values()]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x.mul_(1.1)
        dy.copy_(dy.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), f"replay {i}"


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_steps_of_one_token(dtype):
    """Tokens one by one against caches with room, captured once: what the passes over the
    whole sequences give for those rows (within the bounds of both)."""
    say(f"packed steps {dtype}")
    x, _, w, starts, pos, fr = setup(dtype, 3)
    room, first = 96, torch.tensor([45, 1, 80, 19], device="cuda") - 1  # the last tokens of each
    q, k, v = split(kernels.rms_norm(x, w["norm"]) @ w["qkv"])
    qr, kr = kernels.head_norm_rotary(q, k, pos, fr, q_weight=w["q"], k_weight=w["k"])
    want = O.attention(qr, kr, v, starts.tolist(), scale=SCALE, causal=True)["out"]
    whole = kernels.packed_attention(qr, kr, v, starts, scale=SCALE, causal=True)
    last = starts[1:].long() - 1
    cache_k, cache_v = (torch.full((KV, len(LENS) * room, D), torch.nan, dtype=dtype, device="cuda") for _ in range(2))
    for i, n in enumerate(LENS):
        rows = slice(starts[i].item(), starts[i].item() + n - 1)
        cache_k[:, i * room:i * room + n - 1], cache_v[:, i * room:i * room + n - 1] = kr[:, rows], v[:, rows]
    k_starts = torch.arange(0, (len(LENS) + 1) * room, room, device="cuda", dtype=torch.int32)
    lengths = (first + 1).to(torch.int32)
    slot = k_starts[:-1].long() + first
    one = torch.arange(len(LENS) + 1, device="cuda", dtype=torch.int32)
    q1, k1, v1 = (t[:, last].contiguous() for t in (q, k, v))
    p1 = pos[:, last].contiguous()

    def step():
        a, b = kernels.head_norm_rotary(q1, k1, p1, fr, q_weight=w["q"], k_weight=w["k"])
        cache_k.index_copy_(1, slot, b)
        cache_v.index_copy_(1, slot, v1)
        return kernels.packed_attention(a, cache_k, cache_v, one, scale=SCALE, causal=True, k_starts=k_starts, k_lengths=lengths)

    got = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    value, bound = (t[:, last] for t in want)
    O.check(got, (value, bound), "token")
    O.check(whole[:, last], (value, bound), "whole")
    for _ in range(3):
        cache_k.index_fill_(1, slot, torch.nan)
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, got)
