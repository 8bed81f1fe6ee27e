"""The heads' norm with rotation on the GPU, against 64 bits and value by value (the
bounds' derivation: tests/rotary_oracle.py)."""

from __future__ import annotations

import math

import pytest
import torch

from foldjax_amd import kernels
from tests import rotary_oracle as R
from tests.gpu_util import say
from tests.packed_oracle import check

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32
DTYPES = pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def heads(g, lead, count, tokens, d, dtype):
    t = torch.randn(*lead, tokens, count, d, generator=g, device="cuda").to(dtype)
    return t.transpose(-3, -2)


def weights(g, d, dtype):
    return [(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype) for _ in range(2)]


def freqs(pairs):
    return 10000.0 ** -(torch.arange(pairs, dtype=torch.float64, device="cuda") / max(pairs, 1))


def places(axes, tokens, lead=(), far=0, dtype=torch.int32):
    g = torch.Generator().manual_seed(tokens)
    return (torch.randint(0, 2000, (axes, *lead, tokens), generator=g) + far).to("cuda", dtype)


def run(q, k, wq, wk, pos, fr, sections, interleaved, dq, dk, eps=1e-6):
    more = {"q_weight": wq, "k_weight": wk, "eps": eps, "sections": sections, "interleaved": interleaved}
    yq, yk = kernels.head_norm_rotary(q, k, pos, fr, **more)
    gq, gk, gwq, gwk = kernels.head_norm_rotary_backward(dq, dk, q, k, pos, fr, **more)
    for x, w, y, dy, dx, dw, name in ((q, wq, yq, dq, gq, gwq, "q"), (k, wk, yk, dk, gk, gwk, "k")):
        if x is None:
            assert y is None and dx is None and dw is None
            continue
        ref = R.norm_rotary(x, w, pos, fr, sections or (fr.shape[0],), interleaved, eps, dy)
        check(y, ref[0], f"y {name}")
        check(dx, ref[1], f"dx {name}")
        assert (dw is None) == (w is None)
        if w is not None:
            check(dw, ref[2], f"dw {name}")


@DTYPES
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("d,sections", [(8, (4,)), (24, (4, 4, 4)), (24, (8,)), (32, (16,)), (40, (20,)), (64, (16, 8)),
                                        (128, (16, 24, 24)), (128, (5, 3, 7, 1)), (72, (0, 36)), (256, (128,)), (64, (0,))])
def test_widths_and_axes(d, sections, interleaved, dtype):
    say(f"rotary {d} {sections} {interleaved} {dtype}")
    g = gen(d)
    tokens = 37
    q, dq = (heads(g, (), 5, tokens, d, dtype) for _ in range(2))
    k, dk = (heads(g, (), 2, tokens, d, dtype) for _ in range(2))
    wq, wk = weights(g, d, dtype)
    run(q, k, wq, wk, places(len(sections), tokens), freqs(sum(sections)), sections, interleaved, dq, dk)


@DTYPES
@pytest.mark.parametrize("lead,h,kv,tokens", [((), 1, 1, 1), ((3,), 4, 4, 1), ((2, 2), 3, 1, 5), ((), 8, 2, 700), ((8,), 16, 16, 33),
                                              ((), 12, 0, 5000), ((), 40, 8, 9)])
@pytest.mark.parametrize("norm", ["both", "none", "q"])
def test_shapes_and_norms(lead, h, kv, tokens, norm, dtype):
    say(f"rotary {lead} {h} {kv} {tokens} {norm} {dtype}")
    g = gen(h)
    d = 32
    q, dq = (heads(g, lead, h, tokens, d, dtype) for _ in range(2))
    k, dk = ((heads(g, lead, kv, tokens, d, dtype) for _ in range(2)) if kv else (None, None))
    wq, wk = weights(g, d, dtype)
    wq = None if norm == "none" else wq
    wk = wk if norm == "both" and kv else None
    run(q, k, wq, wk, places(1, tokens, lead, dtype=torch.int64), freqs(16), None, False, dq, dk)


@DTYPES
def test_positions_for_all_items_and_far_ones(dtype):
    """Positions of 2^31 - 2000 and more: the angles are exact to 2^-24 of a turn."""
    say(f"rotary far {dtype}")
    g = gen(3)
    q, dq = (heads(g, (2,), 2, 50, 64, dtype) for _ in range(2))
    k, dk = (heads(g, (2,), 1, 50, 64, dtype) for _ in range(2))
    wq, wk = weights(g, 64, dtype)
    for far in (0, 10**6, 2**31 - 2000 - 1):
        run(q, k, wq, wk, places(1, 50, far=far), freqs(32), (32,), False, dq, dk)
    run(q, k, wq, wk, -places(1, 50, far=10**5), freqs(32), (32,), True, dq, dk)


@DTYPES
def test_strides_outputs_and_inputs_that_are_outputs(dtype):
    say(f"rotary strides {dtype}")
    g = gen(4)
    q = heads(g, (), 4, 21, 64, dtype)
    k = heads(g, (), 2, 21, 64, dtype)
    wq, wk = weights(g, 64, dtype)
    pos, fr = places(1, 21), freqs(32)
    more = {"q_weight": wq, "k_weight": wk}
    yq, yk = kernels.head_norm_rotary(q, k, pos, fr, **more)
    odd = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    turned = k.transpose(1, 2).contiguous().transpose(1, 2)
    for a, b in ((q.contiguous(), k.contiguous()), (odd, turned)):
        got = kernels.head_norm_rotary(a, b, pos, fr, **more)
        assert torch.equal(got[0], yq) and torch.equal(got[1], yk)
    # keys into their places in a cache, whose other places stay as they are
    cache = torch.full((2, 100, 64), 7.0, dtype=dtype, device="cuda")
    a = q.clone()
    got = kernels.head_norm_rotary(a, k, pos, fr, q_out=a, k_out=cache[:, 40:61], **more)
    assert got[0] is a and torch.equal(a, yq) and torch.equal(cache[:, 40:61], yk)
    assert (cache[:, :40] == 7).all() and (cache[:, 61:] == 7).all()
    b = k.clone()
    kernels.head_norm_rotary(q, b, pos, fr, k_out=b, **more)
    assert torch.equal(b, yk)
    # a gradient that is one row for all tokens
    one = torch.ones(4, 1, 64, dtype=dtype, device="cuda").expand(4, 21, 64)
    args = (q, None, pos, fr)
    x = kernels.head_norm_rotary_backward(one, None, *args, q_weight=wq)
    y = kernels.head_norm_rotary_backward(one.contiguous(), None, *args, q_weight=wq)
    assert torch.equal(x[0], y[0]) and torch.equal(x[2], y[2])


@DTYPES
def test_rows_of_zeros_and_of_large_values(dtype):
    """A row of zeros is zeros, its gradients those of x / sqrt(eps); a NaN stays in its row."""
    say(f"rotary zeros {dtype}")
    g = gen(5)
    q, dq = (heads(g, (), 2, 9, 32, dtype).contiguous() for _ in range(2))
    q[:, 3] = 0
    q[:, 4] *= 1e15
    wq, _ = weights(g, 32, dtype)
    run(q, None, wq, None, places(1, 9), freqs(16), None, False, dq, None)
    want = kernels.head_norm_rotary(q, None, places(1, 9), freqs(16), q_weight=wq)[0]
    q[1, 5, 7] = math.nan
    got = kernels.head_norm_rotary(q, None, places(1, 9), freqs(16), q_weight=wq)[0]
    assert got[1, 5].isnan().all()
    got[1, 5] = want[1, 5]
    assert torch.equal(got, want)


def test_streams_graphs_and_the_same_bits():
    say("rotary graphs")
    g = gen(6)
    q, dq = (heads(g, (), 8, 300, 128, BF16) for _ in range(2))
    k, dk = (heads(g, (), 2, 300, 128, BF16) for _ in range(2))
    wq, wk = weights(g, 128, BF16)
    pos, fr = places(1, 300), freqs(64)
    more = {"q_weight": wq, "k_weight": wk}

    def step():
        return [*kernels.head_norm_rotary(q, k, pos, fr, **more),
                *kernels.head_norm_rotary_backward(dq, dk, q, k, pos, fr, **more)]

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        pos.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))
        q.float().sum().item()


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
def test_gradients_against_differences(interleaved):
    """The gradient along a direction of length 1 is the change of sum(y dy) along it, in
    float32: the difference's own error is its third derivative's, h^2, and 2^-22 / h of the
    terms' absolute sum."""
    say(f"rotary differences {interleaved}")
    g = gen(31)
    d, tokens = 24, 40
    q, dq = (heads(g, (2,), 3, tokens, d, torch.float32) for _ in range(2))
    k, dk = (heads(g, (2,), 1, tokens, d, torch.float32) for _ in range(2))
    wq, wk = weights(g, d, torch.float32)
    pos, fr, more = places(2, tokens), freqs(12), {"sections": (4, 8), "interleaved": interleaved}
    grads = kernels.head_norm_rotary_backward(dq, dk, q, k, pos, fr, q_weight=wq, k_weight=wk, **more)
    inputs = [q, k, wq, wk]

    def value(args):
        y = kernels.head_norm_rotary(args[0], args[1], pos, fr, q_weight=args[2], k_weight=args[3], **more)
        return sum((a.double() * b.double()).sum() for a, b in zip(y, (dq, dk))), sum(
            (a.double() * b.double()).abs().sum() for a, b in zip(y, (dq, dk)))

    step = 1e-2
    size = value(inputs)[1]
    for i, t in enumerate(inputs):
        way = torch.randn(t.shape, generator=g, device="cuda")
        way /= way.norm()
        ends = [value([x + sign * step * way if x is t else x for x in inputs])[0] for sign in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * step)
        want = (grads[i].double() * way.double()).sum()
        assert abs(slope - want) <= 2.0**-22 / step * size + 10 * step**2 * grads[i].double().norm(), i
