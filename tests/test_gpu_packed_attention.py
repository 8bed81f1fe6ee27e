"""Attention over packed sequences on the GPU, against 64 bits and value by value
(the bounds' derivation: tests/packed_oracle.py)."""

from __future__ import annotations

import math

import pytest
import torch

from foldjax_amd import kernels
from tests import packed_oracle as O
from tests.gpu_util import say

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def heads(g, tokens, count, d, dtype, by=1.0, major="token"):
    t = (by * torch.randn(tokens, count, d, generator=g, device="cuda")).to(dtype).transpose(0, 1)
    return t.contiguous() if major == "head" else t


def inputs(lens, h, kv, d, dtype, *, tail=0, seed=0, major="token"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(lens) + tail
    return (heads(g, n, h, d, dtype, 1.3, major), heads(g, n, kv, d, dtype, 1.3, major), heads(g, n, kv, d, dtype, 1.0, major),
            heads(g, n, h, d, dtype, 1.0, major))


def run(q, k, v, st, dout=None, **more):
    if dout is None:
        return {"out": kernels.packed_attention(q, k, v, st, **more)}
    out, lse, rest = kernels.packed_attention(q, k, v, st, return_lse=True, **more)
    dq, dk, dv = kernels.packed_attention_backward(dout, q, k, v, out, lse, rest, st, **more)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def compare(got, want):
    for name, bound in want.items():
        O.check(got[name], bound, name)


# lengths of zero and one, of whole tiles and blocks and one more or less
RAGGED = [[37], [1], [1, 0, 1, 2], [0, 0, 5], [16, 17, 15], [63, 64, 65], [127, 128, 129, 1], [0, 200, 0, 33, 0]]


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("lens", RAGGED, ids=str)
def test_lengths(lens, causal, dtype):
    for h, kv, d in ((4, 4, 24), (4, 1, 64), (6, 2, 128)):
        say(f"packed {lens} {causal} {dtype} {h} {kv} {d}")
        q, k, v, dout = inputs(lens, h, kv, d, dtype, tail=3, seed=d)
        more = {"scale": d**-0.5, "causal": causal}
        got = run(q, k, v, ints(starts(lens)), dout, **more)
        torch.cuda.synchronize()
        compare(got, O.attention(q, k, v, starts(lens), dout=dout, **more))
        assert all((t[:, sum(lens):] == 0).all() for t in got.values())


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 64, 72, 96, 120, 128])
def test_widths(d, dtype):
    say(f"packed width {d} {dtype}")
    lens = [70, 9, 131]
    q, k, v, dout = inputs(lens, 4, 2, d, dtype, seed=d)
    more = {"scale": d**-0.5, "causal": True}
    compare(run(q, k, v, ints(starts(lens), torch.int64), dout, **more), O.attention(q, k, v, starts(lens), dout=dout, **more))


# enough rows for tiles of a wave's own (one and two), and more
@pytest.mark.parametrize("lens,h,kv,d,dtype", [
    ([1003, 499, 546], 16, 16, 24, BF16), ([1500, 3, 701], 16, 4, 64, BF16), ([2048], 16, 16, 128, BF16),
    ([2200, 1, 300], 8, 1, 128, BF16), ([700, 324], 16, 16, 32, FP32), ([900, 200], 16, 4, 64, FP32),
    ([600, 450], 16, 8, 128, FP32),
])
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_rows_of_their_own(lens, h, kv, d, dtype, causal):
    say(f"packed own rows {lens} {h} {kv} {d} {dtype} {causal}")
    q, k, v, dout = inputs(lens, h, kv, d, dtype, seed=5)
    more = {"scale": d**-0.5, "causal": causal}
    compare(run(q, k, v, ints(starts(lens)), dout, **more), O.attention(q, k, v, starts(lens), dout=dout, **more))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("nq", [1, 2, 5])
@pytest.mark.parametrize("h,kv,d", [(8, 2, 128), (4, 4, 32), (16, 1, 64)])
def test_tokens_against_a_cache(h, kv, d, nq, dtype):
    """Caches with room, whose unused places hold infinities and NaN; lengths of
    zero, below the queries' and of whole blocks."""
    lens, cap = [1000, 0, 1, 128, 1023, 129, 4], 1024
    say(f"packed cache {h} {kv} {d} {nq} {dtype}")
    g = torch.Generator(device="cuda").manual_seed(nq)
    n = len(lens)
    q, dout = (heads(g, n * nq, h, d, dtype) for _ in range(2))
    k, v = (heads(g, n * cap, kv, d, dtype, major="head") for _ in range(2))
    for i, m in enumerate(lens):
        k[:, i * cap + m:(i + 1) * cap] = math.inf
        v[:, i * cap + m:(i + 1) * cap] = math.nan
    qs, ks = [nq * i for i in range(n + 1)], [cap * i for i in range(n + 1)]
    more = {"scale": d**-0.5, "causal": True}
    got = run(q, k, v, ints(qs), dout, k_starts=ints(ks), k_lengths=ints(lens), **more)
    compare(got, O.attention(q, k, v, qs, k_starts=ks, k_lengths=lens, dout=dout, **more))


def test_long_cache_split_over_workgroups():
    say("packed long cache")
    lens, cap, h, kv, d = [16001, 9, 5000], 16384, 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    q = heads(g, 3, h, d, BF16)
    k, v = (heads(g, 3 * cap, kv, d, BF16, major="head") for _ in range(2))
    ks = [0, cap, 2 * cap, 3 * cap]
    got = run(q, k, v, ints([0, 1, 2, 3]), k_starts=ints(ks), k_lengths=ints(lens), scale=0.125, causal=True)
    compare(got, O.attention(q, k, v, [0, 1, 2, 3], k_starts=ks, k_lengths=lens, scale=0.125, causal=True))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_strides_and_alignment(dtype):
    """Heads side by side, tokens side by side, slices of wider rows, and tensors that
    have to be copied; the same results from all."""
    say(f"packed strides {dtype}")
    lens, d = [40, 25, 70], 32
    q, k, v, dout = inputs(lens, 4, 2, d, dtype, seed=1, major="head")
    more = {"scale": 0.2, "causal": True}
    want = run(q, k, v, ints(starts(lens)), dout, **more)

    def in_wider(t):  # every second 32 channels of rows of 64
        w = torch.full((*t.shape[:2], 64), math.nan, dtype=dtype, device="cuda")
        w[..., 32:] = t
        return w[..., 32:]

    def odd(t):  # an address that is no multiple of 16 bytes
        w = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape)
        return w.copy_(t)

    def turned(t):  # channels apart
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    for form in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), in_wider, odd, turned):
        got = run(*(form(t) for t in (q, k, v)), ints(starts(lens)), form(dout), **more)
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_out_and_the_rows_behind_the_last_sequence():
    say("packed out")
    lens, d = [40, 25], 24
    q, k, v, _ = inputs(lens, 4, 4, d, BF16, tail=30, seed=2)
    st = ints(starts(lens))
    want = kernels.packed_attention(q, k, v, st, scale=0.2)
    assert (want[:, 65:] == 0).all()
    for long in (False, True):  # rows of their own, and a cache over several workgroups
        if long:
            k, v = (t.repeat(1, 40, 1) for t in (k, v))
            ks = ints([0, 1500, 3700])
            more = {"k_starts": ks, "scale": 0.2}
        else:
            more = {"scale": 0.2}
        want = kernels.packed_attention(q, k, v, st, **more)
        out = torch.full((95, 4, 32), 7.0, dtype=BF16, device="cuda")[..., :24].transpose(0, 1)
        got = kernels.packed_attention(q, k, v, st, out=out, **more)
        assert got is out and torch.equal(out[:, :65], want[:, :65]) and (out[:, 65:] == 7.0).all()


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_digits_of_rows_with_one_heavy_key(dtype):
    """dP - D is what the other keys leave of it: within the bounds, which are
    relative to that."""
    say(f"packed heavy key {dtype}")
    n, d = 70, 64
    q, k, v, dout = inputs([n], 2, 2, d, dtype, seed=9)
    k = k.contiguous()
    k[:, 11] = 4.0 * torch.sign(q.float().mean(1)).to(dtype)
    q = (0.05 * q.float() + 0.5 * k[:, 11:12].float()).to(dtype)  # scores of about 60 at key 11, of 1 elsewhere
    got = run(q, k, v, ints([0, n]), dout, scale=0.125)
    compare(got, O.attention(q, k, v, [0, n], scale=0.125, dout=dout))


def test_scores_far_from_zero():
    """Maxima beyond 2^24 in log2 units: ties share the weight, whatever the rounding
    of the maximum."""
    say("packed far scores")
    d = 32
    q = torch.full((1, 20, d), 2.0**14, dtype=BF16, device="cuda")
    k = torch.full((1, 20, d), 2.0**14, dtype=BF16, device="cuda")
    k[:, 10:] = -k[:, 10:]
    g = torch.Generator(device="cuda").manual_seed(1)
    v, dout = (torch.randn(1, 20, d, generator=g, device="cuda").to(BF16) for _ in range(2))
    got = run(q, k, v, ints([0, 20]), dout, scale=0.3)
    want = v[:, :10].double().mean(1, keepdim=True).expand(1, 20, d)
    # ten equal weights, exact, and their sum; the output's rounding
    assert ((got["out"].double() - want).abs() <= 2.0**-8 * want.abs() + 1e-6).all()
    assert all(torch.isfinite(t).all() for t in got.values())
    # dv: each row's tenth of dO for the first ten keys, none for the others (0.1 rounded to bf16)
    dv = 0.1 * dout.double().sum(1, keepdim=True)
    assert ((got["dv"][:, :10].double() - dv).abs() <= 2.0**-8 * (0.1 * dout.double().abs().sum(1) + dv.abs()) + 1e-6).all()
    assert (got["dv"][:, 10:] == 0).all()


def test_the_same_bits_each_time():
    say("packed determinism")
    lens = [900, 700, 448]
    q, k, v, dout = inputs(lens, 8, 2, 128, BF16, seed=4)
    more = {"scale": 0.09, "causal": True}
    a, b = (run(q, k, v, ints(starts(lens)), dout, **more) for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_offsets_that_lead_out_of_the_buffers():
    """Taken as the buffers' ends (below zero: the start): as if the lengths had ended there."""
    say("packed offsets out of range")
    lens = [40, 25, 30]
    q, k, v, _ = inputs(lens, 4, 2, 64, BF16, seed=2)
    want = kernels.packed_attention(q, k, v, ints([0, 40, 95]), scale=0.1)
    for dt in (torch.int32, torch.int64):
        got = kernels.packed_attention(q, k, v, ints([-7, 40, 2**31 - 1], dt), scale=0.1)
        assert torch.equal(got, want)
    big = ints([0, 40, 2**40], torch.int64)
    assert torch.equal(kernels.packed_attention(q, k, v, big, scale=0.1, k_lengths=ints([1000, 2**31 - 1])), want)
    assert (kernels.packed_attention(q, k, v, ints([0, 40, 95]), scale=0.1, k_lengths=ints([-5, -1])) == 0).all()


def test_streams_and_graphs():
    """On another stream than the current one's, and captured: a replay takes the
    lengths and inputs that are there."""
    say("packed streams and graphs")
    lens = [300, 200, 12]
    q, k, v, dout = inputs(lens, 4, 2, 64, BF16, seed=6)
    st = ints(starts(lens))
    more = {"scale": 0.125, "causal": True}
    want = run(q, k, v, st, dout, **more)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, k, v, st, dout, **more)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = run(q, k, v, st, dout, **more)
    for i in range(4):
        st.copy_(ints(starts([300 - 50 * i, 200 + 40 * i, 12 + 10 * i])))
        q.copy_(q + 0.01 * i)
        g.replay()
        torch.cuda.synchronize()
        want = run(q, k, v, st, dout, **more)
        assert all(torch.equal(held[n], want[n]) for n in want)
        (dout.float() * 2).sum().item()


def test_two_captured_calls_keep_their_workspaces():
    say("packed two graphs")
    cap, h, kv, d = 4096, 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(8)
    k, v = (heads(g, cap, kv, d, BF16, major="head") for _ in range(2))
    qs = [heads(g, 1, h, d, BF16) for _ in range(2)]
    more = {"k_starts": ints([0, cap]), "k_lengths": ints([cap - 5]), "scale": 0.125, "causal": True}
    st = ints([0, 1])
    want = [kernels.packed_attention(q, k, v, st, **more) for q in qs]
    graphs, held = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, q in zip(graphs, qs):
        with torch.cuda.graph(graph):
            held.append(kernels.packed_attention(q, k, v, st, **more))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        for s, graph in zip((a, b), graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, want))


def test_without_tokens():
    say("packed without tokens")
    q = torch.zeros(4, 0, 32, dtype=BF16, device="cuda")
    k = torch.zeros(2, 0, 32, dtype=BF16, device="cuda")
    assert kernels.packed_attention(q, k, k, ints([0, 0, 0]), scale=1.0).shape == (4, 0, 32)
    q = torch.ones(4, 5, 32, dtype=BF16, device="cuda")
    out, lse, rest = kernels.packed_attention(q, k, k, ints([0, 2, 5]), k_starts=ints([0, 0, 0]), scale=1.0, return_lse=True)
    assert (out == 0).all() and (rest == 0).all()
    dq, dk, dv = kernels.packed_attention_backward(q, q, k, k, out, lse, rest, ints([0, 2, 5]), k_starts=ints([0, 0, 0]), scale=1.0)
    assert (dq == 0).all() and dk.shape == dv.shape == k.shape


def test_gradients_against_differences():
    """The gradient along a direction is the change of sum(out * dout) along it, in
    float32: the difference's own error is its third derivative's, h^2, and 2^-24 / h of
    the terms' absolute sum."""
    say("packed differences")
    lens, d = [33, 20], 16
    q, k, v, dout = inputs(lens, 4, 2, d, FP32, seed=11)
    st, more = ints(starts(lens)), {"scale": 0.25, "causal": True}
    g = run(q, k, v, st, dout, **more)
    gen = torch.Generator(device="cuda").manual_seed(12)
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        way = torch.randn(t.shape, generator=gen, device="cuda")
        way /= way.norm()
        step = 1e-2

        def value(sign):
            args = [x + sign * step * way if x is t else x for x in (q, k, v)]
            return (kernels.packed_attention(*args, st, **more).double() * dout.double()).sum()

        slope = (value(1) - value(-1)) / (2 * step)
        want = (g[name].double() * way.double()).sum()
        noise = 2.0**-22 / step * (g["out"].double() * dout.double()).abs().sum()
        assert abs(slope - want) <= noise + 10 * step**2 * g[name].double().norm()
