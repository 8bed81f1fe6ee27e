"""Packed attention's longer ways on the GPU: tiles in the order of their work, many
sequences, launches in parts, caches past 32 bits, workspaces, against 64 bits value by
value (the bounds' derivation: tests/packed_oracle.py)."""

from __future__ import annotations

import pytest
import torch

from foldjax_amd import _lib, kernels
from tests import packed_oracle as O
from tests.gpu_util import say
from tests.test_gpu_packed_attention import BF16, FP32, compare, heads, inputs, ints, run, starts

pytestmark = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])


# so much work that the tiles are sorted by it: long sequences, with short ones between
@DTYPES
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_tiles_in_the_order_of_their_work(causal, dtype):
    say(f"packed sorted {causal} {dtype}")
    lens = [3500, 0, 130, 2371]
    q, k, v, dout = inputs(lens, 8, 2, 32, dtype, tail=1000, seed=21)
    more = {"scale": 0.18, "causal": causal}
    got = run(q, k, v, ints(starts(lens)), dout, **more)
    compare(got, O.attention(q, k, v, starts(lens), dout=dout, **more))
    assert all((t[:, sum(lens):] == 0).all() for t in got.values())


@DTYPES
def test_sorted_tiles_against_caches(dtype):
    """Chunks of new tokens: queries and caches of different lengths, one cache without
    room left, one shorter than its queries."""
    say(f"packed sorted caches {dtype}")
    lens, room, length = [2000, 900, 50, 1300], [3000, 900, 70, 4000], [2700, 900, 20, 3999]
    g = torch.Generator(device="cuda").manual_seed(22)
    q, dout = (heads(g, sum(lens), 8, 64, dtype) for _ in range(2))
    k, v = (heads(g, sum(room), 2, 64, dtype, major="head") for _ in range(2))
    for i, n in enumerate(length):
        at = starts(room)[i]
        k[:, at + n:at + room[i]] = torch.nan
        v[:, at + n:at + room[i]] = torch.inf
    more = {"scale": 0.125, "causal": True}
    got = run(q, k, v, ints(starts(lens), torch.int64), dout, k_starts=ints(starts(room), torch.int64),
              k_lengths=ints(length, torch.int64), **more)
    compare(got, O.attention(q, k, v, starts(lens), k_starts=starts(room), k_lengths=length, dout=dout, **more))


# at and past the number of sequences of which a wave's lanes hold one each
@DTYPES
@pytest.mark.parametrize("count", [62, 63, 64, 65, 300])
def test_many_sequences(count, dtype):
    say(f"packed {count} sequences {dtype}")
    lens = [(7 * i * i) % 41 * (i % 5 != 2) for i in range(count)]
    q, k, v, dout = inputs(lens, 4, 2, 24, dtype, tail=9, seed=count)
    more = {"scale": 0.2, "causal": True}
    got = run(q, k, v, ints(starts(lens)), dout, **more)
    compare(got, O.attention(q, k, v, starts(lens), dout=dout, **more))
    assert all((t[:, sum(lens):] == 0).all() for t in got.values())


def test_many_sequences_sorted():
    say("packed many sequences sorted")
    lens = [30 + i for i in range(40)] + [6000, 0, 5000] + [3 * i for i in range(40)] + [4000]
    q, k, v, dout = inputs(lens, 16, 2, 16, BF16, seed=23)
    more = {"scale": 0.25, "causal": True}
    compare(run(q, k, v, ints(starts(lens)), dout, **more), O.attention(q, k, v, starts(lens), dout=dout, **more))


def test_more_tiles_than_a_launch_has():
    """70000 sequences of one token: each has its own value, and dS is what float32 leaves
    of dP - D, two sums of d + 2 products."""
    say("packed 70000 sequences")
    n, d = 70000, 8
    q, k, v, dout = inputs([n], 2, 1, d, BF16, tail=1, seed=24)
    got = run(q, k, v, torch.arange(n + 1, device="cuda", dtype=torch.int32), dout, scale=0.3, causal=True)
    assert torch.equal(got["out"][:, :n], v[:, :n].expand(2, n, d)) and (got["out"][:, n:] == 0).all()
    dv = dout.double().sum(0, keepdim=True)
    dv[:, n:] = 0
    assert ((got["dv"].double() - dv).abs() <= 2.0**-8 * dv.abs() + 2.0**-22 * dout.double().abs().sum(0, keepdim=True)).all()
    left = 0.3 * 2 * (d + 2) * 2.0**-24 * 1.05 * (dout.double().abs() * v.double().abs()).sum(-1, keepdim=True)
    assert (got["dq"].double().abs() <= left * k.double().abs()).all()
    assert (got["dk"].double().abs() <= (left * q.double().abs()).sum(0, keepdim=True)).all()


def test_caches_past_32_bits():
    """Two caches in 17 million places of 256 bytes, the second all of them but a few: one
    key of each has nearly all the weight, which the 2^24 others share e^-30 of at most."""
    say("packed cache past 32 bits")
    d, tk, first = 128, 17_000_000, 100
    k, v = (torch.zeros(1, tk, d, dtype=BF16, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(25)
    q = torch.ones(2, 2, d, dtype=BF16, device="cuda")
    for at in (40, tk - 3):
        k[:, at] = 0.5  # a score of 32
        v[:, at] = torch.randn(d, generator=g, device="cuda").to(BF16)
    more = {"k_starts": ints([0, first, tk]), "k_lengths": ints([90, tk - first - 1]), "scale": 0.5, "causal": True}
    dout = heads(g, 2, 2, d, BF16)
    got = run(q, k, v, ints([0, 1, 2]), dout, **more)
    for row, at in ((0, 40), (1, tk - 3)):
        want = v[0, at].double()
        assert ((got["out"][:, row].double() - want).abs() <= (2.0**-8 + 2e-6) * want.abs()).all()
        want = dout[:, row].double().sum(0)
        size = dout[:, row].double().abs().sum(0)
        assert ((got["dv"][0, at].double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-8 * size + 2e-6 * size).all()
    assert (got["dv"][0, -1] == 0).all() and (got["dk"][0, -1] == 0).all() and (got["dk"][0, 90:100] == 0).all()


@DTYPES
@pytest.mark.parametrize("lens,room,h,kv,d", [([1] * 3, 4000, 8, 2, 64), ([1], 16384, 4, 4, 24), ([2, 1, 5], 1500, 8, 1, 128),
                                              ([3500, 130, 2371], 0, 8, 2, 32), ([70, 9, 131], 0, 4, 2, 40)])
def test_writes_stay_in_the_workspace(lens, room, h, kv, d, dtype):
    """The workspaces, of just the size that is asked for, lie between bytes that stay."""
    say(f"packed workspace {lens} {room} {dtype}")
    g = torch.Generator(device="cuda").manual_seed(26)
    caches = [room] * len(lens) if room else lens
    q, dout = (heads(g, sum(lens), h, d, dtype) for _ in range(2))
    k, v = (heads(g, sum(caches), kv, d, dtype) for _ in range(2))
    st, ks = ints(starts(lens)), ints(starts(caches))
    want = run(q, k, v, st, dout, scale=0.1, k_starts=ks, causal=True)
    lib = _lib.load()
    sizes = [f(sum(lens), sum(caches), len(lens), h, kv, d, 0 if dtype is FP32 else 1)
             for f in (lib.fjx_packed_attention_workspace_size, lib.fjx_packed_attention_bwd_workspace_size)]
    guard, real, asked = 4096, torch.empty, []
    around = []

    def empty(*shape, **more):
        if more.get("dtype") is not torch.uint8:
            return real(*shape, **more)
        n, = shape
        asked.append(n)
        t = torch.full((n + 2 * guard,), 0xA5, dtype=torch.uint8, device="cuda")
        around.append(t)
        return t[guard:guard + n]

    torch.empty = empty
    try:
        got = run(q, k, v, st, dout, scale=0.1, k_starts=ks, causal=True)
    finally:
        torch.empty = real
    assert asked == [n for n in sizes if n]
    assert all((t[:guard] == 0xA5).all() and (t[-guard:] == 0xA5).all() for t in around)
    assert all(torch.equal(got[n], want[n]) for n in want)


# so many workgroups that a wave has two tiles of rows, and of keys; and float32 with two waves a tile
@pytest.mark.parametrize("lens,h,kv,d,dtype", [([330] * 20 + [1700], 16, 16, 24, BF16), ([400, 37, 363] * 11, 16, 16, 64, BF16),
                                               ([900, 1, 700], 16, 16, 128, FP32), ([2000, 1100], 16, 8, 128, FP32)])
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_many_workgroups(lens, h, kv, d, dtype, causal):
    say(f"packed many workgroups {len(lens)} {d} {dtype} {causal}")
    q, k, v, dout = inputs(lens, h, kv, d, dtype, seed=27)
    more = {"scale": d**-0.5, "causal": causal}
    compare(run(q, k, v, ints(starts(lens)), dout, **more), O.attention(q, k, v, starts(lens), dout=dout, **more))


@pytest.mark.parametrize("h,kv", [(1024, 1), (96, 1), (90, 2), (1000, 1000)])
def test_many_heads(h, kv):
    """Groups of heads that are no powers of two and of more heads than a tile has rows."""
    say(f"packed heads {h} {kv}")
    lens = [3, 1, 17]
    q, k, v, dout = inputs(lens, h, kv, 8, BF16, tail=2, seed=h)
    more = {"scale": 0.35, "causal": True}
    compare(run(q, k, v, ints(starts(lens)), dout, **more), O.attention(q, k, v, starts(lens), dout=dout, **more))
    room = [100, 90, 300]  # a cache, walked by waves with keys of their own
    g = torch.Generator(device="cuda").manual_seed(h)
    k, v = (heads(g, sum(room), kv, 8, BF16) for _ in range(2))
    got = run(q, k, v, ints(starts(lens)), dout, k_starts=ints(starts(room)), **more)
    compare(got, O.attention(q, k, v, starts(lens), k_starts=starts(room), dout=dout, **more))


def test_gradients_of_keys_without_queries():
    say("packed no queries")
    k = torch.ones(2, 50, 32, dtype=BF16, device="cuda")
    q = torch.ones(4, 0, 32, dtype=BF16, device="cuda")
    more = {"k_starts": ints([0, 20, 45]), "scale": 1.0}
    out, lse, rest = kernels.packed_attention(q, k, k, ints([0, 0, 0]), return_lse=True, **more)
    for t in kernels.packed_attention_backward(q, q, k, k, out, lse, rest, ints([0, 0, 0]), **more):
        assert t.shape[1] in (0, 50) and (t == 0).all()


def test_offsets_of_two_types_and_of_every_second_place():
    say("packed offsets of two types")
    lens, d = [40, 25, 30], 32
    q, k, v, dout = inputs(lens, 4, 2, d, BF16, seed=28)
    st = starts(lens)
    want = run(q, k, v, ints(st), dout, scale=0.2, k_starts=ints(st), k_lengths=ints([40, 20, 30]))
    apart = torch.stack([ints(st), ints(st) - 7], 1)[:, 0]
    got = run(q, k, v, apart, dout, scale=0.2, k_starts=ints([*st[:-1], 2**40], torch.int64), k_lengths=ints([40, 20, 2**33 + 1], torch.int64))
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_heads_that_are_one():
    """k and v broadcast over heads, q over tokens: taken by copies, gradients of each place."""
    say("packed broadcast")
    lens, d = [30, 9], 16
    q, k, v, dout = inputs(lens, 4, 4, d, FP32, seed=29)
    q, k, v = q[:, :1].expand(-1, 39, -1), k[:1].expand(4, -1, -1), v[:1].expand(4, -1, -1)
    got = run(q, k, v, ints(starts(lens)), dout, scale=0.3, causal=True)
    compare(got, O.attention(q, k, v, starts(lens), scale=0.3, causal=True, dout=dout))


@DTYPES
@pytest.mark.parametrize("size", [2.0**10, 2.0**12, 2.0**20, 2.0**23])
def test_equal_scores_of_any_size(size, dtype):
    """Scores that are all the same have the same weights, 1 / 20, however far from zero, beside
    rows of small scores: the weight's own rounding, a sum of 20 and the output's."""
    say(f"packed equal scores {size} {dtype}")
    n, d = 20, 32
    root = 2.0 ** int(torch.tensor(size).log2().item() // 2)
    q, k = (torch.zeros(2, n, d, dtype=dtype, device="cuda") for _ in range(2))
    q[0, :, 0], k[..., 0] = size / root, root
    g = torch.Generator(device="cuda").manual_seed(30)
    v, dout = (torch.randn(2, n, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    got = run(q, k, v, ints([0, n]), dout, scale=0.7)
    u = torch.finfo(dtype).eps / 2 + 40 * 2.0**-24
    want, room = v.double().mean(1, keepdim=True), v.double().abs().mean(1, keepdim=True)
    assert ((got["out"].double() - want).abs() <= u * (2 * room + want.abs())).all()
    want, room = dout.double().mean(1, keepdim=True), dout.double().abs().mean(1, keepdim=True)
    assert ((got["dv"].double() - want).abs() <= u * (2 * room + want.abs())).all()


def test_captured_with_other_lengths():
    """A captured step whose tiles are sorted and whose key tiles have parts: a replay orders
    and deals them by the lengths that are there; two such graphs at once keep their own."""
    say("packed captured sorted")
    tokens, more = 6200, {"scale": 0.18, "causal": True}
    q, k, v, dout = inputs([tokens], 8, 2, 32, BF16, seed=32)
    plans = [[3000, 2100, 1000], [40, 6000, 100], [6100, 0, 100], [2000, 2000, 2200]]
    sides = []
    for i in range(2):
        st, graph = ints(starts(plans[i])), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run(q, k, v, st, dout, **more)
        sides.append((st, graph, held, torch.cuda.Stream()))
    for turn in range(4):
        for i, (st, graph, _, stream) in enumerate(sides):
            st.copy_(ints(starts(plans[(turn + i) % 4])))
        for _, graph, _, stream in sides:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for st, _, held, _ in sides:
            want = run(q, k, v, st, dout, **more)
            assert all(torch.equal(held[n], want[n]) for n in want), turn
