"""How calls of packed attention are cut (tests/packed_plan.py), on the CPU."""

from __future__ import annotations

import ctypes
import random

from foldjax_amd import _lib
from tests.packed_plan import plans


def calls(count, seed):
    rng = random.Random(seed)
    log = lambda most: int(2 ** rng.uniform(0, most))  # noqa: E731
    for _ in range(count):
        kv = rng.choice([1, 2, 4, 6, 16])
        seqs = log(8)
        yield log(15), log(18), seqs, kv * rng.choice([1, 2, 4, 8]), kv, 8 * rng.randint(1, 16), rng.random() < 0.6


def test_the_library_is_cut_so():
    """The workspaces of the rules as compiled here are those that the library asks for."""
    lib = _lib.load()
    some = list(calls(3000, 1))
    sizes = set()
    for c, p in zip(some, plans(some)):
        assert lib.fjx_packed_attention_workspace_size(*c[:6], int(c[6])) == p.forward_bytes, c
        assert lib.fjx_packed_attention_bwd_workspace_size(*c[:6], int(c[6])) == p.backward_bytes, c
        sizes.add((p.forward[:3], p.forward.sorted, p.splits > 1, p.keys[:3], p.keys.sorted, p.parts > 1))
    assert len(sizes) > 20


def test_tiles_cover_the_rows():
    """Tiles for every row, one more for each sequence and for the rows behind the last."""
    some = list(calls(2000, 2))
    for (tq, tk, seqs, heads, kv, _, _), p in zip(some, plans(some)):
        for form, rows in ((p.forward, tq * heads // kv), (p.dq, tq * heads // kv), (p.keys, tk)):
            assert form.count == rows // (16 * form.groups * form.tiles) + seqs + 1


def test_two_tiles_a_wave_where_they_were_measured_faster():
    """Forward: from 768 workgroups of 64 rows on at more than 64 channels, 1024 below; a wave
    has all keys of a block from 2048 and 3200 on."""
    for d, pairs, alone in ((128, 768, 2048), (72, 768, 2048), (64, 1024, 3200), (24, 1024, 3200)):
        wgs = [640, pairs - 2, pairs, alone - 2, alone, 2 * alone]
        got = plans([(n * 16, n * 16, 4, 4, 2, d, True) for n in wgs])
        assert [p.forward[1:3] for p in got] == [(2, 1), (2, 1), (2, 2), (2, 2), (1, 2), (1, 2)], d
        assert all(p.forward.tiles == 1 for p in plans([(n * 16, n * 16, 4, 4, 2, d, False) for n in wgs]))


def test_calls_up_to_the_stated_sizes_fit_a_launch():
    """2^28 rows of queries and of keys and 2^20 heads times offsets: below 2^23 workgroups."""
    rng = random.Random(3)
    some = []
    for _ in range(20000):
        heads = rng.choice([1, 2, 3, 8, 16, 96, 128, 1024])
        kv = rng.choice([n for n in range(1, heads + 1) if heads % n == 0])
        most = lambda bits: 2**bits if rng.random() < 0.4 else int(2 ** rng.uniform(0, bits))  # noqa: E731
        seqs = max(1, most(20) // heads - 1)
        some.append((max(1, most(28) // heads), max(1, most(28) // kv), seqs, heads, kv, 8 * rng.randint(1, 16), rng.random() < 0.5))
    workgroups = [max(p.forward.count * p.splits, p.dq.count, p.keys.count * p.parts) * c[4] for c, p in zip(some, plans(some))]
    assert max(workgroups) < 2**23
    assert max(workgroups) > 2**21  # the largest of them are not far from it


def test_the_limit_of_a_launch():
    """Just below 2^23 workgroups a call is taken (and refused for its workspace), at it not."""
    lib = _lib.load()
    for tokens, code in (((1 << 26) - 64 * 4, 3), (1 << 26, 2)):
        a = _lib.PackedAttentionArgs(tokens_q=tokens, tokens_k=40, sequences=2, heads=8, kv_heads=8, head_dim=32, dtype=1, scale=1.0,
                                     q=0x1000, k=0x1000, v=0x1000, out=0x1000, q_starts=0x1000, k_starts=0x1000, lse=0x1000)
        b = _lib.PackedAttentionBwdArgs(fwd=a, dout=0x1000, dq=0x1000, dk=0x1000, dv=0x1000)
        for name in ("q_strides", "k_strides", "v_strides", "out_strides"):
            setattr(b.fwd, name, (32, 256))
        for name in ("dout_strides", "dq_strides", "dk_strides", "dv_strides"):
            setattr(b, name, (32, 256))
        assert lib.fjx_packed_attention_bwd(ctypes.byref(b), None) == code, lib.fjx_last_error()
        if code == 2:
            assert "up to 2^28" in lib.fjx_last_error().decode()
