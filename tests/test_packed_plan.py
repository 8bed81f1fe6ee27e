"""How calls of packed attention are cut (tests/packed_plan.py), on the CPU."""

from __future__ import annotations

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
