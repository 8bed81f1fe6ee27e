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
