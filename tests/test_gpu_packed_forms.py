"""Every form in which packed attention is launched, against 64 bits value by value (the
bounds' derivation: tests/packed_oracle.py). What each call launches is asserted on the
CPU from the rules themselves, so that a rule that moves leaves no form untested."""

from __future__ import annotations

import pytest
import torch

from tests import packed_oracle as O
from tests.gpu_util import say
from tests.packed_plan import plans
from tests.test_gpu_packed_attention import BF16, FP32, compare, inputs, ints, run, starts

TAIL = 77  # rows behind the last sequence
KEYWISE, ROWS, SHARED, PAIRS, PAIRS_SHARED = (1, 4, 1), (4, 1, 1), (4, 2, 1), (4, 1, 2), (4, 2, 2)  # groups, ks, tiles

# lengths, heads, key/value heads, width, type; forms of the forward pass, dq, dk and dv; sorted by work
SHORT, CROPS, LONG, MANY = [37], [1003, 499, 546], [2000, 1500, 700], [330] * 20 + [1700]
CASES = [
    *((SHORT, 4, 4, d, t, KEYWISE, KEYWISE, KEYWISE, False) for d in (24, 64, 128) for t in (BF16, FP32)),
    *(([200, 37, 163] * 11, 16, 16, d, t, ROWS, ROWS, ROWS, False) for d in (24, 64, 128) for t in (BF16, FP32)),
    *((CROPS, 16, 16, d, BF16, SHARED, SHARED, SHARED, False) for d in (24, 64)),
    ([903, 446, 1], 16, 16, 128, BF16, SHARED, SHARED, SHARED, False),
    *((LONG, 16, 16, d, FP32, SHARED, SHARED, SHARED, True) for d in (24, 64, 128)),
    *((LONG, 16, 16, d, BF16, PAIRS_SHARED, PAIRS_SHARED, SHARED, True) for d in (24, 64, 128)),
    *((MANY, 16, 16, d, BF16, PAIRS_SHARED, PAIRS, PAIRS, False) for d in (24, 64)),
    (MANY, 16, 16, 128, BF16, PAIRS, PAIRS, SHARED, False),
    ([3400], 16, 4, 128, BF16, PAIRS_SHARED, PAIRS_SHARED, SHARED, False),
    ([2200, 2000], 32, 32, 64, BF16, PAIRS_SHARED, PAIRS, PAIRS, True),
    ([2200, 2000], 32, 32, 128, BF16, PAIRS, PAIRS, SHARED, True),
    *(([3300, 3100], 32, 32, d, BF16, PAIRS, PAIRS, PAIRS, True) for d in (24, 64)),
    *(([6400], 32, 32, d, BF16, PAIRS, PAIRS, PAIRS, False) for d in (24, 64)),
    ([4100, 0, 100], 32, 8, 64, BF16, PAIRS_SHARED, PAIRS, SHARED, True),
    ([4100, 0, 100], 32, 8, 128, BF16, PAIRS, PAIRS, SHARED, True),
]
NAMES = [f"{len(c[0])} sequences of up to {max(c[0])} heads {c[1]} on {c[2]} of {c[3]} {'fp32' if c[4] is FP32 else 'bf16'}" for c in CASES]


def test_what_is_launched():
    tokens = [sum(c[0]) + TAIL for c in CASES]
    found = plans([(n, n, len(c[0]), c[1], c[2], c[3], c[4] is BF16) for n, c in zip(tokens, CASES)])
    seen = set()
    for (lens, _, _, d, dtype, *forms, ordered), p, name in zip(CASES, found, NAMES):
        assert [p.forward[:3], p.dq[:3], p.keys[:3]] == forms, name
        assert p.forward.sorted == p.dq.sorted == p.keys.sorted == ordered, name
        width = 32 if d <= 32 else 64 if d <= 64 else 128
        seen |= {(k, dtype, width, form, ordered) for k, form in zip(("forward", "dq", "keys"), forms)}
    of = lambda *part: {s[3:] for s in seen if s[:3] == part}  # noqa: E731
    for width in (32, 64, 128):
        for kernel in ("forward", "dq"):
            assert {f for f, _ in of(kernel, BF16, width)} == {KEYWISE, ROWS, SHARED, PAIRS, PAIRS_SHARED}, (kernel, width)
            assert {f for f, _ in of(kernel, FP32, width)} == {KEYWISE, ROWS, SHARED}, (kernel, width)
        assert {f for f, _ in of("keys", FP32, width)} == {KEYWISE, ROWS, SHARED}, width
        assert {f for f, _ in of("keys", BF16, width)} == {KEYWISE, ROWS, SHARED} | ({PAIRS} if width <= 64 else set()), width
        # two tiles a wave, in the order of their work and not
        assert {(PAIRS_SHARED, True), (PAIRS_SHARED, False), (PAIRS, True), (PAIRS, False)} <= of("forward", BF16, width)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("case", CASES, ids=NAMES)
def test_forms(case, causal):
    lens, h, kv, d, dtype = case[:5]
    say(f"packed form {len(lens)} {max(lens)} {h} {kv} {d} {dtype} {causal}")
    q, k, v, dout = inputs(lens, h, kv, d, dtype, tail=TAIL, seed=len(lens) + d)
    more = {"scale": d**-0.5, "causal": causal}
    got = run(q, k, v, ints(starts(lens)), dout, **more)
    compare(got, O.attention(q, k, v, starts(lens), dout=dout, **more))
    assert all((t[:, sum(lens):] == 0).all() for t in got.values())
    torch.cuda.empty_cache()
