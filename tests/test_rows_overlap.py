"""Outputs that lie over inputs: the rule that tells (``fjx_overlap.hpp``, compiled for
the host, against sets of places), and the calls of the heads' norm that it refuses, at
the C ABI (fake pointers; every call here is refused before a launch)."""

from __future__ import annotations

import ctypes
import random
import subprocess
from pathlib import Path

import pytest

from foldjax_amd import _lib

ROOT = Path(__file__).resolve().parent.parent
PROGRAM = r"""
#include <cstdio>
#include "fjx_overlap.hpp"
int main() {
  long long v[16];
  for (;;) {
    for (int i = 0; i < 16; ++i)
      if (std::scanf("%lld", v + i) != 1) return 0;
    fjx::RowSet r[2];
    for (int i = 0; i < 2; ++i) {
      const long long* p = v + 8 * i;
      r[i] = {(uintptr_t)p[0], {p[1], p[2], p[3]}, {p[4], p[5], p[6]}, p[7]};
    }
    std::printf("%d %d\n", (int)fjx::rows_meet(r[0], r[1]), (int)fjx::rows_equal(r[0], r[1]));
  }
}
"""


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    at = tmp_path_factory.mktemp("overlap")
    (at / "p.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'foldjax_amd' / 'csrc'}", str(at / "p.cpp"), "-o", str(at / "p")],
                   check=True, capture_output=True, text=True)

    def ask(pairs):
        text = "\n".join(" ".join(map(str, [*a, *b])) for a, b in pairs)
        out = subprocess.run([str(at / "p")], input=text, check=True, capture_output=True, text=True).stdout
        return [tuple(int(x) for x in line.split()) for line in out.splitlines()]

    return ask


def places(row):
    at, ni, nh, nt, si, sh, st, width = row
    return {at + i * si + h * sh + t * st + w for i in range(ni) for h in range(nh) for t in range(nt) for w in range(width)}


def test_the_rule_against_sets_of_places(rule):
    rng = random.Random(7)
    pairs = []
    for _ in range(4000):
        width = rng.choice([1, 2, 4])
        strides = [rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 48]) for _ in range(3)]

        def row():
            s = strides if rng.random() < 0.7 else [rng.randrange(0, 30) for _ in range(3)]
            return [1000 + rng.randrange(0, 60), *(rng.randrange(0, 5) for _ in range(3)), *s, width]

        pairs.append((row(), row()))
    seen = set()
    for (a, b), (meet, same) in zip(pairs, rule(pairs)):
        want = bool(places(a) & places(b))
        assert meet == want, (a, b)
        if same and places(a):
            assert places(a) == places(b)
        seen.add((want, a[4:] == b[4:]))
    assert len(seen) == 4


def test_large_views(rule):
    """Views of one projection of 2^30 tokens, token by token and head by head, and views
    whose steps have nothing in common, which count as meeting where that is not soon seen."""
    tokens, d = 1 << 30, 256
    wide = 10 * d
    q, k, v = ([1 << 20, 1, n, tokens, 0, d, wide, d] for n in (6, 2, 2))
    k[0] += 6 * d
    v[0] += 8 * d
    first = [*q[:2], 2, *q[3:]]
    last = [q[0] + 5 * d, *k[1:]]
    shifted = [q[0] + wide, *q[1:]]
    apart = [q[0] + (tokens * wide), *q[1:]]
    by_head = [[1 << 20, 3, n, 4096, 10 * 4096 * d, 4096 * d, d, d] for n in (8, 2)]
    by_head[1][0] += 8 * 4096 * d
    odd = [1 << 20, 100, 100, 100, 7 * 16, 1009 * 16, 100003 * 16, 16], [(1 << 20) + 16, 90, 90, 90, 11 * 16, 1013 * 16, 100019 * 16, 16]
    got = rule([(q, k), (k, v), (q, v), (q, first), (q, last), (q, shifted), (q, apart), (q, q), by_head, odd])
    assert [m for m, _ in got] == [0, 0, 0, 1, 1, 1, 0, 1, 0, 1]
    assert [s for _, s in got] == [0, 0, 0, 0, 0, 0, 0, 1, 0, 0]


def rotary(**more):
    """2 items of 8 tokens, 4 query heads and 2 of keys of 32 channels in bf16 (64 bytes),
    each buffer 16 KiB from the next."""
    a = _lib.HeadNormRotaryArgs(items=2, heads=4, kv_heads=2, tokens=8, head_dim=32, dtype=1, axes=1, sections=(16, 0, 0, 0), eps=1e-6,
                                q=0x10000, k=0x14000, q_weight=0x20000, k_weight=0x20000, positions=0x21000, frequencies=0x22000,
                                q_out=0x18000, k_out=0x1C000)
    for name in ("q_strides", "q_out_strides"):
        setattr(a, name, (1024, 32, 128))
    for name in ("k_strides", "k_out_strides"):
        setattr(a, name, (1024, 32, 128))
    for n, v in more.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("more", [
    {"k": 0x10000, "k_out": 0x10000},                    # keys that are the queries' first heads, in place
    {"k": 0x10000 + 2 * 64, "k_out": 0x10000 + 2 * 64},  # their last heads
    {"k_out": 0x10000 + 3 * 64},                         # one head of the queries
    {"q_out": 0x14000},                                  # the keys' place
    {"q_out": 0x10000 + 256},                            # its own input, a token on
    {"q_out": 0x10000, "q_out_strides": (1024, 256, 32)},  # the same buffer, turned
    {"k_out": 0x18000 + 64},                             # both outputs
    {"k_out": 0x18000 + 15 * 256},                       # one token of both
], ids=str)
def test_outputs_over_inputs_are_refused(more):
    lib = _lib.load()
    a = rotary(**more)
    assert lib.fjx_head_norm_rotary_fwd(ctypes.byref(a), None) == 1
    assert "two buffers" in lib.fjx_last_error().decode()


@pytest.mark.parametrize("dq,dk,more", [
    (0x30000, 0x30000 + 64, {}), (0x30000, 0x10000, {}), (0x1C000, 0x34000, {}), (0x18000 + 256, 0x34000, {}),
    (0x14000, 0x34000, {"q_weight": None}),
], ids=str)
def test_gradients_over_inputs_are_refused(dq, dk, more):
    lib = _lib.load()
    size = lib.fjx_head_norm_rotary_bwd_workspace_size(2, 4, 2, 8, 32)
    b = _lib.HeadNormRotaryBwdArgs(rotary(**more), dq, dk, (1024, 32, 128), (1024, 32, 128), 0x40000, 0x41000, 0x50000, size)
    assert lib.fjx_head_norm_rotary_bwd(ctypes.byref(b), None) == 1
    assert "two buffers" in lib.fjx_last_error().decode()


def packed(**more):
    """40 tokens in 2 sequences, 4 query heads on 2, 32 channels in bf16, token by token."""
    a = _lib.PackedAttentionArgs(tokens_q=40, tokens_k=40, sequences=2, heads=4, kv_heads=2, head_dim=32, dtype=1, scale=1.0,
                                 q=0x10000, k=0x14000, v=0x18000, out=0x1C000, q_starts=0x20000, k_starts=0x20000)
    for name in ("q_strides", "k_strides", "v_strides", "out_strides", "rest_strides"):
        setattr(a, name, (32, 128))
    for n, v in more.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("more", [
    {"out": 0x10000}, {"out": 0x10000 + 256}, {"out": 0x10000 - 39 * 256},  # the queries, a token on, their first token
    {"out": 0x10000, "out_strides": (40 * 32, 32)},                        # turned
    {"out": 0x14000 - 2 * 64}, {"out": 0x18000 + 39 * 256},                # a head of keys, the last token's values
    {"k": 0x10000 + 4 * 64, "k_strides": (32, 256), "q_strides": (32, 256), "out": 0x10000 + 3 * 64, "out_strides": (32, 256)},
], ids=str)
def test_attention_over_its_inputs_is_refused(more):
    lib = _lib.load()
    assert lib.fjx_packed_attention_fwd(ctypes.byref(packed(**more)), None) == 1
    assert "out must not overlap" in lib.fjx_last_error().decode()
