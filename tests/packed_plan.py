"""The rules by which a call of packed attention is cut (``fjx_packed_plan.hpp``),
compiled for the host: what the library launches for given counts."""

from __future__ import annotations

import functools
import subprocess
import tempfile
from pathlib import Path
from typing import NamedTuple

ROOT = Path(__file__).resolve().parent.parent
PROGRAM = r"""
#include <cstdio>
#include "fjx_packed_plan.hpp"
using namespace fjx;
int main() {
  long long tq, tk, seqs, heads, kvh, d;
  int bf;
  while (std::scanf("%lld %lld %lld %lld %lld %lld %d", &tq, &tk, &seqs, &heads, &kvh, &d, &bf) == 7) {
    const PackedPlan f = packed_fwd_plan(tq, tk, seqs, heads, kvh, d, bf), b = packed_bwd_plan(tq, tk, seqs, heads, kvh, d, bf);
    auto form = [](const PackedForm& x, size_t order) {
      std::printf("%d %d %d %d %d ", x.groups, x.ks, x.tiles, x.count, order != 0);
    };
    form(f.rows, f.rows_order);
    form(b.rows, b.rows_order);
    form(b.keys, b.keys_order);
    std::printf("%d %d %zu %zu\n", f.splits, b.splits, f.part_o + f.part_ml + f.rows_order,
                2 * b.part_o + b.part_ml + b.rows_order + b.keys_order);
  }
}
"""


class Form(NamedTuple):
    groups: int  # of waves with rows (keys) of their own
    ks: int      # waves that share a group's rows and split the keys
    tiles: int   # 16-row tiles of a wave
    count: int   # tiles for one key/value head
    sorted: bool


class Plan(NamedTuple):
    forward: Form
    dq: Form
    keys: Form
    splits: int  # of the keys (forward)
    parts: int   # of the heads that share keys, at most (dk and dv)
    forward_bytes: int
    backward_bytes: int


@functools.cache
def _program():
    at = Path(tempfile.mkdtemp(prefix="packed_plan_"))
    (at / "p.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'foldjax_amd' / 'csrc'}", str(at / "p.cpp"), "-o", str(at / "p")],
                   check=True, capture_output=True, text=True)
    return str(at / "p")


def plans(calls):
    """A Plan for each (tokens_q, tokens_k, sequences, heads, kv_heads, head_dim, bf16)."""
    text = "\n".join(" ".join(str(int(x)) for x in c) for c in calls)
    out = subprocess.run([_program()], input=text, check=True, capture_output=True, text=True).stdout
    found = []
    for line in out.splitlines():
        v = [int(x) for x in line.split()]
        forms = [Form(*v[5 * i:5 * i + 4], bool(v[5 * i + 4])) for i in range(3)]
        found.append(Plan(*forms, *v[15:]))
    return found
