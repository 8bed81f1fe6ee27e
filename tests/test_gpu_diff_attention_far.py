"""Differential attention under biases far from zero, as masks are written that
add a large number to every score of a row: the softmax does not see what a row's
scores have in common, however large it is. The bounds are those of
tests/test_gpu_diff_attention.py: rows that are all far have queries of zeros, so
that their scores are the bias alone, which every float32 step keeps."""

from __future__ import annotations

import pytest
import torch

from tests.gpu_util import say
from tests.test_gpu_diff_attention import call, check, grads, make, on_gpu, reference

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
FAR = [-300.0, -1e5, -1e9, -1e10, -1e20, -1e30, 1e9, 1e20]
# few rows (waves that share them) and many
FORMS = [((2,), 24, 200, 32), ((1,), 7, 300, 64), ((64,), 8, 70, 32), ((64,), 8, 130, 64)]


def far(lead, nq, nk, d, dtype, value):
    t = make(lead, 2, 2, nq, nk, d, dtype, bias="plane", mask="none", seed=nk)
    b = t["bias"]
    b[..., 0, :] = value  # a row with nothing near
    b[..., 1, : nk // 2] = value  # and with two distances
    b[..., 1, nk // 2 :] = 2 * value
    b[..., 2, : nk - 1] = value  # one key and the rest far from it
    b[..., 3, 1:] = value
    # the rows whose weight is among far keys: at 1e9 a float32's step is 64, more
    # than their scores differ by
    t["q"][..., : 4 if value > 0 else 2, :] = 0.0
    return t


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("value", FAR)
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_rows_far_from_zero(form, value, dtype):
    say(f"far bias {form} {value} {dtype}")
    t = far(*form, dtype, value)
    want, terms = reference(t)
    check("out", call(on_gpu(t)), want["out"], terms["out"], dtype)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("value", [-1e9, -1e10, -1e30])
def test_one_token_against_far_keys(value, dtype):
    """Keys split over workgroups: whole splits are far, or all of them."""
    say(f"far splits {value} {dtype}")
    t = make((2,), 4, 2, 1, 3000, 64, dtype, bias="plane", mask="none", seed=1)
    t["bias"][0, :, :, 100:] = value
    t["bias"][1, :2] = value
    t["q"][1] = 0.0
    want, terms = reference(t)
    check("out", call(on_gpu(t)), want["out"], terms["out"], dtype)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("value", FAR)
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_gradients_of_rows_far_from_zero(form, value, dtype):
    """The weights of such a row add up to one in the backward pass as well."""
    say(f"far bias, gradients {form} {value} {dtype}")
    t = far(*form, dtype, value)
    t["bias"][..., 4, :] = t["bias"][..., 5, :] - 300.0  # distances at which scores still count
    want, terms = reference(t, backward=True)
    g = on_gpu(t)
    got = grads(g, call(g, return_lse=True)[1])
    for name in ("dq", "dk", "dv", "dlam", "dbias"):
        check(name, got[name], want[name], terms[name], dtype)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("value", [-1e5, -1e9, -1e30])
@pytest.mark.parametrize("rows", [3, 20, 40])
def test_shared_bias_far_from_zero(rows, value, dtype):
    """A plane that the rows of a pair tensor share, whole queries of it far."""
    say(f"far shared bias {rows} {value} {dtype}")
    t = make((2, rows), 2, 2, 70, 70, 32, dtype, bias="shared", mask="tail", seed=4)
    t["bias"][..., 60:, :] = value
    t["q"][..., 60:, :] = 0.0
    want, terms = reference(t, backward=True)
    g = on_gpu(t)
    out, lse = call(g, return_lse=True)
    check("out", out, want["out"], terms["out"], dtype)
    got = grads(g, lse)
    for name in ("dq", "dk", "dv", "dlam", "dbias"):
        check(name, got[name], want[name], terms[name], dtype)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("value", [-1e5, -1e10])
@pytest.mark.parametrize("lead,heads,kv", [((48,), 2, 2), ((24,), 6, 3), ((2,), 8, 2), ((70,), 4, 2)], ids=str)
def test_gradients_of_far_rows_in_several_blocks(lead, heads, kv, value, dtype):
    """Query blocks with far rows and without, of heads that share keys, in the
    forms of every number of workgroups."""
    say(f"far blocks {lead} {heads} {kv} {value} {dtype}")
    t = make(lead, heads, kv, 150, 90, 32, dtype, bias="plane", mask="none", seed=heads)
    for rows in (slice(20, 22), slice(140, 150)):  # blocks 0 and 2 of 64, 0 and 1 of 128
        t["bias"][..., heads - 1, rows, :] = value
        t["q"][..., -2:, rows, :] = 0.0
    want, terms = reference(t, backward=True)
    g = on_gpu(t)
    out, lse = call(g, return_lse=True)
    check("out", out, want["out"], terms["out"], dtype)
    got = grads(g, lse)
    for name in ("dq", "dk", "dv", "dlam", "dbias"):
        check(name, got[name], want[name], terms[name], dtype)
