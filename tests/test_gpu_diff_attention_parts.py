"""The bf16 gradients' own accuracy: dS and the maps' difference go into their
products as two bf16 parts, so that dq, dk and dv are off by their own rounding and
by little else. Bounds, per element: half a step of the result, 2^-8; the parts'
second rounding, 2^-8 2^-8 = 2^-16 of a term (of two operands at most: 2^-15); the
weights' float32 error, 2^-13 of a term (see tests/test_gpu_diff_attention.py). In
the norm: roundings spread evenly over half a step of at most 2^-8 of the value are
2^-8 / sqrt(3) of it in the root mean square (less where values are not all just
above a power of two); 1e-7 of the terms for float32. One part alone is
beyond them, as an emulation on the CPU shows."""

from __future__ import annotations

import math

import pytest
import torch

from tests.gpu_util import say
from tests.test_gpu_diff_attention import BF, BIAS_MASK, MANY, SHAPES, SLACK, call, grads, make, on_gpu, reference

EACH = SLACK + 2.0**-15
NORM = 2.0**-8 / math.sqrt(3.0)


def faults(got, want, terms):
    got = got.double().cpu()
    over = ((got - want).abs() - (2.0**-8 * want.abs() + EACH * terms)).max()
    err, most = float((got - want).norm()), NORM * float(want.norm()) + 1e-7 * float(terms.norm())
    found = [] if over <= 1e-30 else [f"{float(over):.2e} past the bound"]
    return found + ([] if err <= most else [f"{err / max(float(want.norm()), 1e-30):.2e} in norm"])


def rounded(x, parts):
    high = x.to(BF).double()
    return high if parts == 1 else high + (x - high).to(BF).double()


def emulated(t, parts):
    """dq, dk and dv with dS and the maps' difference in `parts` bf16 parts, all else
    in float64; no mask, heads of their own."""
    q, k, v, do, lv = (t[n].double() for n in ("q", "k", "v", "dout", "lam"))
    lam = ((lv[0] * lv[1]).sum(-1).exp() - (lv[2] * lv[3]).sum(-1).exp() + t["init"])[:, None, None]
    s = t["scale"] * torch.matmul(q, k.transpose(-1, -2)) + t["bias"].double().repeat_interleave(2, -3)
    p = torch.softmax(s, -1).unflatten(-3, (-1, 2))
    dp = torch.matmul(do, v.transpose(-1, -2))
    comb = p[..., 0, :, :] - lam * p[..., 1, :, :]
    ds = []
    for m, by in ((0, 1.0), (1, -lam)):
        pm = p[..., m, :, :]
        ds.append(rounded(by * pm * (dp - (pm * dp).sum(-1, keepdim=True)), parts))
    ds = torch.stack(ds, -3).flatten(-4, -3)
    out = {"dq": t["scale"] * torch.matmul(ds, k), "dk": t["scale"] * torch.matmul(ds.transpose(-1, -2), q),
           "dv": torch.matmul(rounded(comb, parts).transpose(-1, -2), do)}
    return {n: x.to(BF) for n, x in out.items()}


@pytest.mark.parametrize("shape", [((2,), 2, 2, 65, 63, 32), ((3,), 4, 4, 100, 257, 32), ((1,), 4, 4, 130, 129, 64)], ids=str)
def test_the_bounds_tell_two_parts_from_one(shape):
    t = make(*shape, BF, bias="plane", seed=sum(shape[1:]))
    want, terms = reference(t, backward=True)
    two, one = emulated(t, 2), emulated(t, 1)
    for name in two:
        assert not faults(two[name], want[name], terms[name]), name
        assert faults(one[name], want[name], terms[name]), name


@pytest.mark.gpu
@pytest.mark.parametrize("bias,mask", BIAS_MASK)
@pytest.mark.parametrize("shape", SHAPES + MANY, ids=str)
def test_gradients_are_off_by_their_own_rounding(shape, bias, mask):
    say(f"two parts {shape} bias {bias} mask {mask}")
    t = make(*shape, BF, bias=bias, mask=mask, seed=sum(shape[1:]))
    want, terms = reference(t, backward=True)
    g = on_gpu(t)
    got = grads(g, call(g, return_lse=True)[1])
    for name in ("dq", "dk", "dv"):
        found = faults(got[name], want[name], terms[name])
        assert not found, (name, found)
