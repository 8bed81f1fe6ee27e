"""Differential attention's gradients in rows where one key has nearly all the
weight: dq is then a small difference of large sums, wherever that key stands.

The bound of dq_t's elements, from the formula in float64 with P the weights,
D = sum P dP, V = sum P |dP - D|, T = sum P |dP - D| |k| and K = max |k|:
- half a step of the result (bf16 2^-8, float32 2^-24 of the value);
- the kernel sums P (dP - c) k around a centre c that the keys so far give, and
  corrects by (D - c) sum P k. A centre taken from keys of weight A is within
  V / A of D, and A is at least 1/16 for all but the first keys (for those the
  terms add up to less than 4 V): terms of at most T + 32 V K, each off by the
  second rounding of its two bf16 parts, 2^-8 2^-8 = 2^-16;
- the weights' own float32 error, 2^-13 of a weight (as in
  tests/test_gpu_diff_attention.py), on the terms and on D: T + V K;
- dP's float32 error e = 65 2^-24 sum |dO| |v|, of which the common part goes out
  with D: 2 e K sum P (1 - P)."""

from __future__ import annotations

import math

import pytest
import torch

from foldjax_amd import kernels
from tests.gpu_util import say

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0**-8, F32: 2.0**-24}
HEADS = 2


def weights(t):
    """P_t and lambda in float64; [..., H, nq, nk]."""
    q, k = t["q"].double(), t["k"].double()
    if t["mask"] is not None:
        k = torch.where(t["mask"][..., None, :, None], k, 0.0)
    s = t["scale"] * torch.matmul(q, k.transpose(-1, -2))
    if t["bias"] is not None:
        s = s + t["bias"].double().repeat_interleave(2, -3)
    if t["mask"] is not None:
        s = s.masked_fill(~t["mask"][..., None, None, :], -math.inf)
    p = torch.softmax(s, -1)
    lv = t["lam"].double()
    lam = (lv[0] * lv[1]).sum(-1).exp() - (lv[2] * lv[3]).sum(-1).exp() + t["init"]
    return p[..., 0::2, :, :], p[..., 1::2, :, :], lam[:, None, None], k


def check_dq(t, dq):
    p1, p2, lam, k = weights(t)
    v = t["v"].double()
    if t["mask"] is not None:
        v = torch.where(t["mask"][..., None, :, None], v, 0.0)
    do = t["dout"].double()
    dp = torch.matmul(do, v.transpose(-1, -2))
    e = 65 * 2.0**-24 * torch.matmul(do.abs(), v.abs().transpose(-1, -2)).amax(-1, keepdim=True)
    got = dq.double().cpu()
    assert torch.isfinite(got).all()
    for m, (p, by) in enumerate(((p1, torch.ones_like(lam)), (p2, -lam))):
        km = k[..., m::2, :, :]
        away = dp - (p * dp).sum(-1, keepdim=True)
        by = by * t["scale"]
        want = by * torch.matmul(p * away, km)
        T = torch.matmul(p * away.abs(), km.abs())
        V = (p * away.abs()).sum(-1, keepdim=True)
        K = km.abs().amax(-2, keepdim=True)
        G = (p * (1 - p)).sum(-1, keepdim=True)
        bound = by.abs() * ((2.0**-13 + 2.0**-16) * T + (2.0**-13 + 32 * 2.0**-16) * V * K + 2 * e * G * K)
        bound = bound + HALF[dq.dtype] * want.abs()
        over = (got[..., m::2, :, :] - want).abs() / bound
        assert over.max() <= 1.0, f"map {m + 1}: {float(over.max()):.1f} times the bound"


def sharp(lead, nq, nk, d, dtype, where, seed=0):
    """Query rows that point at one key each, with 1 - P from 1e-2 to 1e-7."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"v": r(*lead, HEADS, nk, 2 * d).to(dtype), "dout": r(*lead, HEADS, nq, 2 * d).to(dtype), "lam": 0.15 * r(4, HEADS, d),
         "init": 0.4, "scale": d**-0.5, "bias": None, "mask": None}
    k = r(*lead, 2 * HEADS, nk, d)
    t["k"] = (k / k.norm(dim=-1, keepdim=True) * math.sqrt(d)).to(dtype)
    lo = torch.empty(2 * HEADS, dtype=torch.long)
    lo[0::2], lo[1::2] = {"first": (0, 0), "middle": (nk // 2, nk // 2), "last": (nk - 16, nk - 16), "one each": (0, nk - 16),
                          "masked start": (nk - 100, nk - 40)}[where]
    at = lo[:, None] + torch.randint(0, 16, (*lead, 2 * HEADS, nq), generator=g)
    point = torch.gather(t["k"].float(), -2, at[..., None].expand(*at.shape, d))
    t["q"] = ((3.0 + 2.0 * torch.rand(*at.shape, 1, generator=g)) * math.sqrt(32 / d) * point).to(dtype)
    if where == "masked start":
        t["mask"] = (torch.arange(nk) >= 130).expand(*lead, nk).contiguous()
        t["k"].masked_fill_(~t["mask"][..., None, :, None], math.nan)
        t["v"].masked_fill_(~t["mask"][..., None, :, None], math.nan)
    return t


def run(t):
    """The outputs and gradients of the library for the tensors of ``t``."""
    c = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in t.items()}
    more = {"lambda_init": c["init"], "scale": c["scale"], "bias": c["bias"], "mask": c["mask"]}
    out, lse = kernels.diff_attention(c["q"], c["k"], c["v"], c["lam"], return_lse=True, **more)
    g = kernels.diff_attention_backward(c["dout"], c["q"], c["k"], c["v"], c["lam"], lse, **more)
    torch.cuda.synchronize()
    return out, dict(zip(("dq", "dk", "dv", "dbias", "dlam"), g))


# few rows (the waves of a workgroup share them) and many (each has its own)
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("where", ["first", "middle", "last", "one each", "masked start"])
@pytest.mark.parametrize("lead,nq,nk,d", [((2,), 20, 300, 32), ((2,), 5, 700, 64), ((64,), 9, 300, 32), ((64,), 4, 290, 64)],
                         ids=str)
def test_dq_where_one_key_has_the_weight(lead, nq, nk, d, where, dtype):
    say(f"sharp rows {lead} {nq} x {nk} d {d} {where} {dtype}")
    t = sharp(lead, nq, nk, d, dtype, where, seed=nk + d)
    _, got = run(t)
    check_dq(t, got["dq"])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lead,nq", [((2,), 20), ((64,), 9)], ids=str)
def test_dq_where_equal_keys_share_the_weight(lead, nq, dtype):
    """Copies of one key and value, in several blocks, with the weight between
    them: no key has the most of it, and dP is still the same for nearly all."""
    say(f"equal keys {lead} {dtype}")
    t = sharp(lead, nq, 400, 32, dtype, "last", seed=7)
    for name in ("k", "v"):
        t[name][..., 100:140, :] = t[name][..., 384:385, :]
        t[name][..., 360:, :] = t[name][..., 384:385, :]
    t["q"] = (t["q"].float() * 0 + 4.0 * t["k"][..., 384:385, :].float()).to(dtype)
    _, got = run(t)
    check_dq(t, got["dq"])
