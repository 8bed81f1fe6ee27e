"""The digits of packed attention's statistics and of dq.

The statistics are the row's maximum M and log2 of the sum of its unrounded weights: with
the sum of the rounded ones every weight of a row's gradients would be off by what their
rounding is of it, up to 2^-8 in bf16. dq takes dS in two bf16 parts. The bounds here leave
room for neither, as an emulation on the CPU shows.

w = 2^-24, u: half a step of the tensors' type, e_w: a weight's float32 error
(tests/packed_oracle.py). What the forward call gives, out and ``rest``, is taken as it is:
D is rowsum(dO (out + rest)), so that the rounding of the weights that were applied is no
error of the gradients' own.
  M + log2 l: e_w of the sum and half a step of each, in log2 units
  D: (d + 2) w sum |dO||out|;  dP - D, sums that begin at -D: (d + 3) w (sum |dO||v| + |D|)
  dS = P (dP - D): P times those, and (parts + 2 e_w + 2 w) |dS|, where two bf16 parts leave
      2^-8 2^-8 = 2^-16 and float32 w
  dq: scale times dS's errors and (2 nk + 8) w |dS| through |k|, w |dq|, and its own u |dq|
"""

from __future__ import annotations

import math

import pytest
import torch

from tests.gpu_util import say
from tests.packed_oracle import spans

F64, BF, FP = torch.float64, torch.bfloat16, torch.float32
W = 2.0**-24


def starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def reference(q, k, v, dout, kept, q_starts, *, scale, causal, k_starts=None, k_lengths=None):
    """(log2 of the rows' sums, its bound, dq, its bound) in 64 bits; kept: out + rest."""
    u = torch.finfo(q.dtype).eps / 2
    parts = 2.0**-16 if q.dtype is BF else W
    (h, tq, d), g = q.shape, q.shape[0] // k.shape[0]
    logs, logs_err = (torch.zeros(h, tq, dtype=F64, device=q.device) for _ in range(2))
    dq, err = (torch.zeros(q.shape, dtype=F64, device=q.device) for _ in range(2))
    for q0, nq, k0, nk in spans(q_starts, q_starts if k_starts is None else k_starts, k_lengths):
        if not nq or not nk:
            logs[:, q0:q0 + nq] = math.inf
            continue
        i = torch.arange(nq, device=q.device)[:, None] + nk - nq
        seen = torch.arange(nk, device=q.device)[None] <= (i if causal else nk)
        for head in range(h):
            rows, at = (head, slice(q0, q0 + nq)), (head // g, slice(k0, k0 + nk))
            qs, ks, vs, do, o = q[rows].to(F64), k[at].to(F64), v[at].to(F64), dout[rows].to(F64), kept[rows].to(F64)
            s = torch.where(seen, scale * (qs @ ks.T), -math.inf)
            log = s.logsumexp(-1, keepdim=True)
            there = log > -math.inf
            p = torch.where(there, (s - log).exp(), 0.0)
            top = torch.where(there, s.amax(-1, keepdim=True), 0.0)
            size = scale * (qs.abs() @ ks.abs().T)
            e_w = (d + 2) * W * size + 12 * W * (top.abs() + (s - top).abs().nan_to_num(200.0, 200.0).clamp_max(200.0)) + (nk + 12) * W
            e_w = torch.where(seen, e_w, 0.0)
            logs[rows] = torch.where(there, log / math.log(2.0), math.inf)[:, 0]
            logs_err[rows] = (1.5 * e_w.amax(-1) + 4 * W * (logs[rows].abs().nan_to_num(0.0, 0.0) + 16)) * 1.05
            D = (do * o).sum(-1, keepdim=True)
            ds = p * (do @ vs.T - D)
            terms = (d + 2) * W * (do.abs() * o.abs()).sum(-1, keepdim=True) + (d + 3) * W * (do.abs() @ vs.abs().T + D.abs())
            err_ds = p * terms + (parts + 2 * e_w + 2 * W + (2 * nk + 8) * W) * ds.abs()
            dq[rows] = scale * (ds @ ks)
            err[rows] = scale * (err_ds @ ks.abs())
    return logs, logs_err, dq, 1.05 * (err + (u + W) * dq.abs()) + 1e-30


def over(got, value, bound):
    """By how much the worst value is past its bound, 1 being just within."""
    got = got.double()
    same = (got == value) | (got.isinf() & value.isinf())
    return torch.where(same, 0.0, (got - value).abs() / bound).max().item()


def rounded(x, parts):
    high = x.to(BF).double()
    return high if parts == 1 else high + (x - high).to(BF).double()


def emulated(q, k, v, dout, *, scale, parts=2, sums="unrounded"):
    """One sequence in bf16: (out + rest, log2 of the rows' sums, dq), all in float64 but for
    the forward weights' rounding, dS in ``parts`` and the sum of weights that are not
    ``unrounded``. Maxima as the kernels keep them, up to 8 of log2 behind the row's own."""
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    s = scale * torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.log(2.0)
    top = s.amax(-1, keepdim=True)
    first = s[..., :16].amax(-1, keepdim=True)
    m = torch.where(top > first + 8, top, first)
    p = (s - m).exp2()
    pr = rounded(p, 1)
    kept = rounded(torch.matmul(pr, v) / pr.sum(-1, keepdim=True), 2)
    logs = m + (p if sums == "unrounded" else pr).sum(-1, keepdim=True).log2()
    ds = (s - logs).exp2() * (torch.matmul(dout, v.transpose(-1, -2).contiguous()) - (dout * kept).sum(-1, keepdim=True))
    return kept, logs[..., 0], (scale * torch.matmul(rounded(ds, parts), k)).to(BF)


def tensors(lens, h, kv, d, dtype, *, seed, common=0.0, device="cpu", by=1.3, keys=None):
    """[heads, tokens, width] of a bf16 or float32 sublayer, token by token; common: of all keys."""
    g = torch.Generator(device=device).manual_seed(seed)
    n, nk = sum(lens), sum(lens if keys is None else keys)
    make = lambda t, c, f: f * torch.randn(t, c, d, generator=g, device=device)  # noqa: E731
    q, k, v, dout = make(n, h, by), make(nk, kv, by), make(nk, kv, 1.0), make(n, h, 1.0)
    k += common * torch.randn(1, kv, d, generator=g, device=device)
    return tuple(t.to(dtype).transpose(0, 1) for t in (q, k, v, dout))


@pytest.mark.parametrize("n,d,common", [(60, 24, 0.0), (130, 64, 0.0), (257, 32, 4.0)])
def test_the_bounds_tell_what_loses_digits(n, d, common):
    q, k, v, dout = tensors([n], 2, 2, d, BF, seed=n, common=common)
    more = {"scale": d**-0.5}
    kept, logs, dq = emulated(q, k, v, dout, **more)
    want = reference(q, k, v, dout, kept, [0, n], causal=False, **more)
    assert over(logs, *want[:2]) <= 1 and over(dq, *want[2:]) <= 1
    assert over(emulated(q, k, v, dout, parts=1, **more)[2], *want[2:]) > 3
    _, logs, dq = emulated(q, k, v, dout, sums="rounded", **more)
    assert over(logs, *want[:2]) > 10 and over(dq, *want[2:]) > 1


def compare(q, k, v, dout, st, device_starts, more, ints):
    from foldjax_amd import kernels

    on = {n: ints(m) if isinstance(m, list) else m for n, m in more.items()}
    out, lse, rest = kernels.packed_attention(q, k, v, device_starts, return_lse=True, **on)
    assert torch.equal(out, kernels.packed_attention(q, k, v, device_starts, **on))  # asked for or not
    dq = kernels.packed_attention_backward(dout, q, k, v, out, lse, rest, device_starts, **on)[0]
    kept = out.double() + (0 if rest is None else rest.double())
    logs, logs_err, want, err = reference(q, k, v, dout, kept, st, **more)
    worst = over(lse.double().sum(-1), logs, logs_err), over(dq, want, err)
    assert max(worst) <= 1, f"statistics and dq: {worst[0]:.3g} and {worst[1]:.3g} of their bounds"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("lens,h,kv,d,common", [
    ([37], 4, 4, 24, 0.0), ([70, 0, 9, 131], 4, 2, 40, 3.0), ([60] * 80, 16, 16, 32, 0.0), ([1003, 499, 546], 16, 16, 24, 0.0),
    ([1500, 3, 701], 16, 4, 64, 4.0), ([2000, 1500, 700], 16, 16, 64, 0.0), ([330] * 20 + [1700], 16, 16, 24, 0.0),
    ([1500, 900], 8, 2, 128, 2.0), ([2200, 2000], 16, 16, 128, 0.0),
], ids=str)
def test_statistics_and_dq(lens, h, kv, d, common, causal, dtype):
    say(f"packed digits {len(lens)} {max(lens)} {h} {kv} {d} {common} {causal} {dtype}")
    q, k, v, dout = tensors(lens, h, kv, d, dtype, seed=d + len(lens), common=common, device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    compare(q, k, v, dout, starts(lens), ints(starts(lens)), {"scale": d**-0.5, "causal": causal}, ints)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("nq,h,kv,d", [(1, 8, 2, 128), (2, 4, 4, 32), (3, 16, 1, 64)])
def test_statistics_of_caches_over_workgroups(nq, h, kv, d, dtype):
    """Keys over several workgroups, whose sums a second kernel joins."""
    say(f"packed digits caches {nq} {h} {kv} {d} {dtype}")
    caches, lens = [5000] * 3, [5000, 0, 3001]
    q, k, v, dout = tensors([nq] * 3, h, kv, d, dtype, seed=nq, device="cuda", keys=caches)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    st = starts([nq] * 3)
    compare(q, k, v, dout, st, ints(st), {"scale": d**-0.5, "causal": True, "k_starts": starts(caches), "k_lengths": lens}, ints)
