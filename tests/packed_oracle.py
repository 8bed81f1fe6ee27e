"""Packed attention in 64 bits, with bounds of what its kernels' roundings can do to
each value.

u: half a step of the tensors' type (bf16 2^-8, float32 2^-24), w: of float32.
A weight p enters the products rounded to the tensors' type, p (1 + e), |e| <= u, after
it was computed with a relative error of at most ``e_w``: the score's float32 sum (d + 2
products, of scale sum |q||k| in all), its fma (half a step of the row's maximum),
log2 of the sum and v_exp_f32 (together below 8 w of the exponent's size plus 4 w).
Sums of n terms in float32 are off by at most n w of the terms' absolute sum.

  out = sum p v / sum p, the same p in both:   2 (u + e_w) sum p |v|, and its own u |out|
  D = sum over d of dO out, of weights off by (u + e_w) and an output kept to 2^-16 (bf16;
      float32 2^-24):  2 (u + e_w) sum_j p |dP - D| + (2^-16 or w + d w) sum |dO||out|
  dP: (d + 2) w sum |dO||v|
  dS = p (dP - D):  p (err D + err dP) + (u + 2 e_w) |dS|
  dq, dk: scale times dS's errors through |k| or |q|, and their own u
  dv: (u + 2 e_w) sum p |dO|, and its own u
"""

from __future__ import annotations

import torch


def spans(q_starts, k_starts, k_lengths):
    for s in range(len(q_starts) - 1):
        nk = k_starts[s + 1] - k_starts[s] if k_lengths is None else k_lengths[s]
        yield q_starts[s], q_starts[s + 1] - q_starts[s], k_starts[s], nk


def attention(q, k, v, q_starts, *, scale, causal=False, k_starts=None, k_lengths=None, dout=None):
    """{name: (value, bound)} in float64 for out and, with dout, dq, dk and dv."""
    f64 = torch.float64
    u, w = torch.finfo(q.dtype).eps / 2, 2.0**-24
    kept = 2.0**-16 if q.dtype is torch.bfloat16 else w
    (h, _, d), kvh = q.shape, k.shape[0]
    g = h // kvh
    zero = lambda t: torch.zeros(t.shape, dtype=f64, device=t.device)  # noqa: E731
    val = {"out": zero(q), "dq": zero(q), "dk": zero(k), "dv": zero(v)}
    err = {n: zero(t) for n, t in val.items()}
    for q0, nq, k0, nk in spans(q_starts, q_starts if k_starts is None else k_starts, k_lengths):
        if not nq or not nk:
            continue
        i = torch.arange(nq, device=q.device)[:, None] + nk - nq
        part = torch.arange(nk, device=q.device)[None] <= (i if causal else nk)
        for head in range(h):
            at = head // g, slice(k0, k0 + nk)
            rows = head, slice(q0, q0 + nq)
            qs, ks, vs = q[rows].to(f64), k[at].to(f64), v[at].to(f64)
            s = torch.where(part, scale * (qs @ ks.T), -torch.inf)
            top = s.amax(-1, keepdim=True)
            top = torch.where(top == -torch.inf, 0.0, top)
            e = (s - top).exp()
            p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
            size = scale * (qs.abs() @ ks.abs().T)
            e_w = ((d + 2) * w * size + 12 * w * (top.abs() + (s - top).abs().clamp_max(200.0)) + (nk + 12) * w)
            e_w = torch.where(part, e_w, 0.0)
            o = p @ vs
            val["out"][rows] = o
            err["out"][rows] = 2 * ((p * (u + e_w)) @ vs.abs()) + (u + nk * w) * o.abs()
            if dout is None:
                continue
            do = dout[rows].to(f64)
            dp = do @ vs.T
            D = (do * o).sum(-1, keepdim=True)
            ds = p * (dp - D)
            err_d = 2 * (p * (u + e_w) * (dp - D).abs()).sum(-1, keepdim=True) + (kept + (d + 2) * w) * (
                do.abs() * o.abs()).sum(-1, keepdim=True)
            err_ds = p * (err_d + (d + 2) * w * (do.abs() @ vs.abs().T)) + (u + 2 * e_w) * ds.abs()
            val["dq"][rows] = scale * (ds @ ks)
            val["dk"][at] += scale * (ds.T @ qs)
            val["dv"][at] += p.T @ do
            err["dq"][rows] = scale * ((err_ds + nk * w * ds.abs()) @ ks.abs())
            err["dk"][at] += scale * ((err_ds + nq * g * w * ds.abs()).T @ qs.abs())
            err["dv"][at] += (p * (u + 2 * e_w + nq * g * w)).T @ do.abs()
    for n in ("dq", "dk", "dv"):
        err[n] += u * val[n].abs()
    return {n: (val[n], 1.05 * err[n] + 1e-30) for n in val if dout is not None or n == "out"}


def check(got, value_and_bound, name):
    value, bound = value_and_bound
    got = got.double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - value).abs() / bound
    assert over.max() <= 1.0, f"{name}: {over.max().item():.3g} of its bound at {over.argmax().item()}"
