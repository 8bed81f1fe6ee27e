"""The heads' norm and rotation in 64 bits, by complex numbers and differentiation,
with bounds of what the kernels' roundings can do to each value.

u: half a step of the tensors' type, w = 2^-24. A row's sums of d terms in float32 are
off by at most d w of the terms' absolute sum, v_rsq_f32 by 2 w; cosines and sines by
4 w (float32's of an angle reduced in 64 bits and rounded, below pi w, and their own).
  y: (d + 16) w (|n_a| + |n_b|), and its own u |y|
  dx = rstd (t - h mean(t h)): (4 d + 40) w rstd (|t| + |h| mean |t h|) over the turned
      gradient's |dy_a| + |dy_b|, and its own u |dx|
  dw: (rows + 2 d + 40) w sum |dn h|
"""

from __future__ import annotations

import torch


def _order(d, pairs, interleaved, device):
    """Channels with the members of a pair side by side."""
    o = torch.arange(2 * pairs, device=device)
    if not interleaved:
        o = o.view(2, -1).T.reshape(-1)
    return torch.cat([o, torch.arange(2 * pairs, d, device=device)])


def turn(x, positions, frequencies, sections, interleaved, back=False):
    d, pairs = x.shape[-1], frequencies.shape[0]
    lead = x.shape[:-3]
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(x.device)
    p = positions.double()
    if positions.dim() == 2:
        p = p.view(p.shape[0], *[1] * len(lead), p.shape[1]).expand(-1, *lead, -1)
    angle = p[axis].movedim(0, -1) * frequencies  # [..., T, pairs]
    z = torch.polar(torch.ones_like(angle), -angle if back else angle).unsqueeze(-3)
    order = _order(d, pairs, interleaved, x.device)
    x = x[..., order]
    t = torch.view_as_real(torch.view_as_complex(x[..., :2 * pairs].unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
    return torch.cat([t, x[..., 2 * pairs:]], -1)[..., torch.argsort(order)]


def both(x, frequencies, interleaved):
    """|a| + |b| for the members of a pair, |x| for the others."""
    order = _order(x.shape[-1], frequencies.shape[0], interleaved, x.device)
    y = x.abs()[..., order]
    n = 2 * frequencies.shape[0]
    y = torch.cat([y[..., :n].unflatten(-1, (-1, 2)).sum(-1, keepdim=True).expand(*y.shape[:-1], n // 2, 2).flatten(-2), y[..., n:]], -1)
    return y[..., torch.argsort(order)]


def norm_rotary(x, weight, positions, frequencies, sections, interleaved=False, eps=1e-6, dy=None):
    """(y, bound), and with dy also (dx, bound) and (dweight, bound) or None."""
    u, w, d = torch.finfo(x.dtype).eps / 2, 2.0**-24, x.shape[-1]
    xf = x.double()
    rstd = (xf.square().mean(-1, keepdim=True) + eps).rsqrt() if weight is not None else torch.ones_like(xf[..., :1])
    h = xf * rstd
    wf = weight.double() if weight is not None else torch.ones(d, dtype=torch.float64, device=x.device)
    n = h * wf
    args = positions, frequencies, sections, interleaved
    y = turn(n, *args)
    out = [(y, 1.05 * ((d + 16) * w * both(n, frequencies, interleaved) + u * y.abs()) + 1e-30)]
    if dy is None:
        return out
    dn = turn(dy.double(), *args, back=True)
    size = both(dy.double(), frequencies, interleaved)
    if weight is None:
        return [*out, (dn, 1.05 * (16 * w * size + u * dn.abs()) + 1e-30), None]
    t, ts = dn * wf, size * wf.abs()
    dx = rstd * (t - h * (t * h).mean(-1, keepdim=True))
    bound = (4 * d + 40) * w * rstd * (ts + h.abs() * (ts * h.abs()).mean(-1, keepdim=True)) + u * dx.abs()
    dims = tuple(range(x.dim() - 1))
    rows = x.numel() // d
    return [*out, (dx, 1.05 * bound + 1e-30),
            ((dn * h).sum(dims), 1.05 * (rows + 2 * d + 40) * w * (size * h.abs()).sum(dims) + 1e-30)]
