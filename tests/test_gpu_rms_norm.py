"""RMS norm, its 8-bit output and its gradients against float64 on the CPU.

Tolerances: a result is off by half a step of its type (bf16 2^-8, fp32 2^-24)
and by float32's arithmetic, for a row of c channels at most (c + 8) 2^-24 of
the sums of absolute terms: 2^-10 at 8192 channels for a sum in one chain, and
below 2^-16 for the tree sums the kernels use (chains of at most 40, then at most
8 levels: 48 2^-24). A code is off by half a step of 8 bits (e4m3: 2^-4 of
the value, or 2^-10 of the unit below 2^-6; int8: half), plus one more where
float32 puts a value on the other side of a tie, which the tests allow as
2^-16 of the value."""

from __future__ import annotations

import math

import pytest
import torch

from foldjax_amd import kernels
from tests.gpu_util import say

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0**-8, F32: 2.0**-24}
SUMS = 2.0**-16
WIDTHS = [8, 64, 72, 128, 136, 256, 384, 512, 520, 1024, 1032, 2048, 2056, 4096, 4104, 8192]


def tensors(rows, c, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return [x.to(dtype) for x in (r(rows, c), 3 * r(rows, c), 1 + 0.3 * r(c), r(rows, c), r(rows, c))]


def reference(x, res, w, eps):
    h = x.double() + (0 if res is None else res.double())
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double(), h


def near(got, want, dtype, slack=0.0):
    got = got.double().cpu()
    over = (got - want).abs() - (HALF[dtype] + SUMS) * want.abs() - slack
    assert over.max() <= 0, float(over.max())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("rows", [1, 3, 37, 1000])
def test_norm_and_gradients(rows, c, dtype):
    say(f"rms norm {rows} x {c} {dtype}")
    x, res, w, dy, dh = tensors(rows, c, dtype, seed=c)
    eps = 1e-6
    y, h = kernels.rms_norm(x.cuda(), w.cuda(), residual=res.cuda(), eps=eps)
    want, hw = reference(x, res, w, eps)
    near(h, hw, dtype)
    near(y, want, dtype)
    alone = kernels.rms_norm(x.cuda(), w.cuda(), eps=eps)
    near(alone, reference(x, None, w, eps)[0], dtype)

    stored = h.double().cpu().requires_grad_(True)
    wl = w.double().requires_grad_(True)
    out = stored / torch.sqrt(stored.square().mean(-1, keepdim=True) + eps) * wl
    ((out * dy.double()).sum() + (stored * dh.double()).sum()).backward()
    dx, dw = kernels.rms_norm_backward(dy.cuda(), h, w.cuda(), dh=dh.cuda(), eps=eps)
    with torch.no_grad():
        rstd = 1 / torch.sqrt(stored.square().mean(-1, keepdim=True) + eps)
        n = stored * rstd
        t = dy.double() * wl
        terms = rstd * (t.abs() + n.abs() * (t * n).abs().mean(-1, keepdim=True)) + dh.double().abs()
    near(dx, stored.grad, dtype, slack=SUMS * terms)
    assert dw.dtype == F32
    near(dw, wl.grad, F32, slack=SUMS * (dy.double() * n).abs().sum(0))
    # without the sum's own gradient
    dx0, _ = kernels.rms_norm_backward(dy.cuda(), h, w.cuda(), eps=eps)
    near(dx0, stored.grad - dh.double(), dtype, slack=SUMS * terms)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("c", [64, 128, 384, 512, 1024, 1152, 8192])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_codes(c, group, codes, dtype):
    if group and c % group:
        pytest.skip("the group does not divide the channels")
    say(f"rms norm codes {c} {group} {codes} {dtype}")
    x, res, w, _, _ = tensors(29, c, dtype, seed=c + group)
    x[3] = 0
    res[3] = 0
    q, scale, h = kernels.rms_norm(x.cuda(), w.cuda(), residual=res.cuda(), codes=codes, group=group)
    assert q.dtype == (torch.float8_e4m3fn if codes == "e4m3" else torch.int8) and q.shape == x.shape
    assert scale.dtype == F32 and scale.shape == (29, c // group if group else 1)
    y, hw = reference(x, res, w, 1e-6)
    near(h, hw, dtype)
    most = 448.0 if codes == "e4m3" else 127.0
    yg = y.unflatten(-1, (-1, group or c))
    top = yg.abs().amax(-1)
    near(scale, top / most, F32)
    code = q.double() if codes == "int8" else q.float().double()
    code = code.cpu().unflatten(-1, (-1, group or c))
    want = torch.where(top[..., None] > 0, yg / (top[..., None] / most), 0.0)
    half = torch.full_like(want, 0.5) if codes == "int8" else torch.maximum(want.abs() * 2.0**-4, torch.tensor(2.0**-10))
    assert ((code - want).abs() <= half + 2 * SUMS * want.abs()).all()
    assert code.abs().max() == most and (code[3] == 0).all() and (scale[3] == 0).all()


def test_values_that_are_not_finite_stay_visible():
    say("rms norm NaN")
    x, res, w, _, _ = tensors(6, 128, BF)
    x[1, 5] = math.nan
    x[4, 100] = math.inf
    y, h = kernels.rms_norm(x.cuda(), w.cuda(), residual=res.cuda())
    assert y[1].isnan().all() and h[1, 5].isnan() and y[4, 100].isnan() and (y[4, :100] == 0).all()
    assert torch.isfinite(y[[0, 2, 3, 5]]).all()
    for codes in ("e4m3", "int8"):
        for group, at in ((0, 0), (64, 1)):
            q, s, _ = kernels.rms_norm(x.cuda(), w.cuda(), residual=res.cuda(), codes=codes, group=group)
            assert s[1].isnan().all() and s[4, at].isnan() and torch.isfinite(s[[0, 2, 3, 5]]).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_in_place_strided_and_leading_axes(dtype):
    say(f"rms norm in place {dtype}")
    x, res, w, dy, dh = (t.cuda() for t in tensors(60, 128, dtype))
    y, h = kernels.rms_norm(x, w, residual=res)
    x3 = x.view(3, 4, 5, 128)
    y3, h3 = kernels.rms_norm(x3, w, residual=res.view(3, 4, 5, 128))
    assert torch.equal(y3.view(60, 128), y) and torch.equal(h3.view(60, 128), h)
    wide = torch.zeros(60, 200, dtype=dtype, device="cuda")
    wide[:, 3:131] = x
    assert torch.equal(kernels.rms_norm(wide[:, 3:131], w, residual=res)[0], y)
    dx, dw = kernels.rms_norm_backward(dy, h, w, dh=dh)
    for target in ("dy", "dh"):
        a, b = dy.clone(), dh.clone()
        into = a if target == "dy" else b
        dx2, dw2 = kernels.rms_norm_backward(a, h, w, dh=b, out=into)
        assert dx2.data_ptr() == into.data_ptr() and torch.equal(into, dx) and torch.equal(dw2, dw)
    xi, ri = x.clone(), res.clone()
    y2, h2 = kernels.rms_norm(xi, w, residual=ri, out=xi, sum_out=ri)
    assert y2.data_ptr() == xi.data_ptr() and torch.equal(xi, y) and torch.equal(ri, h)


def test_graph():
    say("rms norm graph")
    x, res, w, dy, dh = (t.cuda() for t in tensors(500, 384, BF))

    def both():
        y, h = kernels.rms_norm(x, w, residual=res)
        q, s, _ = kernels.rms_norm(x, w, residual=res, codes="e4m3", group=128)
        return [y, h, q.view(torch.uint8), s, *kernels.rms_norm_backward(dy, h, w, dh=dh)]

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(3):
        x.mul_(1.1)
        dy.add_(0.1 * i)
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {i}"
