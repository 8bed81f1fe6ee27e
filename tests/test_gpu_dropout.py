"""Dropout against Philox 4x32-10 restated in Python integers (whose known
answers are checked on the CPU, tests/test_operator_arguments.py), bit for bit
in what is kept; the values by the type's own rounding: half a step (bf16
2^-8, fp32 2^-24), and in float32 the scale's and the product's (2^-23 of the
scaled term)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from foldjax_amd import kernels
from tests.gpu_util import say
from tests.philox import words

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0**-8, F32: 2.0**-24}


def mask_of(shape, shared, p, seed, offset):
    full = (1,) * max(0, 4 - len(shape)) + tuple(shape)
    full = (int(np.prod(full[:-3])),) + full[-3:]
    m = [1 if (a - 4) in shared else n for a, n in enumerate(full)]
    keep = words(int(np.prod(m)), seed, offset) >= np.uint64(int(p * 2**32))
    return torch.from_numpy(np.broadcast_to(keep.reshape(m), full).copy()).reshape(shape)


def make(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype), (3 * torch.randn(*shape, generator=g)).to(dtype)


SHAPES = [(8,), (5, 8), (3, 7, 24), (2, 9, 11, 128), (2, 2, 3, 5, 16), (1, 1, 1, 8), (1, 70, 3, 64), (1, 3, 70, 64)]
SHARED = [(), (-3,), (-2,), (-3, -2), (-1,), (-3, -1), (-2, -1), (-3, -2, -1)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("shared", SHARED, ids=str)
def test_values_and_gradient(shape, shared, dtype):
    if any(len(shape) < -a for a in shared):
        pytest.skip("no such axis")
    say(f"dropout {shape} shared {shared} {dtype}")
    p, seed, offset = 0.3, 2**63 + 12345, 2**40 + 17
    x, res = make(shape, dtype)
    keep = mask_of(shape, shared, p, seed, offset)
    more = {"p": p, "seed": seed, "offset": offset, "shared": shared}
    out = kernels.dropout_add(x.cuda(), residual=res.cuda(), **more).cpu()
    term = torch.where(keep, x.double() / (1 - p), 0.0)
    want = res.double() + term
    assert ((out.double() - want).abs() <= HALF[dtype] * want.abs() + 2.0**-23 * term.abs()).all()
    assert torch.equal(out[~keep], res[~keep])
    dx = kernels.dropout_backward(res.cuda(), **more).cpu()
    want = torch.where(keep, res.double() / (1 - p), 0.0)
    assert ((dx.double() - want).abs() <= (HALF[dtype] + 2.0**-23) * want.abs()).all() and (dx[~keep] == 0).all()


def test_long_runs_are_cut_and_counted():
    """Runs longer than a thread takes, in number enough that they are cut, and
    a mask index past 2^32 / 8 of nothing but the offset's low word."""
    say("dropout long runs")
    for shape, shared in (((1, 300, 300, 128), (-3,)), ((1, 300, 300, 128), (-2,)), ((1, 300, 301, 128), ()),
                          ((2, 333, 100, 64), (-3, -1)), ((3, 129, 130, 64), (-3, -2))):
        x, res = make(shape, BF)
        out = kernels.dropout_add(x.cuda(), p=0.25, seed=9, offset=2**64 - 1, residual=res.cuda(), shared=shared).cpu()
        keep = mask_of(shape, shared, 0.25, 9, 2**64 - 1)
        want = res.double() + torch.where(keep, x.double() / 0.75, 0.0)
        assert ((out.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-23 * x.double().abs()).all(), (shape, shared)


def test_p_zero_and_near_one():
    say("dropout extremes of p")
    x, res = make((40, 64), F32)
    assert torch.equal(kernels.dropout_add(x.cuda(), p=0.0, seed=1).cpu(), x)
    p = 1 - 2.0**-40  # the threshold is 2^32 - 1
    out = kernels.dropout_add(x.cuda(), p=p, seed=1, residual=res.cuda()).cpu()
    assert torch.equal(out, res)


def test_dropped_values_are_not_looked_at_and_masked_positions_are_zero():
    say("dropout NaN")
    x, res = make((4, 6, 6, 32), BF)
    keep = mask_of(x.shape, (-3,), 0.5, 3, 0)
    x[~keep] = float("nan")
    om = torch.ones(4, 6, 6)
    om[:, 5] = 0
    om[:, :, 5] = 0
    res[:, 5] = float("inf")
    out = kernels.dropout_add(x.cuda(), p=0.5, seed=3, residual=res.cuda(), shared=(-3,), out_mask=om.cuda()).cpu()
    assert torch.isfinite(out).all() and (out[om == 0] == 0).all()
    assert torch.equal(out[(om != 0)[..., None] & ~keep], res[(om != 0)[..., None] & ~keep])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_in_place_and_strided(dtype):
    say(f"dropout in place {dtype}")
    x, res = (t.cuda() for t in make((2, 20, 20, 64), dtype))
    more = {"p": 0.25, "seed": 5, "shared": (-2,)}
    want = kernels.dropout_add(x, residual=res, **more)
    a, b = x.clone(), res.clone()
    assert kernels.dropout_add(a, residual=res, out=a, **more).data_ptr() == a.data_ptr() and torch.equal(a, want)
    assert torch.equal(kernels.dropout_add(x, residual=b, out=b, **more), want) and torch.equal(b, want)
    t = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(kernels.dropout_add(t, residual=res, **more), want)
    z = x.clone()
    kernels.dropout_add(z, residual=z, out=z, **more)
    assert torch.equal(z, kernels.dropout_add(x, residual=x, **more))


def test_a_step_on_the_device_and_a_graph():
    """The step is added to the offset where the kernel runs, so that replays
    of one captured call draw new masks."""
    say("dropout graph")
    x, res = (t.cuda() for t in make((2, 30, 30, 64), BF))
    step = torch.zeros((), dtype=torch.int64, device="cuda")
    call = lambda **m: kernels.dropout_add(x, p=0.25, seed=11, residual=res, shared=(-3,), **m)  # noqa: E731
    first = call(offset=100)
    assert torch.equal(call(offset=100, step=step), first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(offset=100, step=step)
        step += 1
    seen = []
    for i in range(4):
        graph.replay()
        want = call(offset=100 + i)
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"replay {i}"
        seen.append(got.clone())
    assert not any(torch.equal(a, b) for i, a in enumerate(seen) for b in seen[:i])


def test_share_kept():
    """Of a million independent elements, the share kept is 1 - p to five
    standard deviations."""
    say("dropout share")
    x = torch.ones(1024, 1024, device="cuda")
    for p in (0.1, 0.25, 0.5):
        kept = float((kernels.dropout_add(x, p=p, seed=77) != 0).double().mean())
        assert abs(kept - (1 - p)) <= 5 * (p * (1 - p) / 2**20) ** 0.5
