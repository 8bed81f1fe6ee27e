"""Differential attention against its definition in float64 on the CPU: both
directions, every head layout, lengths from one key to many, masks that leave
rows empty, padding that holds NaN, strides, streams, graphs.

Tolerances. A bf16 result is off by half a step of its own rounding, 2^-8 of
the value; in the gradients' products dS and the maps' difference are rounded
to bf16 once more, 2^-8 a term. float32: a score is a dot product of up to 64
terms, off by at most 64 2^-24 of the sum of |terms| (here below 12, in log2
units: 5e-5), the exponential by one step; 2^-13 of the sum of |weight x value|
covers both and the bf16 weights' 16 bits. Independent roundings add up as
their root mean square in a norm, well below the worst case: bf16 2^-8 in all,
float32 1e-5."""

from __future__ import annotations

import math

import pytest
import torch

from foldjax_amd import kernels
from tests.gpu_util import say

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
SLACK = 2.0**-13
HALF = {BF: 2.0**-8, F32: 2.0**-24}
NORM = {BF: 2.0**-8, F32: 1e-5}
LOWEST_KEPT = -torch.finfo(F32).max / math.log2(math.e)


def make(lead, heads, kv, nq, nk, d, dtype, *, bias="plane", mask="none", seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"q": 1.2 * r(*lead, 2 * heads, nq, d), "k": 1.2 * r(*lead, 2 * kv, nk, d), "v": r(*lead, kv, nk, 2 * d),
         "dout": r(*lead, heads, nq, 2 * d)}
    t = {n: x.to(dtype) for n, x in t.items()}
    t["lam"] = 0.15 * r(4, heads, d)
    t["bias"] = None
    if bias != "none":
        planes = {"plane": lead, "shared": lead[:-1] + (1,) if lead else (), "one": ()}[bias]
        t["bias"] = (1.5 * r(*planes, heads, nq, nk)).to(dtype)
    t["mask"] = None
    if mask != "none":
        m = torch.rand(*lead, nk, generator=g) > 0.3
        if mask == "tail":
            m[:] = torch.arange(nk) < max(1, nk - nk // 3)
        if mask == "empty":
            m.view(-1, nk)[-1] = False
        t["mask"] = m
        # whatever an earlier computation left in the padding
        t["k"].masked_fill_(~m[..., None, :, None], math.nan)
        t["v"].masked_fill_(~m[..., None, :, None], math.inf)
        if t["bias"] is not None and bias == "plane":
            t["bias"].masked_fill_(~m[..., None, None, :], math.nan)
    t.update(init=0.4, scale=d**-0.5, heads=heads, kv=kv, lead=lead)
    return t


def reference(t, *, backward=False):
    """The definition, and the sums of absolute terms that the tolerances are
    relative to. Gradients by autograd."""
    f64 = torch.float64
    lead, heads, kv = t["lead"], t["heads"], t["kv"]
    n = len(lead)
    there = torch.ones(*lead, t["k"].shape[-2], dtype=torch.bool) if t["mask"] is None else t["mask"]
    at = there[..., None, :, None]
    leaf = lambda x: x.to(f64).requires_grad_(backward)  # noqa: E731
    q, lam = leaf(t["q"]), leaf(t["lam"])
    k = leaf(torch.where(at, t["k"].to(f64), 0.0))
    v = leaf(torch.where(at, t["v"].to(f64), 0.0))
    part = there[..., None, None, :]
    bias = None
    if t["bias"] is not None:
        b = t["bias"].to(f64)
        if b.dim() < n + 3:
            b = b.reshape((1,) * (n + 3 - b.dim()) + tuple(b.shape))
        ok = b.isnan() | (b > LOWEST_KEPT)
        part = part & ok
        bias = leaf(torch.where(ok & there[..., None, None, :] if t["bias"].isnan().any() else ok, b, 0.0))
    over = lambda x: x.repeat_interleave(heads // kv, n)  # noqa: E731
    vv = over(v)

    def soft(m):
        s = torch.matmul(q[(..., slice(m, None, 2), slice(None), slice(None))],
                         over(k[(..., slice(m, None, 2), slice(None), slice(None))]).transpose(-1, -2)) * t["scale"]
        if bias is not None:
            s = s + bias
        top = torch.where(part, s, -math.inf).amax(-1, keepdim=True).clamp_min(-1e300).detach()
        e = torch.where(part, torch.exp(torch.where(part, s - top, 0.0)), 0.0)
        return e / e.sum(-1, keepdim=True).clamp_min(1e-300)

    p1, p2 = soft(0), soft(1)
    l = ((lam[0] * lam[1]).sum(-1).exp() - (lam[2] * lam[3]).sum(-1).exp() + t["init"])[:, None, None]
    a = p1 - l * p2
    out = torch.matmul(a, vv)
    res = {"out": out.detach()}
    w = (p1 + l.abs() * p2).detach()
    terms = {"out": torch.matmul(w, vv.detach().abs())}
    if not backward:
        return res, terms
    do = t["dout"].to(f64)
    (out * do).sum().backward()
    res.update(dq=q.grad, dk=k.grad, dv=v.grad, dlam=lam.grad)
    # |dS| <= P (|dP| + |D|) with |dP| <= |dO| |v|
    with torch.no_grad():
        dp = torch.matmul(do.abs(), vv.abs().transpose(-1, -2))
        dq, dk = torch.zeros_like(q), torch.zeros_like(over(k).repeat_interleave(2, n)) * 0
        dk = torch.zeros(*lead, 2 * heads, *k.shape[-2:], dtype=f64)
        sum_ds = 0.0
        for m, p in ((0, p1), (1, l.abs() * p2)):
            ds = p * dp + p * (p * dp).sum(-1, keepdim=True)
            sel = (..., slice(m, None, 2), slice(None), slice(None))
            dq[sel] = t["scale"] * torch.matmul(ds, over(k[sel]).abs())
            dk[sel] = t["scale"] * torch.matmul(ds.transpose(-1, -2), q[sel].abs())
            sum_ds = sum_ds + ds
        fold = lambda x, per: x.unflatten(n, (kv, heads // kv, per)).sum(n + 1).flatten(n, n + 1)  # noqa: E731
        terms.update(dq=dq, dk=fold(dk, 2), dv=fold(torch.matmul(w.transpose(-1, -2), do.abs()), 1))
        d2 = (p2 * dp).sum((-1, -2)).reshape(-1, heads).sum(0)
        e = torch.stack([(lam[0] * lam[1]).sum(-1).exp()] * 2 + [(lam[2] * lam[3]).sum(-1).exp()] * 2)
        terms["dlam"] = (e * d2)[..., None] * lam[[1, 0, 3, 2]].abs()
        if bias is not None:
            res["dbias"] = bias.grad.reshape(t["bias"].shape)
            for axis in range(n):
                if bias.shape[axis] == 1:
                    sum_ds = sum_ds.sum(axis, keepdim=True)
            terms["dbias"] = sum_ds.reshape(t["bias"].shape)
    return res, terms


def on_gpu(t):
    return {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in t.items()}


def call(t, **more):
    return kernels.diff_attention(t["q"], t["k"], t["v"], t["lam"], lambda_init=t["init"], scale=t["scale"],
                                  bias=t["bias"], mask=t["mask"], **more)


def grads(t, lse, **more):
    g = kernels.diff_attention_backward(t["dout"], t["q"], t["k"], t["v"], t["lam"], lse, lambda_init=t["init"],
                                        scale=t["scale"], bias=t["bias"], mask=t["mask"], **more)
    return dict(zip(("dq", "dk", "dv", "dbias", "dlam"), g))


def check(name, got, want, terms, dtype):
    half = HALF[got.dtype] if got.dtype in HALF else HALF[dtype]
    got = got.double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    # a gradient's products: each term rounded once more in the tensors' type
    each = SLACK + (HALF[dtype] if name in ("dq", "dk", "dv") else 0.0)
    over = (got - want).abs() - (half * want.abs() + each * terms)
    assert over.max() <= 1e-30, f"{name}: {float(over.max()):.2e} past the bound"
    norm = NORM[dtype] if name != "dlam" else 1e-5
    err = float((got - want).norm())
    assert err <= norm * float(want.norm()) + 1e-7 * float(terms.norm()), f"{name}: {err / float(want.norm()):.2e} in norm"


# lead, heads, kv heads, nq, nk, d
SHAPES = [
    ((), 1, 1, 1, 1, 32),
    ((1,), 2, 1, 1, 1, 64),
    ((2,), 3, 3, 7, 5, 32),
    ((1,), 4, 2, 16, 64, 64),
    ((2,), 2, 2, 65, 63, 32),
    ((1, 5), 2, 2, 33, 33, 32),
    ((2, 3), 1, 1, 64, 64, 64),
    ((3,), 6, 2, 100, 257, 32),
    ((1,), 4, 1, 130, 129, 64),
]
BIAS_MASK = [("none", "none"), ("plane", "holes"), ("shared", "tail"), ("one", "empty"), ("none", "empty")]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("bias,mask", BIAS_MASK)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(shape, bias, mask, dtype):
    say(f"diff attention {shape} bias {bias} mask {mask} {dtype}")
    t = make(*shape, dtype, bias=bias, mask=mask, seed=sum(shape[1:]))
    want, terms = reference(t, backward=True)
    g = on_gpu(t)
    out, lse = call(g, return_lse=True)
    check("out", out, want["out"], terms["out"], dtype)
    got = grads(g, lse)
    torch.cuda.synchronize()
    for name in ("dq", "dk", "dv", "dlam", "dbias"):
        if name == "dbias" and t["bias"] is None:
            assert got["dbias"] is None
            continue
        check(name, got[name], want[name], terms[name], dtype)


# as many rows and keys as make 64 of them a workgroup's, with waves that share a
# block's keys (queries) and without
MANY = [
    ((4, 20), 4, 2, 70, 130, 32),
    ((16,), 8, 8, 65, 130, 32),
    ((11,), 6, 6, 129, 129, 32),
    ((9,), 10, 5, 40, 256, 32),
    ((24,), 6, 6, 66, 64, 32),
    ((2, 10), 8, 4, 48, 100, 64),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("bias,mask", BIAS_MASK)
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_many_rows(shape, bias, mask, dtype):
    test_forward_and_gradients(shape, bias, mask, dtype)


# few rows against many keys: the keys split over waves and workgroups
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", [((3,), 8, 2, 1, 2000, 64), ((1,), 4, 4, 2, 4099, 32), ((2,), 8, 1, 3, 1023, 32),
                                   ((1,), 2, 2, 17, 700, 64), ((1,), 1, 1, 1, 128, 32), ((1,), 1, 1, 1, 129, 64)], ids=str)
@pytest.mark.parametrize("bias,mask", [("none", "none"), ("plane", "holes"), ("none", "empty")])
def test_few_rows_long_keys(shape, bias, mask, dtype):
    say(f"diff attention, few rows {shape} bias {bias} mask {mask} {dtype}")
    t = make(*shape, dtype, bias=bias, mask=mask, seed=5)
    want, terms = reference(t)
    check("out", call(on_gpu(t)), want["out"], terms["out"], dtype)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("low", ["-inf", "lowest"])
def test_rows_that_the_bias_leaves_empty(low, dtype):
    say(f"empty rows by the bias {low} {dtype}")
    t = make((2,), 2, 2, 40, 70, 32, dtype, bias="plane")
    value = -math.inf if low == "-inf" else torch.finfo(dtype).min
    t["bias"][0, :, 3] = value
    t["bias"][1, 1, 39] = value
    t["bias"][:, :, :, 60:] = value
    t["bias"][0, 0, 5, :69] = value  # nothing but what is beyond 60: empty too
    want, terms = reference(t, backward=True)
    g = on_gpu(t)
    out, lse = call(g, return_lse=True)
    assert torch.all(out[0, :, 3] == 0) and torch.all(out[1, 1, 39] == 0) and torch.all(out[0, 0, 5] == 0)
    check("out", out, want["out"], terms["out"], dtype)
    got = grads(g, lse)
    assert torch.all(got["dq"][0, :, 3] == 0)
    for name in ("dq", "dk", "dv", "dlam", "dbias"):
        check(name, got[name], want[name], terms[name], dtype)


@pytest.mark.parametrize("nk", [70, 3000])
def test_large_scores_and_a_late_maximum(nk):
    """Scores of hundreds whose largest comes in the last block: the running
    maximum moves, by more than the slack, at every block."""
    say(f"large scores nk {nk}")
    t = make((1,), 2, 2, 20, nk, 32, F32, bias="plane")
    t["bias"] += torch.linspace(-300.0, 300.0, nk)
    want, terms = reference(t)
    # scores up to 400: their float32 steps of 2^-15 go into the exponential whole
    got = call(on_gpu(t)).double().cpu()
    assert ((got - want["out"]).abs() <= 2.0**-12 * terms["out"] + 2.0**-24 * want["out"].abs()).all()


def test_nearly_equal_maps_keep_their_difference():
    """q_1 = q_2 and k_1 = k_2 with lambda near one: the maps cancel to 1 %, and
    the result is still good to the type's own rounding."""
    say("nearly equal maps")
    t = make((2,), 2, 2, 64, 200, 32, BF, bias="plane")
    t["q"][..., 1::2, :, :] = t["q"][..., 0::2, :, :]
    t["k"][..., 1::2, :, :] = t["k"][..., 0::2, :, :]
    t["lam"].zero_()
    t["init"] = 0.99
    want, terms = reference(t)
    got = call(on_gpu(t)).double().cpu()
    # 2^-8 a value; the weights' 2^-16 of terms 200 times the result is 2^-8 again
    assert float((got - want["out"]).norm()) <= 2.0**-8 * float(want["out"].norm())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_strides_and_layouts(dtype):
    """Token-major projections, a packed qkv buffer, an offset that breaks the
    alignment, a bias with a wide row, an output in token-major order."""
    say(f"strides {dtype}")
    t = make((2,), 2, 2, 50, 50, 32, dtype, bias="plane", mask="tail")
    want, terms = reference(t, backward=True)
    g = on_gpu(t)
    packed = torch.empty(2, 50, 4 * 32 + 4 * 32 + 2 * 64, dtype=dtype, device="cuda")
    q = packed[..., :128].view(2, 50, 4, 32).transpose(1, 2)
    k = packed[..., 128:256].view(2, 50, 4, 32).transpose(1, 2)
    v = packed[..., 256:].view(2, 50, 2, 64).transpose(1, 2)
    q.copy_(g["q"]), k.copy_(g["k"]), v.copy_(g["v"])
    wide = torch.full((2, 2, 50, 83), math.nan, dtype=dtype, device="cuda")
    wide[..., 7:57] = g["bias"]
    odd = torch.empty(g["dout"].numel() + 1, dtype=dtype, device="cuda")[1:].view(g["dout"].shape)
    odd.copy_(g["dout"])
    g.update(q=q, k=k, v=v, bias=wide[..., 7:57], dout=odd, mask=g["mask"].to(torch.int32) * 5)
    out = torch.full((2, 50, 2, 64), 7.0, dtype=dtype, device="cuda")
    got, lse = call(g, return_lse=True, out=out.transpose(1, 2))
    assert got.data_ptr() == out.data_ptr()
    check("out", out.transpose(1, 2), want["out"], terms["out"], dtype)
    gr = grads(g, lse)
    for name in ("dq", "dk", "dv", "dlam", "dbias"):
        check(name, gr[name], want[name], terms[name], dtype)
    assert grads(g, lse, bias_grad=False)["dbias"] is None


def test_long_cache_offsets_past_32_bits():
    """One token against the far end of a cache of more than 2^31 elements
    (4.6 GB): the rows past the middle are addressed in 64 bits."""
    say("long cache")
    nk, d = 4_200_000, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = torch.empty(nk, 8 * d, dtype=BF, device="cuda")  # k: 2 heads x 2 maps, v: 2 heads
    cache.normal_(generator=g)
    k = cache[:, :4 * d].view(nk, 4, d).transpose(0, 1)
    v = cache[:, 4 * d:].view(nk, 2, 2 * d).transpose(0, 1)
    q = torch.randn(4, 1, d, generator=g, device="cuda").to(BF)
    lam = torch.zeros(4, 2, d, device="cuda")
    mask = torch.zeros(nk, dtype=torch.bool, device="cuda")
    mask[-1000:] = True
    mask[:3] = True
    out = kernels.diff_attention(q, k, v, lam, lambda_init=0.5, scale=0.125, mask=mask)
    sel = torch.cat([torch.arange(3), torch.arange(nk - 1000, nk)])
    t = {"q": q.cpu(), "k": k[:, sel.cuda()].cpu(), "v": v[:, sel.cuda()].cpu(), "lam": lam.cpu(), "bias": None, "mask": None,
         "init": 0.5, "scale": 0.125, "heads": 2, "kv": 2, "lead": ()}
    want, terms = reference(t)
    check("out", out, want["out"], terms["out"], BF)


def test_same_bits_again_and_rows_of_a_batch_alone():
    say("same bits")
    t = on_gpu(make((4, 3), 4, 2, 90, 90, 32, BF, bias="shared", mask="holes"))
    out, lse = call(t, return_lse=True)
    first = grads(t, lse)
    for _ in range(3):
        o, l = call(t, return_lse=True)
        again = grads(t, l)
        assert torch.equal(o, out) and torch.equal(l, lse)
        assert all(torch.equal(again[n], first[n]) for n in first)


def test_another_stream_and_a_graph():
    """The call on a side stream, and captured: replays see new inputs, and eager
    work between them changes nothing."""
    say("stream and graph")
    t = on_gpu(make((2, 3), 2, 2, 70, 70, 32, BF, bias="shared", mask="tail"))
    few = on_gpu(make((2,), 4, 2, 1, 900, 64, BF, bias="none", mask="tail"))

    def both():
        out, lse = call(t, return_lse=True)
        return [out, call(few), *grads(t, lse).values()]

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(3):
        t["q"].mul_(1.0 + 0.1 * i)
        few["q"].mul_(1.0 - 0.1 * i)
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {i}"


def test_gradients_against_differences():
    """The float32 kernels' gradients against central differences of the float64
    definition, in a few directions."""
    say("differences")
    t = make((2,), 2, 1, 9, 21, 32, F32, bias="plane", mask="holes", seed=3)
    t["bias"] = torch.nan_to_num(t["bias"])
    g = on_gpu(t)
    got = grads(g, call(g, return_lse=True)[1])
    gen = torch.Generator().manual_seed(0)
    do = t["dout"].double()
    for name, key in (("dq", "q"), ("dk", "k"), ("dv", "v"), ("dbias", "bias"), ("dlam", "lam")):
        direction = torch.randn(t[key].shape, generator=gen).double()
        if key in ("k", "v"):
            direction[~t["mask"][:, None, :, None].expand_as(direction)] = 0.0
        h = 1e-5
        ends = []
        for sign in (1, -1):
            moved = dict(t)
            moved[key] = torch.nan_to_num(t[key].double(), posinf=0.0) + sign * h * direction
            ends.append(float((reference(moved)[0]["out"] * do).sum()))
        want = (ends[0] - ends[1]) / (2 * h)
        have = float((got[name].double().cpu() * direction).sum())
        # float32 gradients: 1e-5 of their norm; the difference's own error is h^2
        assert abs(have - want) <= 1e-5 * float(got[name].double().norm()) * float(direction.norm()) + 1e-6, name


def test_calls_of_one_layout_see_their_own_tensors():
    """Calls of a layout seen before take their pointers anew: other tensors,
    another scale, a tensor of the same strides off its 16 bytes, a mask whose
    values changed in place."""
    say("one layout, other tensors")
    a, b = (make((2,), 2, 2, 33, 40, 32, BF, bias="plane", mask="holes", seed=s) for s in (1, 2))
    for t in (a, b, a):
        want, terms = reference(t, backward=True)
        g = on_gpu(t)
        out, lse = call(g, return_lse=True)
        check("out", out, want["out"], terms["out"], BF)
        got = grads(g, lse)
        for name in ("dq", "dk", "dv", "dlam", "dbias"):
            check(name, got[name], want[name], terms[name], BF)
    g = on_gpu(b)
    for name in ("q", "k", "v", "dout"):
        off = torch.empty(g[name].numel() + 1, dtype=BF, device="cuda")[1:].view(g[name].shape)
        moved = dict(g, **{name: off.copy_(g[name])})
        o, l = call(moved, return_lse=True)
        assert torch.equal(o, call(g)) and torch.equal(grads(moved, l)["dv"], grads(g, l)["dv"])
    g["mask"][:, 5] ^= True
    g["k"], g["v"], g["bias"] = (torch.nan_to_num(g[n], posinf=0.0) for n in ("k", "v", "bias"))
    t = {n: x.cpu() if isinstance(x, torch.Tensor) else x for n, x in g.items()}
    check("out", call(g), *(r["out"] for r in reference(t)), BF)
    t["scale"] = g["scale"] = 0.1
    check("out", call(g), *(r["out"] for r in reference(t)), BF)


def test_arguments_are_taken_by_value_and_never_written_over():
    """A scale given as a tensor counts with what it holds at the call; lambda's
    vectors may start at any element; an output over an input is refused."""
    say("arguments by value")
    t = on_gpu(make((2,), 2, 2, 40, 50, 32, BF))
    scale, init = torch.tensor(0.2), torch.tensor(0.4)
    more = {"bias": t["bias"], "mask": t["mask"]}
    run = lambda s, i, lam=t["lam"]: kernels.diff_attention(t["q"], t["k"], t["v"], lam, scale=s, lambda_init=i, **more)  # noqa: E731
    assert torch.equal(run(scale, init), run(float(scale), float(init)))
    scale.mul_(2.0)
    init.mul_(2.0)
    assert torch.equal(run(scale, init), run(float(scale), float(init)))
    assert not torch.equal(run(scale, init), run(0.2, 0.4))
    lam = torch.empty(t["lam"].numel() + 1, device="cuda")[1:].view_as(t["lam"]).copy_(t["lam"])
    assert torch.equal(run(0.2, 0.4, lam), run(0.2, 0.4))
    x = torch.zeros(2, 2, 50, 64, dtype=BF, device="cuda")
    q, k = x.view(2, 4, 50, 32), torch.randn(2, 4, 50, 32, device="cuda").to(BF)
    for given in ((q, k, k.view(2, 2, 50, 64)), (k, q, k.view(2, 2, 50, 64)), (k, k, x)):
        with pytest.raises(ValueError, match="out must not be"):
            kernels.diff_attention(*given, t["lam"], scale=0.2, lambda_init=0.4, out=x)
