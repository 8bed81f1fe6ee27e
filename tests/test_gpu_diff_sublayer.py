"""The operators as they are used together: an attention sublayer in its
differential form, forward and backward, against float64 autograd on the CPU; and
the Pairformer blocks with the dropout of their triangle updates.

Tolerances. The sublayer in bf16 rounds its values about eight times in a row
(norm, three projections, attention, head norm, output projection, sum), each
by at most 2^-8 of the value, in the root mean square 0.42 of that: 2e-2 in
norm holds ten standard deviations of a chain of eight and its gradients'
sixteen. float32: 2^-24 in place of 2^-8 and sums of up to 384 products; 2e-5."""

from __future__ import annotations

import pytest
import torch

from foldjax_amd import boltz2, kernels, openfold3, protenix
from foldjax_amd import params as P
from foldjax_amd import synthetic as syn
from foldjax_amd.pairformer import PairDropout, PairformerLayerWeights
from tests.gpu_util import say
from tests.test_gpu_dropout import mask_of

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
BAR = {BF: 2e-2, F32: 2e-5}


def sublayer(w, x, residual, bias, mask, drop):
    """h = x + residual; out = h + dropout(W_o norm_heads(diff_attention(norm(h))))"""
    b, n, c = x.shape
    heads, d = w["lam"].shape[1:]
    y, h = kernels.rms_norm(x, w["norm"], residual=residual)
    qkv = y @ w["qkv"].t()
    q, k, v = (t.unflatten(-1, (-1, e)).transpose(1, 2) for t, e in
               zip(qkv.split([2 * heads * d] * 3, -1), (d, d, 2 * d)))
    o = torch.empty(b, n, heads, 2 * d, dtype=x.dtype, device=x.device)
    _, lse = kernels.diff_attention(q, k, v, w["lam"], lambda_init=0.5, scale=d**-0.5, bias=bias, mask=mask,
                                    return_lse=True, out=o.transpose(1, 2))
    u = kernels.rms_norm(o, w["head"])
    upd = u.flatten(2) @ w["out"].t()
    out = kernels.dropout_add(upd, residual=h, **drop)
    return out, (y, h, q, k, v, o, lse, u)


def sublayer_backward(w, dout, kept, bias, mask, drop):
    y, h, q, k, v, o, lse, u = kept
    b, n, c = dout.shape
    d = w["lam"].shape[2]
    dupd = kernels.dropout_backward(dout, **drop)
    flat = lambda t: t.reshape(b * n, -1)  # noqa: E731
    g = {"out": flat(dupd).t() @ flat(u.flatten(2))}
    do, g["head"] = kernels.rms_norm_backward((dupd @ w["out"]).view_as(o), o, w["head"])
    dq, dk, dv, g["bias"], g["lam"] = kernels.diff_attention_backward(
        do.transpose(1, 2), q, k, v, w["lam"], lse, lambda_init=0.5, scale=d**-0.5, bias=bias, mask=mask)
    dqkv = torch.cat([t.transpose(1, 2).flatten(2) for t in (dq, dk, dv)], -1)
    g["qkv"] = flat(dqkv).t() @ flat(y)
    g["x"], g["norm"] = kernels.rms_norm_backward(dqkv @ w["qkv"], h, w["norm"], dh=dout)
    return g, do


def reference(w, x, residual, bias, mask, drop, dout):
    f = lambda t: t.detach().double().cpu().requires_grad_(True)  # noqa: E731
    w = {n: f(t) for n, t in w.items()}
    x, residual, bias = f(x), residual.double().cpu(), f(bias)
    b, n, c = x.shape
    heads, d = w["lam"].shape[1:]
    norm = lambda t, g: t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * g  # noqa: E731
    h = x + residual
    q, k, v = (t.unflatten(-1, (-1, e)).transpose(1, 2) for t, e in
               zip((norm(h, w["norm"]) @ w["qkv"].t()).split([2 * heads * d] * 3, -1), (d, d, 2 * d)))
    part = mask.cpu()[:, None, None, :]
    p = []
    for m in range(2):
        s = torch.matmul(q[:, m::2], k[:, m::2].transpose(-1, -2)) * d**-0.5 + bias
        p.append(torch.softmax(s.masked_fill(~part, float("-inf")), -1))
    lam = ((w["lam"][0] * w["lam"][1]).sum(-1).exp() - (w["lam"][2] * w["lam"][3]).sum(-1).exp() + 0.5)[:, None, None]
    o = torch.matmul(p[0] - lam * p[1], v).transpose(1, 2)
    upd = norm(o, w["head"]).flatten(2) @ w["out"].t()
    keep = mask_of(upd.shape, drop["shared"], drop["p"], drop["seed"], drop["offset"])
    out = h + torch.where(keep, upd / (1 - drop["p"]), 0.0)
    (out * dout.double().cpu()).sum().backward()
    return out.detach(), {**{n: t.grad for n, t in w.items()}, "x": x.grad, "bias": bias.grad}


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n", [1, 45, 130])
def test_sublayer_and_its_gradients(n, dtype):
    say(f"differential sublayer n {n} {dtype}")
    g = torch.Generator().manual_seed(n)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    b, c, heads, d = 2, 384, 6, 32
    w = {"norm": 1 + 0.1 * r(c), "qkv": r(3 * c, c) * c**-0.5, "head": 1 + 0.1 * r(2 * d), "out": r(c, c) * c**-0.5}
    w = {k: t.to(dtype).cuda() for k, t in w.items()}
    w["lam"] = (0.1 * r(4, heads, d)).cuda()
    x, residual, dout = (t.to(dtype).cuda() for t in (r(b, n, c), r(b, n, c), r(b, n, c)))
    bias = r(b, heads, n, n).to(dtype).cuda()
    mask = (torch.arange(n) < max(1, n - n // 5)).expand(b, n).cuda()
    drop = {"p": 0.25, "seed": 17, "offset": 5, "shared": ()}
    out, kept = sublayer(w, x, residual, bias, mask, drop)
    got, do = sublayer_backward(w, dout, kept, bias, mask, drop)
    want_out, want = reference(w, x, residual, bias, mask, drop, dout)
    err = lambda a, b: float((a.double().cpu() - b).norm() / b.norm().clamp_min(1e-30))  # noqa: E731
    assert err(out, want_out) <= BAR[dtype]
    for name, t in got.items():
        if n == 1 and name == "bias":  # one key: its weight is 1 whatever the bias
            assert float(t.double().norm()) <= BAR[dtype]
        elif n == 1 and name == "lam":
            # with one key o = (1 - lambda) v, and the head norm takes the factor out
            # again: dO is orthogonal to v, dlambda = -sum dO v is zero, and what is
            # left is the rounding of its terms
            v = kept[4].transpose(1, 2)
            terms = float((do.double() * v.double()).abs().sum())
            assert float(t.abs().max()) <= BAR[dtype] * terms * float(w["lam"].abs().max()) * 2
        else:
            assert err(t, want[name]) <= BAR[dtype], name


def block(dtype, seed=3):
    return PairformerLayerWeights.random(dtype, "cuda", seed=seed)


def inputs(n, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    s = torch.randn(1, n, 384, generator=g).to(dtype).cuda()
    z = torch.randn(1, n, n, 128, generator=g).to(dtype).cuda()
    mask = (torch.arange(n) < n - 3).float().to(dtype).cuda()[None]
    return s, z, mask, mask[:, :, None] * mask[:, None, :]


def by_hand(tri, z, pm, drop, out_mask=None):
    """The four updates one at a time, each dropped on its own."""
    kinds = ((kernels.trimul, tri.tri_mul_out, {"direction": "outgoing"}),
             (kernels.trimul, tri.tri_mul_in, {"direction": "incoming"}),
             (kernels.triattn, tri.tri_att_start, {"starting": True}), (kernels.triattn, tri.tri_att_end, {"starting": False}))
    for i, (fn, w, k) in enumerate(kinds):
        u = fn(z, pm, w, **k)
        shared = tuple({-3: -2}.get(a, a) for a in drop.shared) if i == 3 else drop.shared
        z = kernels.dropout_add(u, p=drop.p, seed=drop.seed, offset=drop.offset + i, residual=z, shared=shared,
                                out_mask=out_mask)
    return z


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shared", [(-3,), (-3, -1)], ids=str)
def test_blocks_drop_their_triangle_updates(shared, dtype):
    say(f"block dropout {shared} {dtype}")
    w, (s, z, mask, pm) = block(dtype), inputs(21, dtype)
    drop = PairDropout(p=0.25, seed=99, offset=40, shared=shared)
    z0 = z.clone()
    want = by_hand(w.triangle, z, pm, drop)
    assert torch.equal(w.triangle.forward(z, pm, dropout=drop), want) and torch.equal(z, z0)
    donated = z.clone()
    got = w.triangle.forward(donated, pm, dropout=drop, donate=True)
    assert torch.equal(got, want) and got.data_ptr() == donated.data_ptr()
    gated = by_hand(w.triangle, z, pm, drop, out_mask=pm)
    assert torch.equal(w.triangle.forward(z, pm, out_mask=pm, dropout=drop), gated)
    # and the transition and the single track on top, as without dropout
    s1, z1 = boltz2.pairformer_layer_forward(w, s, z, mask, pm, triangle_backend="hip", dropout=drop)
    tri, w.triangle = w.triangle, None
    zt, bias = w._pair_transition(want.clone(), s)
    st = kernels.single_attention(s, None, mask, w.attention, residual=s, pair_bias=bias)
    st = kernels.transition(st, w.transition_s, residual=st)
    w.triangle = tri
    assert torch.equal(z1, zt) and torch.equal(s1, st)


def test_stacks_move_the_offset_and_no_dropout_stays_as_it_was():
    say("stack dropout")
    blocks = [block(BF, 3), block(BF, 30)]
    s, z, mask, pm = inputs(18, BF)
    drop = PairDropout(p=0.2, seed=4)
    s1, z1 = s, z
    for i, w in enumerate(blocks):
        s1, z1 = w.forward(s1, z1, mask, pm, dropout=drop.of_block(i))
    s2, z2 = boltz2.pairformer_module_forward({"layers": blocks}, s, z, mask, pm, triangle_backend="hip", dropout=drop)
    assert torch.equal(s1, s2) and torch.equal(z1, z2)
    plain = boltz2.pairformer_module_forward({"layers": blocks}, s, z, mask, pm, triangle_backend="hip")
    again = boltz2.pairformer_module_forward({"layers": blocks}, s, z, mask, pm, triangle_backend="hip", dropout=None)
    assert torch.equal(plain[1], again[1]) and not torch.equal(plain[1], z2)
    p = protenix.pairformer_block(s, z, pm, blocks[0], triangle_attention_backend="hip", dropout=drop)
    q = blocks[0].forward_protenix(s, z, pm, dropout=drop)
    assert torch.equal(p[1], q[1]) and (p[1][pm == 0] == 0).all()
    o = openfold3.pairformer_block(s, z, blocks[0], single_mask=mask, pair_mask=pm, no_heads_pair=4, no_heads_pair_bias=16,
                                   dropout=drop)
    assert torch.equal(o[1], blocks[0].forward_openfold3(s, z, mask, pm, dropout=drop)[1])


def test_pair_blocks_without_a_single_track():
    """The same sublayers as a whole layer's: the same bits of z."""
    say("pair blocks dropout")
    params = P.pairformer_layer_to_boltz2(syn.pairformer_layer_weights(seed=31))
    s, z, mask, pm = inputs(19, BF)
    drop = PairDropout(p=0.25, seed=6, offset=12)
    tri = {k: params[k] for k in ("tri_mul_out", "tri_mul_in", "tri_att_start", "tri_att_end", "transition_z")}
    _, want = boltz2.pairformer_layer_forward(params, s, z, mask, pm, dropout=drop)
    got = boltz2.pairformer_no_seq_layer_forward(tri, z, pm, dropout=drop)
    assert torch.equal(got, want) and not torch.equal(got, boltz2.pairformer_no_seq_layer_forward(tri, z, pm))
    layer = block(BF)
    w = layer.triangle
    of3 = openfold3.PairBlockParams(tri_mul_out=w.tri_mul_out, tri_mul_in=w.tri_mul_in, tri_att_start=w.tri_att_start,
                                    tri_att_end=w.tri_att_end, pair_transition=layer.transition_z)
    got = openfold3.pair_block(z, of3, pair_mask=pm, no_heads_pair=4, dropout=drop)
    z1 = by_hand(w, z, pm, drop)
    assert torch.equal(got, kernels.transition(z1, layer.transition_z, row_mask=pm, residual=z1))


def test_a_captured_block_drops_anew():
    say("captured block dropout")
    w, (s, z, mask, pm) = block(BF), inputs(16, BF)
    step = torch.zeros((), dtype=torch.int64, device="cuda")
    drop = PairDropout(p=0.25, seed=1, offset=8, step=step)
    w.forward(s, z, mask, pm, dropout=drop)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, got = w.forward(s, z, mask, pm, dropout=drop)
        step += 4
    for i in range(3):
        graph.replay()
        _, want = w.forward(s, z, mask, pm, dropout=PairDropout(p=0.25, seed=1, offset=8 + 4 * i))
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"replay {i}"
