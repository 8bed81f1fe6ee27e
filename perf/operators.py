"""Differential attention, root-mean-square norm and shared-mask dropout as a
caller runs them: what is timed, and against which plain form.

The three make up one attention sublayer in its differential form, beside the
attention core, the LayerNorms and the residual additions of a Pairformer
block: ``diff_attention`` takes the difference of two softmax maps, ``rms_norm``
normalises its heads (or the residual stream) and can leave 8-bit values with
their scales, ``dropout_add`` drops the update and adds the residual. Sizes are
those of the framework's own workloads: token counts of real complexes (245,
499 and 1003 are no multiple of anything), 128 channels of the pair track, 384
of the single one; two differential heads of 2 x 32 for the pair track's four
of 32, six for the single track's 384 channels.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
LOG2E = 1.4426950408889634
CODES = {"e4m3": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}


def listed():
    return [
        # the single track of a peptide: launches and host time are all there is
        _attn("diffattn_single_n37_bf16", items=1, rows=1, heads=6, kv=6, nq=37, nk=37, d=32, bias=True),
        # a training step of the single track: four crops padded to one length, the pair bias trained as well
        _attn("diffattn_step_single_n499_bf16", items=4, rows=1, heads=6, kv=6, nq=499, nk=499, d=32, bias=True,
              mask="tail", step=True),
        # a training step of triangle attention: every row of the pair tensor is an attention of its own, all
        # under one triangle bias, whose gradient is the sum over the rows
        _attn("diffattn_step_triangle_n245_bf16", items=1, rows=245, heads=2, kv=2, nq=245, nk=245, d=32, bias=True,
              mask="tail", step=True),
        # triangle attention of a larger complex, for its structure alone
        _attn("diffattn_triangle_n499_bf16", items=1, rows=499, heads=2, kv=2, nq=499, nk=499, d=32, bias=True),
        # the single track in float32, as Boltz-2 keeps it; one item of the batch is padding throughout
        _attn("diffattn_step_single_n256_fp32", items=2, rows=1, heads=6, kv=6, nq=256, nk=256, d=32, bias=True,
              mask="empty", step=True, dtype="fp32"),
        # the newest token of each of eight sequences against its long cache, four heads to one of the cache
        _attn("diffattn_token_n16384_bf16", items=8, rows=1, heads=8, kv=2, nq=1, nk=16384, d=64, bias=False),
        # the pair track's residual stream normalised into 8-bit rows for the projections that follow
        _norm("rmsnorm_pair_n1003_e4m3", rows=1003 * 1003, c=128, codes="e4m3"),
        # a training step of the single track's norm
        _norm("rmsnorm_step_single_n499_bf16", rows=4 * 499, c=384, step=True),
        # a training step of the heads' norm (64 channels a head) over a pair tensor, in float32
        _norm("rmsnorm_step_heads_n245_fp32", rows=245 * 245 * 2, c=64, step=True, residual=False, dtype="fp32"),
        # the pair track's dropout, one mask for all rows, with its gradient
        _drop("dropout_step_pair_n1003_bf16", batch=1, n=1003, m=1003, c=128, shared="rows", p=0.25, step=True),
        # the single track's dropout, a value of its own for every element
        _drop("dropout_single_n499_fp32", batch=1, n=4, m=499, c=384, shared="none", p=0.1, dtype="fp32"),
        # a peptide's pair tensor, one mask for all columns
        _drop("dropout_pair_n37_bf16", batch=1, n=37, m=37, c=128, shared="columns", p=0.25),
    ]


def _attn(name, *, items, rows, heads, kv, nq, nk, d, bias, mask="none", step=False, dtype="bf16", init=0.5):
    return {"name": name, "op": "diff_attention", "items": items, "rows": rows, "heads": heads, "kv": kv, "nq": nq,
            "nk": nk, "d": d, "bias": bias, "mask": mask, "step": step, "dtype": dtype, "init": init}


def _norm(name, *, rows, c, codes="none", group=0, step=False, residual=True, dtype="bf16"):
    return {"name": name, "op": "rms_norm", "rows": rows, "c": c, "codes": codes, "group": group, "step": step,
            "residual": residual, "dtype": dtype}


def _drop(name, *, batch, n, m, c, shared, p, step=False, dtype="bf16"):
    return {"name": name, "op": "dropout", "batch": batch, "n": n, "m": m, "c": c, "shared": shared, "p": p,
            "step": step, "dtype": dtype}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["single", "triangle", "token", "norm", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "single":
        n = _log(rng, 2, 1003)
        heads = rng.choice([2, 4, 6, 8])
        case = _attn(None, items=rng.randint(1, 4 if n < 500 else 2), rows=1, heads=heads,
                     kv=rng.choice([heads, heads // 2]), nq=n, nk=rng.choice([n, n, _log(rng, 1, 1003)]),
                     d=rng.choice([32, 64]), bias=rng.random() < 0.7, mask=rng.choice(["none", "tail", "empty"]),
                     step=rng.random() < 0.6, dtype=dtype, init=rng.uniform(0.2, 0.8))
    elif op == "triangle":
        step = rng.random() < 0.5
        n = _log(rng, 5, 245 if step else 400)
        case = _attn(None, items=1, rows=rng.randint(max(1, n // 2), n), heads=rng.choice([1, 2]), kv=0, nq=n, nk=n,
                     d=32, bias=True, mask=rng.choice(["none", "tail", "empty"]), step=step, dtype=dtype,
                     init=rng.uniform(0.2, 0.8))
        case["kv"] = case["heads"]
    elif op == "token":
        heads = rng.choice([4, 8])
        case = _attn(None, items=rng.randint(1, 8), rows=1, heads=heads, kv=rng.choice([heads, heads // 4]),
                     nq=rng.choice([1, 1, 2, 5]), nk=_log(rng, 1, 16384), d=rng.choice([32, 64]),
                     bias=rng.random() < 0.3, mask=rng.choice(["none", "tail"]), dtype=dtype,
                     init=rng.uniform(0.2, 0.8))
    elif op == "norm":
        c = rng.choice([64, 128, 136, 256, 384, 512, 768, 1024, 1536, 2048])
        rows = _log(rng, 1, (1 << 26) // c)
        if rng.random() < 0.4:
            group = rng.choice([0, 32, 64, 128])
            case = _norm(None, rows=rows, c=c, codes=rng.choice(["e4m3", "int8"]), group=group if c % max(group, 1) == 0
                         else 0, residual=rng.random() < 0.6)
        else:
            case = _norm(None, rows=rows, c=c, step=rng.random() < 0.6, residual=rng.random() < 0.6, dtype=dtype)
    else:
        n, m = _log(rng, 1, 700), _log(rng, 1, 700)
        case = _drop(None, batch=rng.randint(1, 2), n=n, m=m, c=rng.choice([8, 64, 128]),
                     shared=rng.choice(["none", "rows", "columns", "rows and channels", "columns and channels"]),
                     p=rng.choice([0.1, 0.15, 0.25, 0.5]), step=rng.random() < 0.5, dtype=dtype)
    del case["name"]
    return case


# ------------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)


def prepare(case, seed):
    r, dt, op = _gen(seed), DTYPES[case["dtype"]], case["op"]
    st = {"case": case}
    if op == "diff_attention":
        b, i, h, kv, nq, nk, d = (case[x] for x in ("items", "rows", "heads", "kv", "nq", "nk", "d"))
        # as the projections leave them: token by token, the heads of a token side by side
        st["q"] = (1.2 * r(b, i, nq, 2 * h, d)).to(dt).transpose(2, 3)
        st["k"] = (1.2 * r(b, i, nk, 2 * kv, d)).to(dt).transpose(2, 3)
        st["v"] = r(b, i, nk, kv, 2 * d).to(dt).transpose(2, 3)
        st["dout"] = r(b, i, nq, h, 2 * d).to(dt).transpose(2, 3) if case["step"] else None
        st["lam"] = 0.1 * r(4, h, d)
        st["bias"] = (1.5 * r(b, 1, h, nq, nk)).to(dt) if case["bias"] else None
        st["mask"] = None
        if case["mask"] != "none":  # the last tenth of the keys is padding; or a whole item is
            keys = torch.arange(nk, device=DEVICE)
            real = torch.full((b, i), max(1, nk - nk // 10), device=DEVICE)
            if case["mask"] == "empty":
                real.view(-1)[-1] = 0
            st["mask"] = keys < real[..., None]
            # padding holds whatever an earlier computation left there
            st["k"].masked_fill_(~st["mask"][:, :, None, :, None], math.inf)
            st["v"].masked_fill_(~st["mask"][:, :, None, :, None], math.nan)
            if case["bias"] and case["mask"] == "empty":  # a token that may look at none
                st["bias"][:, :, :, nq // 2, :] = torch.finfo(dt).min
    elif op == "rms_norm":
        rows, c = case["rows"], case["c"]
        st["x"] = r(rows, c).to(dt)
        st["residual"] = (4.0 * r(rows, c)).to(dt) if case["residual"] else None
        st["w"] = (1.0 + 0.2 * r(c)).to(dt)
        st["dy"] = r(rows, c).to(dt) if case["step"] else None
        st["dh"] = r(rows, c).to(dt) if case["step"] and case["residual"] else None
    else:
        shape = (case["batch"], case["n"], case["m"], case["c"])
        st["x"] = r(*shape).to(dt)
        st["residual"] = (4.0 * r(*shape)).to(dt)
        st["dout"] = r(*shape).to(dt) if case["step"] else None
        st["seed"], st["offset"] = 0x9E3779B97F4A7C15 ^ seed, 1000 * seed + 7
    return st


# --------------------------------------------------------------- one pass


def run(st):
    return {"diff_attention": _run_attn, "rms_norm": _run_norm, "dropout": _run_drop}[st["case"]["op"]](st)


def _run_attn(st):
    case = st["case"]
    scale, init = case["d"] ** -0.5, case["init"]
    if own:
        from foldjax_amd import kernels

        more = {"bias": st["bias"], "mask": st["mask"], "lambda_init": init, "scale": scale}
        if not case["step"]:
            return kernels.diff_attention(st["q"], st["k"], st["v"], st["lam"], **more)
        out, lse = kernels.diff_attention(st["q"], st["k"], st["v"], st["lam"], return_lse=True, **more)
        g = kernels.diff_attention_backward(st["dout"], st["q"], st["k"], st["v"], st["lam"], lse, **more)
        return (out, *(x for x in g if x is not None))
    dt, h = st["q"].dtype, case["heads"]
    g = h // case["kv"]
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    if st["mask"] is not None:
        gone = ~st["mask"][:, :, None, :, None]
        k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    pairs = lambda t: t.unflatten(2, (-1, 2))  # noqa: E731  [.., 2 H, n, d] -> [.., H, 2, n, d]
    q, k = pairs(q), pairs(k).repeat_interleave(g, 2)
    v = v.repeat_interleave(g, 2)
    s = scale * torch.matmul(q, k.transpose(-1, -2).contiguous())
    if st["bias"] is not None:
        b = st["bias"].float()
        s = s + b.masked_fill(b * LOG2E == -math.inf, -math.inf).unsqueeze(3)
    if st["mask"] is not None:
        s = s.masked_fill(~st["mask"][:, :, None, None, None, :], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-37)
    l1, l2 = torch.exp((st["lam"][0] * st["lam"][1]).sum(-1)), torch.exp((st["lam"][2] * st["lam"][3]).sum(-1))
    lam = (l1 - l2 + init)[:, None, None]
    a = p[:, :, :, 0] - lam * p[:, :, :, 1]
    out = torch.matmul(a, v).to(dt)
    if not case["step"]:
        return out
    do = st["dout"].float()
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    u = p * dp.unsqueeze(3)
    D = u.sum(-1, keepdim=True)
    ds = u - p * D
    ds[:, :, :, 1] *= -lam
    fold = lambda t: t.unflatten(2, (case["kv"], g)).sum(3)  # noqa: E731  a shared head's gradient
    dq = (scale * torch.matmul(ds, k)).flatten(2, 3)
    dk = fold(scale * torch.matmul(ds.transpose(-1, -2).contiguous(), q)).flatten(2, 3)
    dv = fold(torch.matmul(a.transpose(-1, -2).contiguous(), do))
    dlam = -D[:, :, :, 1, :, 0].sum((0, 1, 3))
    w = torch.stack([dlam * l1, dlam * l1, -dlam * l2, -dlam * l2])[..., None]
    grads = [dq.to(dt), dk.to(dt), dv.to(dt), w * st["lam"][[1, 0, 3, 2]]]
    if st["bias"] is not None:
        grads.insert(3, ds.sum(3).sum(1, keepdim=True).to(dt))
    return (out, *grads)


def _values(codes, scales, dtype):
    return (codes.float().unflatten(-1, (scales.shape[-1], -1)) * scales[..., None]).flatten(-2).to(dtype)


def _run_norm(st):
    case, x, w, res, eps = st["case"], st["x"], st["w"], st["residual"], 1e-6
    if own:
        from foldjax_amd import kernels

        if case["codes"] != "none":
            y = kernels.rms_norm(x, w, residual=res, eps=eps, codes=case["codes"], group=case["group"])
            (codes, scales), h = (y[:2], y[2:])
            return (_values(codes, scales, x.dtype), *h)
        y = kernels.rms_norm(x, w, residual=res, eps=eps)
        if not case["step"]:
            return y
        y, h = (y, x) if res is None else y
        dx, dw = kernels.rms_norm_backward(st["dy"], h, w, dh=st["dh"], eps=eps)
        return (y, dx, dw) if res is None else (y, h, dx, dw)
    dt, wf = x.dtype, w.float()
    hf = x.float() if res is None else x.float() + res.float()
    yf = hf * torch.rsqrt((hf * hf).mean(-1, keepdim=True) + eps) * wf
    h = () if res is None else (hf.to(dt),)
    if case["codes"] != "none":
        kind, most = CODES[case["codes"]]
        yg = yf.unflatten(-1, (-1, case["group"] or case["c"]))
        top = yg.abs().amax(-1, keepdim=True)
        code = yg * (most / top).masked_fill(top == 0, 0.0)
        code = (torch.round(code) if kind is torch.int8 else code).to(kind)
        return (_values(code.flatten(-2), (top / most).squeeze(-1), dt), *h)
    if not case["step"]:
        return (yf.to(dt), *h) if h else yf.to(dt)
    hs = x.float() if res is None else h[0].float()  # the gradient is taken at the stored sum
    rstd = torch.rsqrt((hs * hs).mean(-1, keepdim=True) + eps)
    n, dy = hs * rstd, st["dy"].float()
    t = dy * wf
    dx = rstd * (t - n * (t * n).mean(-1, keepdim=True))
    if st["dh"] is not None:
        dx = dx + st["dh"].float()
    return (yf.to(dt), *h, dx.to(dt), (dy * n).sum(0))


def _keep(case, seed, offset):
    """The kept elements, in the mask's shape: word i % 4 of Philox 4x32-10 of the counter (i / 4, offset) under the
    key ``seed``, for element i of the mask, is at least p 2^32."""
    shape = _mask_shape(case)
    i = torch.arange((math.prod(shape) + 3) // 4, device=DEVICE)
    low = 0xFFFFFFFF
    c = [i & low, i >> 32, torch.full_like(i, offset & low), torch.full_like(i, offset >> 32)]
    key = [seed & low, (seed >> 32) & low]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & low) ^ c[1] ^ key[0], b & low, ((a >> 32) & low) ^ c[3] ^ key[1], a & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    return (torch.stack(c, -1).flatten()[:math.prod(shape)] >= int(case["p"] * 2**32)).view(shape)


def _mask_shape(case):
    sh = case["shared"]
    return (case["batch"], 1 if "rows" in sh else case["n"], 1 if "columns" in sh else case["m"],
            1 if "channels" in sh else case["c"])


def _run_drop(st):
    case, p = st["case"], st["case"]["p"]
    if own:
        from foldjax_amd import kernels

        shared = tuple(a for name, a in (("rows", -3), ("columns", -2), ("channels", -1)) if name in case["shared"])
        more = {"p": p, "seed": st["seed"], "offset": st["offset"], "shared": shared}
        out = kernels.dropout_add(st["x"], residual=st["residual"], **more)
        return (out, kernels.dropout_backward(st["dout"], **more)) if case["step"] else out
    f = _keep(case, st["seed"], st["offset"]).float() * (1.0 / (1.0 - p))
    dt = st["x"].dtype
    out = (st["residual"].float() + st["x"].float() * f).to(dt)
    return (out, (st["dout"].float() * f).to(dt)) if case["step"] else out


# ------------------------------------------------------------------- work


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "diff_attention":
        it, h, kv, nq, nk, d = case["items"] * case["rows"], case["heads"], case["kv"], case["nq"], case["nk"], case["d"]
        q, kvs, o = it * 2 * h * nq * d, it * 4 * kv * nk * d, it * 2 * h * nq * d
        bias = case["items"] * h * nq * nk if case["bias"] else 0
        mask = it * nk if case["mask"] != "none" else 0
        pairs = it * h * nq * nk
        # forward: two scores of d products, one product of the maps' difference with 2 d values
        if not case["step"]:
            return {"bytes": es * (q + kvs + o + bias) + mask + 16 * h * d, "flops": 8 * d * pairs}
        # backward: the scores again, dP, and the gradients of q, k and v
        return {"bytes": es * (2 * q + 2 * kvs + 2 * o + 2 * bias) + mask + 32 * h * d, "flops": 28 * d * pairs}
    if case["op"] == "rms_norm":
        e = case["rows"] * case["c"]
        res = 2 if case["residual"] else 0  # the residual in, the sum out
        if case["codes"] != "none":
            return {"bytes": e * (es * (1 + res) + 1) + 4 * e // (case["group"] or case["c"]) + es * case["c"],
                    "flops": 6 * e}
        if not case["step"]:
            return {"bytes": es * (e * (2 + res) + case["c"]), "flops": 5 * e}
        return {"bytes": es * e * (2 + res + 2 + res // 2) + (es + 4) * case["c"], "flops": 16 * e}
    e = case["batch"] * case["n"] * case["m"] * case["c"]
    return {"bytes": es * e * (5 if case["step"] else 3), "flops": (5 if case["step"] else 3) * e}


# ------------------------------------------------------------------- exact


def exact(case, seed):
    return {"diff_attention": _x_attn, "rms_norm": _x_norm, "dropout": _x_drop}[case["op"]](case, prepare(case, seed))


def _x_attn(case, st):
    """One map at a time, from scores in which a key that takes no part is not there at all."""
    f64, d, kv = torch.float64, case["d"], case["kv"]
    g, scale = case["heads"] // kv, case["d"] ** -0.5
    b, i, _, nq, _ = st["q"].shape
    nk = st["k"].shape[3]
    there = torch.ones(b, i, nk, dtype=torch.bool, device=DEVICE) if st["mask"] is None else st["mask"]
    clean = lambda t: torch.where(there[:, :, None, :, None], t.to(f64), 0.0)  # noqa: E731
    spread = lambda t: t[:, :, :, None].expand(-1, -1, -1, g, -1, -1).reshape(b, i, kv * g, nk, -1)  # noqa: E731
    k, v = clean(st["k"]), spread(clean(st["v"]))
    q = st["q"].to(f64)
    part = there[:, :, None, None, :]
    bias = None
    if st["bias"] is not None:
        bias = st["bias"].to(f64)
        part = part & (bias > -torch.finfo(torch.float32).max / math.log2(math.e))
    lv = st["lam"].to(f64)
    e1, e2 = (lv[0] * lv[1]).sum(-1).exp(), (lv[2] * lv[3]).sum(-1).exp()
    lam = (e1 - e2 + case["init"]).view(-1, 1, 1)

    def soft(t):
        s = torch.matmul(q[:, :, t::2], spread(k[:, :, t::2]).transpose(-1, -2).contiguous()) * scale
        if bias is not None:
            s = s + bias
        s = torch.where(part, s, -math.inf)
        w = torch.where(part, (s - torch.logsumexp(s, -1, keepdim=True)).exp(), 0.0)
        return torch.nan_to_num(w, nan=0.0)

    p1, p2 = soft(0), soft(1)
    a = p1 - lam * p2
    out = torch.matmul(a, v)
    if not case["step"]:
        return out
    do = st["dout"].to(f64)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    joined = lambda t: t.view(b, i, kv, g, nk, -1).sum(3)  # noqa: E731
    dq, dk, dbias, tr = torch.zeros_like(q), torch.zeros_like(k), 0.0, lambda t: t.transpose(-1, -2).contiguous()
    for t, (p, by) in enumerate(((p1, 1.0), (p2, -lam))):
        mean = (p * dp).sum(-1, keepdim=True)
        ds = by * p * (dp - mean)
        dq[:, :, t::2] = scale * torch.matmul(ds, spread(k[:, :, t::2]))
        dk[:, :, t::2] = scale * joined(torch.matmul(tr(ds), q[:, :, t::2].contiguous()))
        dbias = dbias + ds.sum(1, keepdim=True)
    dl = -mean.sum((0, 1, 3, 4))
    dlv = torch.stack([lv[1] * (dl * e1)[:, None], lv[0] * (dl * e1)[:, None], -lv[3] * (dl * e2)[:, None],
                       -lv[2] * (dl * e2)[:, None]])
    dv = joined(torch.matmul(tr(a), do))
    return (out, dq, dk, dv, dbias, dlv) if bias is not None else (out, dq, dk, dv, dlv)


def _x_norm(case, st):
    f64, eps = torch.float64, 1e-6
    x, w = st["x"].to(f64), st["w"].to(f64)
    h = x if st["residual"] is None else x + st["residual"].to(f64)
    y = w * h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    more = () if st["residual"] is None else (h,)
    if case["codes"] != "none":
        most = CODES[case["codes"]][1]
        yg = y.reshape(y.shape[0], -1, case["group"] or case["c"])
        step = yg.abs().amax(-1, keepdim=True) / most
        c = torch.where(step > 0, yg / step, 0.0)
        if case["codes"] == "e4m3":  # three bits behind the leading one, down to 2^-6
            unit = torch.exp2(torch.floor(torch.log2(c.abs().clamp_min(2.0**-6))) - 3)
            c = torch.round(c / unit) * unit
        else:
            c = torch.round(c)
        return ((c * step).reshape(y.shape), *more)
    if not case["step"]:
        return (y, *more) if more else y
    hs = x if st["residual"] is None else h.to(st["x"].dtype).to(f64)
    rms = torch.sqrt(hs.square().mean(-1, keepdim=True) + eps)
    dy = st["dy"].to(f64)
    along = (dy * w * hs).mean(-1, keepdim=True)
    dx = dy * w / rms - hs * along / rms**3
    if st["dh"] is not None:
        dx = dx + st["dh"].to(f64)
    return (y, *more, dx, (dy * hs / rms).sum(0))


def _mulhilo(a, m):
    """The two 32-bit halves of a product of 32-bit numbers, from 16-bit limbs."""
    a0, a1, m0, m1 = a % 65536, a // 65536, m % 65536, m // 65536
    mid = a1 * m0 + a0 * m1 + (a0 * m0) // 65536
    return a1 * m1 + mid // 65536, (mid % 65536) * 65536 + (a0 * m0) % 65536


def _x_drop(case, st):
    shape = _mask_shape(case)
    count = math.prod(shape)
    blocks = torch.arange(-(-count // 4), device=DEVICE)
    two = 2**32
    x0, x1 = blocks % two, blocks // two
    x2, x3 = (torch.full_like(blocks, v) for v in (st["offset"] % two, st["offset"] // two))
    k0, k1 = st["seed"] % two, st["seed"] // two
    for r in range(10):
        h0, l0 = _mulhilo(x0, 3528531795)
        h1, l1 = _mulhilo(x2, 3449720151)
        x0, x1, x2, x3 = (h1 ^ x1 ^ ((k0 + r * 2654435769) % two), l1, h0 ^ x3 ^ ((k1 + r * 3144134277) % two), l0)
    words = torch.empty(blocks.numel() * 4, dtype=torch.int64, device=DEVICE)
    for j, x in enumerate((x0, x1, x2, x3)):
        words[j::4] = x
    keep = (words[:count].view(shape) >= math.floor(case["p"] * two)).expand(st["x"].shape)
    drop = lambda t: torch.where(keep, t.to(torch.float64) / (1.0 - case["p"]), 0.0)  # noqa: E731
    out = st["residual"].to(torch.float64) + drop(st["x"])
    return (out, drop(st["dout"])) if case["step"] else out
