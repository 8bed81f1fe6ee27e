"""Attention over packed sequences and the norm of queries and keys with their
rotation, as a caller runs them: what is timed, and against which plain form.

The two make up the attention sublayer of a sequence track: sequences of
different lengths lie one behind the other, ``head_norm_rotary`` normalises each
head's queries and keys and rotates them by their positions (residue, chain,
copy: up to several axes), ``packed_attention`` lets each sequence's queries see
its own keys, all of them or those up to their own place, and a newest token the
cache of its sequence. Token counts are those of real complexes (37, 245, 499,
1003 are no multiple of anything) and generic lengths up to 16384; 16 heads of
24, 12 of 32 and 6 of 64 are the 384 channels of the single track, 8 heads of
128 on 2 of the cache those of a track of 1024.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one peptide: launches and host time are all there is
        _attn("attn_single_n37_bf16", lens="37", heads=16, kv=16, d=24),
        # a training step over six crops packed without padding between them, the rest of the buffer unused
        _attn("attn_step_crops_bf16", lens="499,245,37,1003,1,150", tail=113, heads=16, kv=16, d=24, step=True),
        # four complexes read at once, heads of 64
        _attn("attn_crops_n1003_bf16", lens="1003,499,999,245", heads=6, kv=6, d=64),
        # prompts of very different lengths, four query heads to one of keys and values
        _attn("attn_prompt_n16384_bf16", lens="9001,4096,3002,245,39,1", heads=8, kv=2, d=128, causal=True),
        # a training step over packed sequences, each token seeing those before it
        _attn("attn_step_prompt_n8192_bf16", lens="4099,2048,1003,999,43", heads=8, kv=2, d=128, causal=True, step=True),
        # the single track in float32, as Boltz-2 keeps it
        _attn("attn_step_n455_fp32", lens="256,199", heads=12, kv=12, d=32, causal=True, step=True, dtype="fp32"),
        # the newest token of each of eight sequences against its cache of up to 16384 tokens
        _token("attn_token_n16384_bf16", lens="16384,12001,16000,9,8192,16383,15000,1003", cap=16384, nq=1, heads=8, kv=2,
               d=128),
        # the newest token of eight sequences, at far positions
        _rot("rotary_token_bf16", tokens=8, heads=8, kv=2, d=128, sections="64", far=1000000),
        # a prompt's queries and keys
        _rot("rotary_prompt_n16384_bf16", tokens=16384, heads=8, kv=2, d=128, sections="64"),
        # a training step over crops: residue, chain and copy take a third of the pairs each
        _rot("rotary_step_crops_bf16", tokens=2048, heads=16, kv=16, d=24, sections="4,4,4", step=True),
        # a training step over long sequences, three axes of different shares
        _rot("rotary_step_n8192_bf16", tokens=8192, heads=8, kv=2, d=128, sections="16,24,24", step=True),
        # a training step in float32: neighbouring channels a pair, half of the channels rotated, no norm
        _rot("rotary_step_n1996_fp32", tokens=1996, heads=12, kv=12, d=32, sections="8", interleaved=True, norm=False,
             step=True, dtype="fp32"),
    ]


def _attn(name, *, lens, heads, kv, d, tail=0, causal=False, step=False, dtype="bf16"):
    """Sequences against themselves; ``tail`` rows behind the last one."""
    return {"name": name, "op": "attention", "lens": lens, "tail": tail, "heads": heads, "kv": kv, "d": d,
            "causal": causal, "step": step, "dtype": dtype}


def _token(name, *, lens, cap, nq, heads, kv, d, dtype="bf16"):
    """The last ``nq`` tokens of each sequence against a cache that holds ``lens`` of ``cap`` keys."""
    return {"name": name, "op": "token", "lens": lens, "cap": cap, "nq": nq, "heads": heads, "kv": kv, "d": d,
            "causal": True, "step": False, "dtype": dtype}


def _rot(name, *, tokens, heads, kv, d, sections, far=0, interleaved=False, norm=True, step=False, dtype="bf16"):
    """``sections``: the rotated pairs of each position axis."""
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv": kv, "d": d, "sections": sections,
            "far": far, "interleaved": interleaved, "norm": norm, "step": step, "dtype": dtype}


def _ints(text):
    return [int(x) for x in text.split(",")]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["crops", "prompt", "token", "rotary"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    lens = lambda most, count: ",".join(str(_log(rng, 1, most)) for _ in range(rng.randint(1, count)))  # noqa: E731
    if op == "crops":
        heads, d = rng.choice([(16, 24), (12, 32), (6, 64), (4, 64), (3, 128)])
        case = _attn(None, lens=lens(1003, 8), tail=rng.choice([0, rng.randint(1, 200)]), heads=heads,
                     kv=heads if rng.random() < 0.7 or heads % 2 else heads // 2, d=d, causal=rng.random() < 0.3,
                     step=rng.random() < 0.6, dtype=dtype)
    elif op == "prompt":
        step = rng.random() < 0.5
        kv = rng.choice([1, 2, 4])
        case = _attn(None, lens=lens(4099, 6), heads=min(8, kv * rng.choice([2, 4])), kv=kv,
                     d=rng.choice([64, 128]), causal=True, step=step, dtype=dtype)
        while work(case)["flops"] > (2e10 if dtype == "fp32" else 1.5e11):
            case["lens"] = ",".join(str(max(1, n // 2)) for n in _ints(case["lens"]))
    elif op == "token":
        cap = _log(rng, 16, 16384)
        kv = rng.choice([1, 2, 8])
        case = _token(None, lens=",".join(str(_log(rng, 1, cap)) for _ in range(rng.randint(1, 8))), cap=cap,
                      nq=rng.choice([1, 1, 1, 2, 5]), heads=kv * rng.choice([1, 4, 8]), kv=kv, d=rng.choice([32, 64, 128]),
                      dtype=dtype)
    else:
        heads, kv, d = rng.choice([(16, 16, 24), (12, 12, 32), (6, 6, 64), (8, 2, 64), (8, 2, 128), (8, 1, 128)])
        half = d // 2
        sections = rng.choice([f"{half}", f"{half // 2}", f"{half - 2 * (half // 3)},{half // 3},{half // 3}"])
        if sum(_ints(sections)) % 4:
            sections = f"{half}"
        case = _rot(None, tokens=_log(rng, 1, 8192), heads=heads, kv=kv, d=d, sections=sections,
                    far=rng.choice([0, 0, 100000]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.7,
                    step=rng.random() < 0.6, dtype=dtype)
    del case["name"]
    return case


# ------------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    r, dt, op = _gen(seed), DTYPES[case["dtype"]], case["op"]
    h, kv, d = case["heads"], case["kv"], case["d"]
    st = {"case": case}
    # as the projections leave them: token by token, the heads of a token side by side
    heads = lambda tokens, count, by=1.0: (by * r(tokens, count, d)).to(dt).transpose(0, 1)  # noqa: E731
    if op == "attention":
        lens = _ints(case["lens"])
        total = sum(lens) + case["tail"]
        st["q"], st["k"], st["v"] = heads(total, h, 1.3), heads(total, kv, 1.3), heads(total, kv)
        st["starts"] = torch.tensor(_starts(lens), dtype=torch.int32, device=DEVICE)
        st["dout"] = heads(total, h) if case["step"] else None
    elif op == "token":
        lens, cap = _ints(case["lens"]), case["cap"]
        st["q"] = heads(len(lens) * case["nq"], h, 1.3)
        st["k"], st["v"] = (t.contiguous() for t in (heads(len(lens) * cap, kv, 1.3), heads(len(lens) * cap, kv)))
        for i, n in enumerate(lens):  # behind a sequence's keys lies whatever was there before
            st["k"][:, i * cap + n:(i + 1) * cap] = math.inf
            st["v"][:, i * cap + n:(i + 1) * cap] = math.nan
        st["starts"] = torch.arange(len(lens) + 1, dtype=torch.int32, device=DEVICE) * case["nq"]
        st["k_starts"] = torch.arange(len(lens) + 1, dtype=torch.int32, device=DEVICE) * cap
        st["k_lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    else:
        t, sections = case["tokens"], _ints(case["sections"])
        st["q"], st["k"] = heads(t, h, 1.5), heads(t, kv, 1.5)
        weight = lambda: (1.0 + 0.2 * r(d)).to(dt) if case["norm"] else None  # noqa: E731
        st["wq"], st["wk"] = weight(), weight()
        place = torch.arange(t, device=DEVICE)
        axes = [place % 1003 + case["far"], place // 100 % 7, place // 37 % 5][:len(sections)]
        st["positions"] = torch.stack(axes).to(torch.int32)
        pairs = sum(sections)
        st["frequencies"] = 10000.0 ** -(torch.arange(pairs, dtype=torch.float64, device=DEVICE) / pairs)
        st["dq"], st["dk"] = (heads(t, h), heads(t, kv)) if case["step"] else (None, None)
    return st


# --------------------------------------------------------------- one pass


def run(st):
    return {"attention": _run_attn, "token": _run_attn, "rotary": _run_rot}[st["case"]["op"]](st)


def _spans(case):
    """(first query, queries, first key, keys) of each sequence."""
    lens = _ints(case["lens"])
    if case["op"] == "token":
        return [(i * case["nq"], case["nq"], i * case["cap"], n) for i, n in enumerate(lens)]
    return [(a, n, a, n) for a, n in zip(_starts(lens), lens)]


def _run_attn(st):
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    scale = case["d"] ** -0.5
    if own:
        from foldjax_amd import kernels

        more = {"scale": scale, "causal": case["causal"]}
        if case["op"] == "token":
            return kernels.packed_attention(q, k, v, st["starts"], k_starts=st["k_starts"], k_lengths=st["k_lengths"], **more)
        if not case["step"]:
            return kernels.packed_attention(q, k, v, st["starts"], **more)
        out, lse, rest = kernels.packed_attention(q, k, v, st["starts"], return_lse=True, **more)
        return (out, *kernels.packed_attention_backward(st["dout"], q, k, v, out, lse, rest, st["starts"], **more))
    dt, g = q.dtype, case["heads"] // case["kv"]
    new = lambda t: torch.zeros(t.shape, dtype=dt, device=t.device)  # noqa: E731
    out = new(q)
    dq, dk, dv = (new(q), new(k), new(v)) if case["step"] else (None, None, None)
    for q0, nq, k0, nk in _spans(case):
        qs = q[:, q0:q0 + nq].float()
        ks, vs = (t[:, k0:k0 + nk].float().repeat_interleave(g, 0) for t in (k, v))
        s = scale * torch.matmul(qs, ks.transpose(1, 2).contiguous())
        if case["causal"]:
            i, j = torch.arange(nq, device=q.device)[:, None], torch.arange(nk, device=q.device)
            s = s.masked_fill(j > i + nk - nq, -math.inf)
        top = s.amax(-1, keepdim=True)
        e = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
        p = e / e.sum(-1, keepdim=True).clamp_min(1e-37)
        o = torch.matmul(p, vs)
        out[:, q0:q0 + nq] = o.to(dt)
        if not case["step"]:
            continue
        do = st["dout"][:, q0:q0 + nq].float()
        ds = p * (torch.matmul(do, vs.transpose(1, 2).contiguous()) - (do * o).sum(-1, keepdim=True))
        fold = lambda t: t.unflatten(0, (case["kv"], g)).sum(1)  # noqa: E731  a shared head's gradient
        dq[:, q0:q0 + nq] = (scale * torch.matmul(ds, ks)).to(dt)
        dk[:, k0:k0 + nk] = fold(scale * torch.matmul(ds.transpose(1, 2).contiguous(), qs)).to(dt)
        dv[:, k0:k0 + nk] = fold(torch.matmul(p.transpose(1, 2).contiguous(), do)).to(dt)
    return (out, dq, dk, dv) if case["step"] else out


def _angles(st):
    """Cosines and sines [tokens, pairs], the angles in 64 bits."""
    axis = [a for a, n in enumerate(_ints(st["case"]["sections"])) for _ in range(n)]
    angle = st["positions"].to(torch.float64)[axis].T * st["frequencies"]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _halves(case, x):
    """The two members of each rotated pair, and the channels behind them."""
    n = 2 * sum(_ints(case["sections"]))
    turned, rest = x[..., :n], x[..., n:]
    if case["interleaved"]:
        return turned[..., 0::2], turned[..., 1::2], rest
    return turned[..., :n // 2], turned[..., n // 2:], rest


def _joined(case, a, b, rest):
    turned = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _run_rot(st):
    case, eps = st["case"], 1e-6
    if own:
        from foldjax_amd import kernels

        more = {"q_weight": st["wq"], "k_weight": st["wk"], "eps": eps, "sections": tuple(_ints(case["sections"])),
                "interleaved": case["interleaved"]}
        y = kernels.head_norm_rotary(st["q"], st["k"], st["positions"], st["frequencies"], **more)
        if not case["step"]:
            return y
        g = kernels.head_norm_rotary_backward(st["dq"], st["dk"], st["q"], st["k"], st["positions"], st["frequencies"],
                                              **more)
        return (*y, *(t for t in g if t is not None))
    cos, sin = _angles(st)
    outs, grads, weights = [], [], []
    for x, w, dy in ((st["q"], st["wq"], st["dq"]), (st["k"], st["wk"], st["dk"])):
        xf = x.float()
        rstd = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + eps) if case["norm"] else None
        y = xf * rstd * w.float() if case["norm"] else xf
        a, b, rest = _halves(case, y)
        outs.append(_joined(case, a * cos - b * sin, a * sin + b * cos, rest).to(x.dtype))
        if not case["step"]:
            continue
        a, b, rest = _halves(case, dy.float())
        dn = _joined(case, a * cos + b * sin, b * cos - a * sin, rest)
        if case["norm"]:
            n, t = xf * rstd, dn * w.float()
            weights.append((dn * n).sum((0, 1)))
            dn = rstd * (t - n * (t * n).mean(-1, keepdim=True))
        grads.append(dn.to(x.dtype))
    return (*outs, *grads, *weights)


# ------------------------------------------------------------------- work


def _pairs(case):
    """(query, key) pairs that take part, a head."""
    total = 0
    for _, nq, _, nk in _spans(case):
        if case["causal"]:
            first = nk - nq + 1  # keys of the first query, where that many are there
            total += sum(max(0, first + i) for i in range(nq)) if first < 1 else nq * first + nq * (nq - 1) // 2
        else:
            total += nq * nk
    return total


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    h, kv, d = case["heads"], case["kv"], case["d"]
    if case["op"] == "rotary":
        e = case["tokens"] * (h + kv) * d
        small = case["tokens"] * 4 * len(_ints(case["sections"]))
        # in and out, of the gradients too
        return {"bytes": es * e * (4 if case["step"] else 2) + small,
                "flops": e * (7 if case["norm"] else 3) * (3 if case["step"] else 1)}
    queries = sum(nq for _, nq, _, _ in _spans(case)) * h * d
    keys = 2 * sum(nk for _, _, _, nk in _spans(case)) * kv * d
    pairs = _pairs(case) * h
    if not case["step"]:
        return {"bytes": es * (2 * queries + keys), "flops": 4 * d * pairs}
    # backward: the scores again, dP, and the gradients of q, k and v
    return {"bytes": es * (4 * queries + 2 * keys), "flops": 14 * d * pairs}


# ------------------------------------------------------------------- exact


def exact(case, seed):
    st = prepare(case, seed)
    return _x_rot(case, st) if case["op"] == "rotary" else _x_attn(case, st)


def _x_attn(case, st):
    """Head by head and at most 1024 queries at a time, from the logarithm of the weights."""
    f64, g, scale = torch.float64, case["heads"] // case["kv"], 1.0 / math.sqrt(case["d"])
    new = lambda t: torch.zeros(t.shape, dtype=f64, device=DEVICE)  # noqa: E731
    out, dq, dk, dv = new(st["q"]), new(st["q"]), new(st["k"]), new(st["v"])
    for q0, nq, k0, nk in _spans(case):
        for h in range(case["heads"]):
            at = h // g, slice(k0, k0 + nk)
            k, v = st["k"][at].to(f64), st["v"][at].to(f64)
            for i0 in range(0, nq, 1024):
                i1 = min(nq, i0 + 1024)
                rows = h, slice(q0 + i0, q0 + i1)
                q = st["q"][rows].to(f64)
                s = (q @ k.T) * scale
                if case["causal"]:
                    own_place = torch.arange(i0, i1, device=DEVICE) + (nk - nq)
                    part = torch.arange(nk, device=DEVICE)[None] <= own_place[:, None]
                    s = torch.where(part, s, -math.inf)
                p = torch.nan_to_num((s - torch.logsumexp(s, -1, keepdim=True)).exp(), nan=0.0)
                out[rows] = p @ v
                if case["step"]:
                    do = st["dout"][rows].to(f64)
                    dp = do @ v.T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                    dq[rows] = scale * (ds @ k)
                    dk[at] += scale * (ds.T @ q)
                    dv[at] += p.T @ do
    return (out, dq, dk, dv) if case["step"] else out


def _x_rot(case, st):
    """The pairs as complex numbers, the gradients by differentiation."""
    f64 = torch.float64
    turn = []
    first = 0
    for axis, n in enumerate(_ints(case["sections"])):
        angle = st["positions"][axis].to(f64)[:, None] * st["frequencies"][None, first:first + n]
        turn.append(torch.polar(torch.ones_like(angle), angle))
        first += n
    turn = torch.cat(turn, -1)
    width = 2 * first
    outs, grads, weights = [], [], []
    for x, w, dy in ((st["q"], st["wq"], st["dq"]), (st["k"], st["wk"], st["dk"])):
        x = x.to(f64).contiguous().requires_grad_(case["step"])
        w = w.to(f64).requires_grad_(case["step"]) if case["norm"] else None
        y = x
        if case["norm"]:
            y = w * x / (x.square().sum(-1, keepdim=True) / case["d"] + 1e-6).sqrt()
        order = torch.arange(width, device=DEVICE)
        if not case["interleaved"]:  # pair i's members side by side
            order = order.view(2, -1).T.reshape(-1)
        z = torch.view_as_complex(y[..., order].unflatten(-1, (-1, 2)).contiguous()) * turn
        y = torch.cat([torch.view_as_real(z).flatten(-2)[..., torch.argsort(order)], y[..., width:]], -1)
        outs.append(y.detach())
        if case["step"]:
            got = torch.autograd.grad(y, [x] + ([w] if case["norm"] else []), dy.to(f64))
            grads.append(got[0])
            weights.extend(got[1:])
    return (*outs, *grads, *weights)
