"""Tensor-level entry points of the HIP triangle kernels.

Torch tensors are used only as device-memory handles: every call passes raw
device pointers, sizes and the current HIP stream through the C ABI of
``include/fjx_tri.h``. There is no other code path -- if the library is
missing, the call raises.

Weights are packed once into the PyTorch ``[out, in]`` layout of the ABI
(``TriMulWeights`` / ``TriAttnWeights``); ``foldjax_amd.params`` builds them
from each port's parameter containers.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, fields
from operator import attrgetter
from typing import ClassVar

import torch

from foldjax_amd import _lib

_DTYPES = {torch.float32: _lib.FJX_DTYPE_F32, torch.bfloat16: _lib.FJX_DTYPE_BF16}


def _code(dtype: torch.dtype) -> int:
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise ValueError(f"the hip triangle kernels take float32 or bfloat16, got {dtype}") from None


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _dev(x: torch.Tensor) -> None:
    if x.device.type != "cuda":
        raise ValueError(f"the hip backend needs device tensors, got a tensor on {x.device}")


def _stream(x: torch.Tensor) -> int:
    # torch.cuda.current_stream(x.device).cuda_stream without its Stream object
    return torch._C._cuda_getCurrentRawStream(x.get_device())


def _prep(t: torch.Tensor | None, dtype: torch.dtype, device) -> torch.Tensor | None:
    if t is None:
        return None
    return t.to(device=device, dtype=dtype).contiguous()


def _same_device(x: torch.Tensor, **operands) -> None:
    """Every operand must live on ``x``'s device: a host tensor's pointer
    handed to a kernel would be read as device memory."""
    for name, t in operands.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device} but the input is on {x.device}; "
                             "every operand must be on the input's device")


def _need_shape(name: str, t: torch.Tensor | None, shape) -> None:
    if t is not None and t.shape != shape and tuple(t.shape) != tuple(int(v) for v in shape):
        raise ValueError(f"{name} must have shape {tuple(int(v) for v in shape)}, got {tuple(t.shape)}")


def _shaped(*pairs) -> bool:
    """Every tensor there and of its shape: the usual case, without a message made."""
    for t, shape in pairs:
        if t is None or t.shape != shape:
            return False
    return True


def _rows_of(m: torch.Tensor | None, shape, dtype: torch.dtype, name: str) -> torch.Tensor | None:
    """A per-row (per-position) mask broadcast to ``shape`` in ``dtype``,
    contiguous, as the kernels index it."""
    if m is None or (m.shape == shape and m.dtype is dtype and m.is_contiguous()):
        return m
    try:
        m = torch.broadcast_to(m, tuple(shape))
    except RuntimeError:
        raise ValueError(f"{name} of shape {tuple(m.shape)} does not broadcast to {tuple(shape)}") from None
    return m.to(dtype=dtype).contiguous()


@dataclass(frozen=True)
class TriMulWeights:
    """Tri-mul weights in the ABI layout (PyTorch ``[out, in]``, a rows first)."""

    norm_in_weight: torch.Tensor  # [c_z]
    norm_in_bias: torch.Tensor  # [c_z]
    p_in_weight: torch.Tensor  # [2 c_h, c_z]
    g_in_weight: torch.Tensor  # [2 c_h, c_z]
    norm_out_weight: torch.Tensor  # [c_h]
    norm_out_bias: torch.Tensor  # [c_h]
    p_out_weight: torch.Tensor  # [c_z, c_h]
    g_out_weight: torch.Tensor  # [c_z, c_z]

    def to(self, dtype: torch.dtype, device) -> "TriMulWeights":
        return TriMulWeights(**{f.name: _prep(getattr(self, f.name), dtype, device) for f in fields(self)})

    def check(self, c_z: int) -> int:
        """Shapes against the pair width ``c_z``; returns ``c_h``."""
        c_h = int(self.norm_out_weight.shape[0])
        in_, proj = (c_z,), (2 * c_h, c_z)
        if _shaped((self.norm_in_weight, in_), (self.norm_in_bias, in_), (self.p_in_weight, proj),
                   (self.g_in_weight, proj), (self.norm_out_bias, (c_h,)), (self.p_out_weight, (c_z, c_h)),
                   (self.g_out_weight, (c_z, c_z))):
            return c_h
        for name, shape in (("norm_in_weight", (c_z,)), ("norm_in_bias", (c_z,)), ("p_in_weight", (2 * c_h, c_z)),
                            ("g_in_weight", (2 * c_h, c_z)), ("norm_out_bias", (c_h,)), ("p_out_weight", (c_z, c_h)),
                            ("g_out_weight", (c_z, c_z))):
            _need_shape(f"tri-mul weight {name}", getattr(self, name), shape)
        return c_h


@dataclass(frozen=True)
class TriAttnWeights:
    """Tri-attn weights in the ABI layout (PyTorch ``[out, in]``)."""

    norm_weight: torch.Tensor  # [c_z]
    norm_bias: torch.Tensor  # [c_z]
    bias_weight: torch.Tensor  # [H, c_z]
    q_weight: torch.Tensor  # [H D, c_z]
    k_weight: torch.Tensor
    v_weight: torch.Tensor
    g_weight: torch.Tensor | None  # [H D, c_z] or None (ungated)
    o_weight: torch.Tensor  # [c_z, H D]

    @property
    def heads(self) -> int:
        return int(self.bias_weight.shape[0])

    def to(self, dtype: torch.dtype, device) -> "TriAttnWeights":
        return TriAttnWeights(**{f.name: _prep(getattr(self, f.name), dtype, device) for f in fields(self)})

    def check(self, c_z: int) -> int:
        """Shapes against the pair width ``c_z``; returns ``heads * head_dim``."""
        hd = int(self.q_weight.shape[0])
        if hd % self.heads:
            raise ValueError(f"q projection width {hd} is not divisible by {self.heads} heads")
        in_, proj = (c_z,), (hd, c_z)
        if _shaped((self.norm_weight, in_), (self.norm_bias, in_), (self.bias_weight, (self.heads, c_z)),
                   (self.q_weight, proj), (self.k_weight, proj), (self.v_weight, proj), (self.o_weight, (c_z, hd))
                   ) and (self.g_weight is None or self.g_weight.shape == proj):
            return hd
        for name, shape in (("norm_weight", (c_z,)), ("norm_bias", (c_z,)), ("bias_weight", (self.heads, c_z)),
                            ("q_weight", (hd, c_z)), ("k_weight", (hd, c_z)), ("v_weight", (hd, c_z)),
                            ("g_weight", (hd, c_z)), ("o_weight", (c_z, hd))):
            _need_shape(f"tri-attn weight {name}", getattr(self, name), shape)
        return hd


@dataclass(frozen=True)
class TransitionWeights:
    """Transition weights, PyTorch ``[out, in]``: ``w_a``/``w_b`` ``[hidden, c]``
    (silu and linear branches), ``w_o`` ``[c, hidden]``; hidden is 4c in every
    port."""

    norm_weight: torch.Tensor
    norm_bias: torch.Tensor
    w_a: torch.Tensor
    w_b: torch.Tensor
    w_o: torch.Tensor

    def to(self, dtype: torch.dtype, device) -> "TransitionWeights":
        return TransitionWeights(**{f.name: _prep(getattr(self, f.name), dtype, device) for f in fields(self)})

    def check(self, c: int) -> int:
        """Shapes against the width ``c``; returns the hidden width."""
        hidden = int(self.w_a.shape[0])
        if _shaped((self.norm_weight, (c,)), (self.norm_bias, (c,)), (self.w_a, (hidden, c)),
                   (self.w_b, (hidden, c)), (self.w_o, (c, hidden))):
            return hidden
        for name, shape in (("norm_weight", (c,)), ("norm_bias", (c,)), ("w_a", (hidden, c)), ("w_b", (hidden, c)),
                            ("w_o", (c, hidden))):
            _need_shape(f"transition weight {name}", getattr(self, name), shape)
        return hidden


@dataclass(frozen=True)
class SingleAttentionWeights:
    """Boltz-2 ``AttentionPairBias`` weights (PyTorch ``[out, in]``) plus the
    layer's ``pre_norm_s`` (None when the caller passes a normalised s)."""

    # fields a packed layer keeps back to back in one buffer (one projection
    # GEMM); stacking layers keeps them so (foldjax_amd.stacking)
    STACK_GROUPS: ClassVar[tuple[tuple[str, ...], ...]] = (("q_weight", "k_weight", "v_weight", "g_weight"),)

    pre_norm_weight: torch.Tensor | None
    pre_norm_bias: torch.Tensor | None
    z_norm_weight: torch.Tensor  # [c_z]
    z_norm_bias: torch.Tensor
    z_weight: torch.Tensor  # [H, c_z]
    q_weight: torch.Tensor  # [c_s, c_s]
    q_bias: torch.Tensor | None  # [c_s]
    k_weight: torch.Tensor
    v_weight: torch.Tensor
    g_weight: torch.Tensor
    o_weight: torch.Tensor

    @property
    def heads(self) -> int:
        return int(self.z_weight.shape[0])

    def to(self, dtype: torch.dtype, device) -> "SingleAttentionWeights":
        """Each weight in ``dtype`` on ``device``; q, k, v and g are stored back
        to back in one ``[4 c_s, c_s]`` buffer (the library then runs their four
        projections as one GEMM)."""
        f = {fl.name: _prep(getattr(self, fl.name), dtype, device) for fl in fields(self)}
        parts = [f[k] for k in ("q_weight", "k_weight", "v_weight", "g_weight")]
        if len({tuple(t.shape) for t in parts}) == 1:
            qkvg = torch.cat(parts, 0)
            f["q_weight"], f["k_weight"], f["v_weight"], f["g_weight"] = qkvg.chunk(4, 0)
        return SingleAttentionWeights(**f)

    def check(self, c_s: int, c_z: int | None) -> None:
        """Shapes against the single width ``c_s`` and (when z is read) the
        pair width ``c_z``."""
        sq = (c_s, c_s)
        if not _shaped((self.q_weight, sq), (self.k_weight, sq), (self.v_weight, sq), (self.g_weight, sq),
                       (self.o_weight, sq)):
            for name in ("q_weight", "k_weight", "v_weight", "g_weight", "o_weight"):
                _need_shape(f"single attention weight {name}", getattr(self, name), sq)
        for name in ("q_bias", "pre_norm_weight", "pre_norm_bias"):
            _need_shape(f"single attention weight {name}", getattr(self, name), (c_s,))
        if c_z is not None:
            for name, shape in (("z_norm_weight", (c_z,)), ("z_norm_bias", (c_z,)), ("z_weight", (self.heads, c_z))):
                _need_shape(f"single attention weight {name}", getattr(self, name), shape)


# per packed weight class, a getter of every field as one tuple
_TENSORS: dict = {}


def _tensors(w) -> tuple:
    get = _TENSORS.get(type(w))
    if get is None:
        get = _TENSORS[type(w)] = attrgetter(*(f.name for f in fields(w)))
    return get(w)


def _like(t: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor | None:
    """``t`` in ``dtype`` and contiguous."""
    if t is None or (t.dtype is dtype and t.is_contiguous()):
        return t
    return t.to(dtype=dtype).contiguous()


def transition(
    x: torch.Tensor,
    w: TransitionWeights,
    *,
    row_mask: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    eps: float = 1e-5,
    pair_bias_for: SingleAttentionWeights | None = None,
    pair_bias_eps: float = 1e-5,
    out_mask: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
):
    """``((silu(LN(x) w_a^T) * (LN(x) w_b^T)) w_o^T [* row_mask] [+ residual])
    [* (out_mask != 0)]`` over the last axis (``fjx_transition_fwd``);
    ``row_mask`` and ``out_mask`` broadcast to ``x.shape[:-1]``.

    ``pair_bias_for``: the weights of the single attention that reads this
    pair transition's output next (``x`` is then ``[..., N, N, 128]``). The
    call returns ``(out, pair_bias)``, ``pair_bias`` being that attention's
    bias ``LN_z(out) w_z^T`` (eps ``pair_bias_eps``) prepared in the
    library's ``[B, H, Np, Np]`` layout, for ``single_attention(...,
    pair_bias=...)``; with 128 channels, a 4x hidden width and at most 16
    heads it is computed in the transition's epilogue, so the pair tensor is
    not read again. The bias takes the attention's dtype: a float32
    attention over a bfloat16 pair track gets a float32 bias computed to
    float32 accuracy.

    ``out``: write the result into this tensor (x's shape, dtype and device,
    contiguous) instead of a new one; it may be ``x`` and/or ``residual``
    (in place)."""
    c = int(x.shape[-1])
    w.check(c)
    _same_device(x, row_mask=row_mask, residual=residual, out_mask=out_mask)
    if residual is not None:
        _need_shape("residual", residual, x.shape)
    if pair_bias_for is not None:
        _same_device(x, pair_bias_for=pair_bias_for.z_weight)
        _need_shape("pair-bias weight z_norm_weight", pair_bias_for.z_norm_weight, (c,))
        _need_shape("pair-bias weight z_norm_bias", pair_bias_for.z_norm_bias, (c,))
        _need_shape("pair-bias weight z_weight", pair_bias_for.z_weight, (pair_bias_for.heads, c))
    _dev(x)
    rows = x.numel() // max(c, 1)
    xf = x.contiguous()
    lib = _lib.load()
    out = _out_buffer(out, x, xf)
    pb = None
    pb_n = pb_heads = 0
    pb_f32 = False
    if pair_bias_for is not None:
        if x.dim() < 3 or x.shape[-3] != x.shape[-2]:
            raise ValueError(f"a pair-bias output needs a pair tensor [..., N, N, C], got {tuple(x.shape)}")
        pb_dtype = pair_bias_for.z_weight.dtype
        pb_f32 = pb_dtype == torch.float32 and x.dtype == torch.bfloat16
        if pb_dtype != x.dtype and not pb_f32:
            raise ValueError(f"a {pb_dtype} pair bias over a {x.dtype} transition is not supported")
        pb_n, pb_heads = int(x.shape[-2]), pair_bias_for.heads
        np_ = (pb_n + 63) // 64 * 64
        pb = torch.empty((rows // (pb_n * pb_n), pb_heads, np_, np_), dtype=pb_dtype, device=x.device)
    rm = _rows_of(row_mask, x.shape[:-1], x.dtype, "row_mask")
    om = _rows_of(out_mask, x.shape[:-1], x.dtype, "out_mask")
    res = _like(residual, x.dtype)
    hidden = int(w.w_a.shape[0])
    ws_bytes = lib.fjx_transition_workspace_size(rows, c, hidden, _code(x.dtype))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    a = _lib.TransitionArgs(
        rows=rows, c=c, dtype=_code(x.dtype), eps=float(eps),
        x=_ptr(xf), norm_weight=_ptr(w.norm_weight), norm_bias=_ptr(w.norm_bias),
        w_a=_ptr(w.w_a), w_b=_ptr(w.w_b), w_o=_ptr(w.w_o),
        row_mask=_ptr(rm), residual=_ptr(res), out=_ptr(out),
        hidden=hidden, workspace=_ptr(ws), workspace_bytes=ws_bytes, out_mask=_ptr(om),
    )
    if pb is not None:
        a.pb_n, a.pb_heads, a.pb_eps = pb_n, pb_heads, float(pair_bias_eps)
        a.pb_norm_weight = _ptr(pair_bias_for.z_norm_weight)
        a.pb_norm_bias = _ptr(pair_bias_for.z_norm_bias)
        a.pb_weight = _ptr(pair_bias_for.z_weight)
        a.pb_out = _ptr(pb)
        a.pb_f32 = 1 if pb_f32 else 0
        _check_weights(pb, pair_bias_for)
    _check_weights(x, w)
    _lib.check(lib.fjx_transition_fwd(ctypes.byref(a), _stream(x)))
    return out if pb is None else (out, pb)


def single_attention(
    s: torch.Tensor,
    z: torch.Tensor | None,
    mask: torch.Tensor | None,
    w: SingleAttentionWeights,
    *,
    inf: float = 1e6,
    eps: float = 1e-5,
    residual: torch.Tensor | None = None,
    pair_bias: torch.Tensor | None = None,
    out_mask: torch.Tensor | None = None,
    extra_bias: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Single-track attention with pair bias (``fjx_single_attention_fwd``).
    ``s`` ``[B, N, c_s]`` (or ``[N, c_s]``), ``z`` ``[B, N, N, c_z]``, ``mask``
    ``[B, N]`` token mask. Returns the update, or ``residual + update``, times
    ``out_mask != 0`` per row when ``out_mask`` (``[B, N]``) is given.
    ``s`` and the weights share one dtype; ``z`` may be float32 or bfloat16
    independently (the Boltz-2 single track runs in float32 over a bfloat16
    pair tensor). ``pair_bias``: the bias ``transition(..., pair_bias_for=w)``
    prepared from this ``z`` in ``s``'s dtype; ``z`` is then not read (and may
    be None). ``extra_bias``: an additive bias broadcasting to ``[B, H, N, N]``
    from a 4-D tensor whose last two axes are ``[N, N]`` (Protenix's
    ``extra_attn_bias``). ``out``: write the result into this tensor (s's
    shape, dtype and device, contiguous); it may be ``s`` when ``residual`` is
    ``s`` (in place)."""
    _same_device(s, z=z, mask=mask, residual=residual, pair_bias=pair_bias, out_mask=out_mask,
                 extra_bias=extra_bias)
    if residual is not None:
        _need_shape("residual", residual, s.shape)
    w.check(int(s.shape[-1]), None if z is None else int(z.shape[-1]))
    squeeze = s.dim() == 2
    sb = s.unsqueeze(0) if squeeze else s
    batch, n, c_s = (int(v) for v in sb.shape)
    zb = None
    c_z = 0
    if z is not None:
        zb = z.unsqueeze(0) if z.dim() == 3 else z
        c_z = int(zb.shape[-1])
        if tuple(zb.shape[:3]) != (batch, n, n):
            raise ValueError(f"z must be [{batch}, {n}, {n}, c_z], got {tuple(z.shape)}")
        _code(zb.dtype)
        zb = zb.contiguous()
    if pair_bias is not None:
        np_ = (n + 63) // 64 * 64
        if (tuple(pair_bias.shape) != (batch, w.heads, np_, np_) or pair_bias.dtype != s.dtype
                or pair_bias.device != s.device or not pair_bias.is_contiguous()):
            raise ValueError(f"pair_bias must be the prepared [{batch}, {w.heads}, {np_}, {np_}] {s.dtype} bias, "
                             f"got {tuple(pair_bias.shape)} {pair_bias.dtype}")
    elif zb is None:
        raise ValueError("single_attention needs z or a prepared pair_bias")
    sb = sb.contiguous()
    mb = _rows_of(mask, (batch, n), s.dtype, "mask")
    om = _rows_of(out_mask, (batch, n), s.dtype, "out_mask")
    eb, eb_sb, eb_sh = None, 0, 0
    if extra_bias is not None:
        if extra_bias.dim() != 4 or tuple(extra_bias.shape[-2:]) != (n, n):
            raise ValueError(f"extra_bias must be a 4-D tensor [B or 1, H or 1, {n}, {n}], got {tuple(extra_bias.shape)}")
        eb = extra_bias.to(dtype=s.dtype)
        if eb.stride(-1) != 1 or eb.stride(-2) != n:
            eb = eb.contiguous()
        try:
            eb = torch.broadcast_to(eb, (batch, w.heads, n, n))
        except RuntimeError:
            raise ValueError(f"extra_bias of shape {tuple(extra_bias.shape)} does not broadcast to "
                             f"[{batch}, {w.heads}, {n}, {n}]") from None
        eb_sb, eb_sh = int(eb.stride(0)), int(eb.stride(1))
    _dev(s)
    res = None
    if residual is not None:
        res = _like(residual, s.dtype)
    lib = _lib.load()
    code = _code(s.dtype)
    if out is not None and out.data_ptr() == s.data_ptr() and (residual is None or residual.data_ptr() != s.data_ptr()):
        raise ValueError("out may be s only when residual is s")
    out = _out_buffer(out, s, sb)
    ws_bytes = lib.fjx_single_attention_workspace_size(batch, n, c_s, w.heads, code)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=s.device)
    a = _lib.SingleAttentionArgs(
        batch=batch, n=n, c_s=c_s, c_z=c_z, heads=w.heads, dtype=code, eps=float(eps), inf=float(inf),
        s=_ptr(sb), z=_ptr(zb), mask=_ptr(mb),
        pre_norm_weight=_ptr(w.pre_norm_weight), pre_norm_bias=_ptr(w.pre_norm_bias),
        z_norm_weight=_ptr(w.z_norm_weight), z_norm_bias=_ptr(w.z_norm_bias), z_weight=_ptr(w.z_weight),
        q_weight=_ptr(w.q_weight), q_bias=_ptr(w.q_bias), k_weight=_ptr(w.k_weight), v_weight=_ptr(w.v_weight),
        g_weight=_ptr(w.g_weight), o_weight=_ptr(w.o_weight),
        residual=_ptr(res), out=_ptr(out), workspace=_ptr(ws), workspace_bytes=ws_bytes,
        pair_bias=_ptr(pair_bias), z_dtype=_code(s.dtype if zb is None else zb.dtype), out_mask=_ptr(om),
        extra_bias=_ptr(eb), extra_bias_stride_b=eb_sb, extra_bias_stride_h=eb_sh,
    )
    _check_weights(s, w)
    _lib.check(lib.fjx_single_attention_fwd(ctypes.byref(a), _stream(s)))
    return out[0] if squeeze else out


def _out_buffer(out: torch.Tensor | None, x: torch.Tensor, flat: torch.Tensor) -> torch.Tensor:
    """The output buffer of a call on ``x`` (flattened as ``flat``): a new
    tensor, or the caller's ``out``, which must be a contiguous tensor of x's
    shape, dtype and device and may be x itself and/or the residual (every
    kernel reads an output position's inputs before it writes it, and only
    the workgroup that writes a position reads it)."""
    if out is None:
        return torch.empty_like(flat)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"out must be a {x.dtype} tensor of shape {tuple(x.shape)} on {x.device}, "
                         f"got {out.dtype} {tuple(out.shape)} on {out.device}")
    if not out.is_contiguous():
        raise ValueError("out must be contiguous")
    return out if out.shape == flat.shape else out.reshape(flat.shape)


def _flatten_pair(x: torch.Tensor, mask: torch.Tensor | None):
    if x.dim() < 3:
        raise ValueError(f"pair tensor must be [..., N, N, C], got shape {tuple(x.shape)}")
    _same_device(x, mask=mask)
    if x.dim() == 4 and x.is_contiguous() and (mask is None or (mask.shape == x.shape[:3] and mask.dtype is x.dtype
                                                                and mask.is_contiguous())):
        batch, n, n2, c = x.shape
        if n == n2:
            return x, mask, (batch,), batch, n, c
    n, n2, c = x.shape[-3:]
    if n != n2:
        raise ValueError(f"pair tensor must be square in its two pair axes, got {tuple(x.shape)}")
    lead = x.shape[:-3]
    batch = 1
    for s in lead:
        batch *= int(s)
    xf = x.contiguous().reshape(batch, n, n, c)
    mf = None
    if mask is not None:
        if tuple(mask.shape[-2:]) != (n, n):
            raise ValueError(f"mask must be [..., {n}, {n}], got {tuple(mask.shape)}")
        mf = torch.broadcast_to(mask, tuple(lead) + (n, n)).to(dtype=x.dtype).contiguous().reshape(batch, n, n)
    return xf, mf, lead, batch, n, c


def trimul(
    x: torch.Tensor,
    mask: torch.Tensor | None,
    w: TriMulWeights,
    direction: str,
    eps: float = 1e-5,
    residual: torch.Tensor | None = None,
    *,
    no_alloc: bool = False,
    out_mask: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Triangle multiplicative update (``fjx_trimul_fwd``); returns the update,
    or ``residual + update`` when ``residual`` is given, times
    ``out_mask != 0`` per position when ``out_mask`` (``[..., N, N]``) is given.

    ``no_alloc``: run ``fjx_trimul_fwd_noalloc`` instead, whose workspace is
    the library's static per-GPU scratch (shapes up to 256 MiB of unpadded
    workspace; calls on one GPU must not overlap). Only the output is allocated
    here, unless ``out`` is given: the result then goes into that tensor (x's
    shape, dtype and device, contiguous), which may be ``x`` and/or
    ``residual`` (in place)."""
    if direction not in ("outgoing", "incoming"):
        raise ValueError(f"Unsupported triangle multiplication direction: {direction!r}")
    _same_device(x, residual=residual, out_mask=out_mask)
    if residual is not None:
        _need_shape("residual", residual, x.shape)
    c_h = w.check(int(x.shape[-1]))
    xf, mf, lead, batch, n, c = _flatten_pair(x, mask)
    om = _rows_of(out_mask, x.shape[:-1], x.dtype, "out_mask")
    _dev(x)
    lib = _lib.load()
    code = _code(x.dtype)
    out = _out_buffer(out, x, xf)
    res = _like(residual, x.dtype)
    ws_bytes = 0 if no_alloc else lib.fjx_trimul_workspace_size(batch, n, c, c_h, code)
    try:
        ws = None if no_alloc else torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=x.device)
    except torch.OutOfMemoryError:
        # a, b and o unpadded and unsplit: slower, but all that a call needs
        least = 3 * ((batch * n * n * c_h * x.element_size() + 255) // 256 * 256)
        if c_h != 128 or c not in (32, 64, 96, 128) or least >= ws_bytes:
            raise
        ws_bytes = least
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
    a = _lib.TriMulArgs(
        batch=batch, n=n, c_z=c, c_h=c_h,
        direction=_lib.FJX_OUTGOING if direction == "outgoing" else _lib.FJX_INCOMING,
        dtype=code, eps=float(eps),
        x=_ptr(xf), mask=_ptr(mf),
        norm_in_weight=_ptr(w.norm_in_weight), norm_in_bias=_ptr(w.norm_in_bias),
        p_in_weight=_ptr(w.p_in_weight), g_in_weight=_ptr(w.g_in_weight),
        norm_out_weight=_ptr(w.norm_out_weight), norm_out_bias=_ptr(w.norm_out_bias),
        p_out_weight=_ptr(w.p_out_weight), g_out_weight=_ptr(w.g_out_weight),
        residual=_ptr(res), out=_ptr(out),
        workspace=_ptr(ws), workspace_bytes=ws_bytes, out_mask=_ptr(om),
    )
    _check_weights(x, w)
    entry = lib.fjx_trimul_fwd_noalloc if no_alloc else lib.fjx_trimul_fwd
    _lib.check(entry(ctypes.byref(a), _stream(x)))
    return out if len(lead) == 1 else out.reshape(tuple(lead) + (n, n, c))


def triattn(
    x: torch.Tensor,
    mask: torch.Tensor | None,
    w: TriAttnWeights,
    starting: bool = True,
    inf: float = 1e9,
    eps: float = 1e-5,
    residual: torch.Tensor | None = None,
    out_mask: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Triangle attention, starting or ending node (``fjx_triattn_fwd``);
    ``out_mask`` (``[..., N, N]``, indexed like the output) and ``out`` (may
    be ``x`` and/or ``residual``: in place) as for ``trimul``."""
    _same_device(x, residual=residual, out_mask=out_mask)
    if residual is not None:
        _need_shape("residual", residual, x.shape)
    hd = w.check(int(x.shape[-1]))
    heads = w.heads
    xf, mf, lead, batch, n, c = _flatten_pair(x, mask)
    om = _rows_of(out_mask, x.shape[:-1], x.dtype, "out_mask")
    _dev(x)
    lib = _lib.load()
    code = _code(x.dtype)
    out = _out_buffer(out, x, xf)
    res = _like(residual, x.dtype)
    ws_bytes = lib.fjx_triattn_workspace_size(batch, n, c, heads, hd // heads, code)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=x.device)
    a = _lib.TriAttnArgs(
        batch=batch, n=n, c_z=c, heads=heads, head_dim=hd // heads,
        starting=1 if starting else 0, dtype=code, eps=float(eps), inf=float(inf),
        x=_ptr(xf), mask=_ptr(mf),
        norm_weight=_ptr(w.norm_weight), norm_bias=_ptr(w.norm_bias), bias_weight=_ptr(w.bias_weight),
        q_weight=_ptr(w.q_weight), k_weight=_ptr(w.k_weight), v_weight=_ptr(w.v_weight),
        g_weight=_ptr(w.g_weight), o_weight=_ptr(w.o_weight),
        residual=_ptr(res), out=_ptr(out),
        workspace=_ptr(ws), workspace_bytes=ws_bytes, out_mask=_ptr(om),
    )
    _check_weights(x, w)
    _lib.check(lib.fjx_triattn_fwd(ctypes.byref(a), _stream(x)))
    return out if len(lead) == 1 else out.reshape(tuple(lead) + (n, n, c))


def triattn_core(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    tri_bias: torch.Tensor,
    mask_bias: torch.Tensor | None,
    *,
    scale: float,
) -> torch.Tensor:
    """``cueq_attention_core`` semantics (``src/foldjax/models/_cueq.py:66-121``).

    q/k/v ``[..., I, H, J, D]``; ``tri_bias`` ``[..., 1, H, J, J]``; additive
    ``mask_bias`` ``[..., I, 1, 1, J]`` (or None); ``scale`` applied inside.
    Leading axes are broadcast and folded into one batch axis.
    """
    _same_device(q, k=k, v=v, tri_bias=tri_bias, mask_bias=mask_bias)
    if q.dim() < 4 or k.shape[-4:] != q.shape[-4:] or v.shape[-4:] != q.shape[-4:]:
        raise ValueError(f"q, k, v must share [..., I, H, J, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if tri_bias.dim() < 4 or tuple(tri_bias.shape[-3:]) != (q.shape[-3], q.shape[-2], q.shape[-2]):
        raise ValueError(f"tri_bias must be [..., 1, H, J, J] for q {tuple(q.shape)}, got {tuple(tri_bias.shape)}")
    if mask_bias is not None and (mask_bias.dim() < 4 or tuple(mask_bias.shape[-4:]) not in
                                  ((q.shape[-4], 1, 1, q.shape[-2]), (1, 1, 1, q.shape[-2]))):
        raise ValueError(f"mask_bias must be [..., I, 1, 1, J] for q {tuple(q.shape)}, got {tuple(mask_bias.shape)}")
    _dev(q)
    lead = torch.broadcast_shapes(q.shape[:-4], tri_bias.shape[:-4],
                                  () if mask_bias is None else mask_bias.shape[:-4])
    rows, heads, n, d = q.shape[-4:]
    batch = 1
    for s in lead:
        batch *= int(s)
    dt = q.dtype

    def fold(t, shape):
        return torch.broadcast_to(t, tuple(lead) + tuple(shape)).to(dtype=dt).contiguous().reshape((batch,) + tuple(shape))

    qf = fold(q, (rows, heads, n, d))
    kf = fold(k, (rows, heads, n, d))
    vf = fold(v, (rows, heads, n, d))
    if tri_bias.shape[-4] != 1:
        raise ValueError("tri_bias must be [..., 1, H, J, J]: the kernel shares one bias across rows")
    bf = fold(tri_bias, (1, heads, n, n)).reshape(batch, heads, n, n)
    mb = None
    if mask_bias is not None:
        mb = torch.broadcast_to(mask_bias, tuple(lead) + (rows, 1, 1, n)).to(torch.float32).contiguous()
        mb = mb.reshape(batch, rows, n)
    lib = _lib.load()
    code = _code(dt)
    out = torch.empty_like(qf)
    ws_bytes = lib.fjx_triattn_core_workspace_size(batch, rows, heads, n, d, code)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=q.device)
    a = _lib.TriAttnCoreArgs(
        batch=batch, rows=rows, heads=heads, n=n, head_dim=d, dtype=code, scale=float(scale),
        q=_ptr(qf), k=_ptr(kf), v=_ptr(vf), tri_bias=_ptr(bf), mask_bias=_ptr(mb),
        out=_ptr(out), workspace=_ptr(ws), workspace_bytes=ws_bytes,
    )
    _lib.check(lib.fjx_triattn_core(ctypes.byref(a), _stream(q)))
    return out.reshape(tuple(lead) + (rows, heads, n, d))


def _launch(entry, args, x: torch.Tensor) -> None:
    """``entry`` on the current stream of ``x``'s device, whichever device is
    the current one."""
    dev = x.get_device()
    if torch._C._cuda_getDevice() == dev:  # torch.cuda.current_device without its lazy start: x is there already
        rc = entry(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = entry(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc)


def _need_dtype(dtype: torch.dtype, **operands) -> None:
    for name, t in operands.items():
        if t is not None and t.dtype is not dtype:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}")


def _same_place(x: torch.Tensor, dtype: torch.dtype, **operands) -> None:
    """Every operand there on ``x``'s device and of ``dtype``."""
    dev = x.get_device()
    for name, t in operands.items():
        if t is not None and (t.dtype is not dtype or t.get_device() != dev):
            _same_device(x, **{name: t})
            _need_dtype(dtype, **{name: t})


def _folded(shape, strides):
    """The stride of the axes taken as one, 0 for one element; None where they
    do not fold."""
    step, count = 0, 1
    for n, s in zip(reversed(shape), reversed(strides)):
        if n == 1:
            continue
        if s != step * count if count > 1 else s == 0:
            return None
        if count == 1:
            step = s
        count *= n
    return step


def _head_rows(t: torch.Tensor, unit: int):
    """Strides {item, head, token} of [..., heads, tokens, width] (0 for an
    axis of one element), where the kernels can take its rows as they lie, whole
    16-byte pieces of ``unit`` elements; None where not."""
    shape, strides = t.shape, t.stride()
    item = _folded(shape[:-3], strides[:-3])
    if item is None or strides[-1] != 1 or t.data_ptr() & 15:
        return None
    head = strides[-3] if shape[-3] > 1 else 0
    token = strides[-2] if shape[-2] > 1 else 0
    if (item | head | token) % unit or (head == 0 and shape[-3] > 1) or (token == 0 and shape[-2] > 1):
        return None
    return item, head, token


def _heads(t: torch.Tensor, unit: int):
    """``t`` and its strides, a copy where its rows cannot be taken as they lie."""
    st = _head_rows(t, unit)
    if st is None:
        t = t.clone(memory_format=torch.contiguous_format)
        st = _head_rows(t, unit)
    return t, st


def _packed(shape):
    """Strides {item, head, token} of a contiguous [..., heads, tokens, width]."""
    width, tokens = shape[-1], shape[-2]
    return shape[-3] * tokens * width, tokens * width, width


# argument blocks of the layouts seen (shapes, strides, types, devices) whose
# tensors were taken as they lay: a call with the same layout sets the pointers
_BLOCKS: dict = {}


def _layout(*tensors):
    return tuple([None if t is None else (t.dtype, t.get_device(), t.shape, t.stride()) for t in tensors])


def _remember(key, value) -> None:
    if len(_BLOCKS) >= 512:
        _BLOCKS.clear()
    _BLOCKS[key] = value


def _diff_attention_args(q, k, v, lambda_vectors, lambda_init, scale, bias, mask):
    """The checked argument block that both directions share (its out strides
    those of a contiguous output), the tensors it points to, the output's shape
    and strides, the elements of a 16-byte piece, and (its key, the workspace of
    the forward call)."""
    lambda_init, scale = float(lambda_init), float(scale)  # values, also of tensors: they are part of the key
    key = (_layout(q, k, v, lambda_vectors, bias, mask), lambda_init, scale)
    seen = _BLOCKS.get(key)
    if seen is not None:
        block, shaped, unit, nbytes = seen
        a = _lib.DiffAttentionArgs.from_buffer_copy(block)
        a.q, a.k, a.v, a.lambda_vectors = qp, kp, vp, lp = q.data_ptr(), k.data_ptr(), v.data_ptr(), lambda_vectors.data_ptr()
        if not (qp | kp | vp | lp) & 15:
            if bias is not None:
                a.bias = bias.data_ptr()
            if mask is not None:
                a.mask = mask.data_ptr()
            return a, (q, k, v, bias, mask, lambda_vectors), shaped, unit, (key, nbytes)
    given = (q, k, v, bias, mask, lambda_vectors)
    dtype = q.dtype
    code = _code(dtype)
    _same_place(q, dtype, k=k, v=v, bias=bias)
    _same_place(q, torch.float32, lambda_vectors=lambda_vectors)
    _same_device(q, mask=mask)
    qs, ks = q.shape, k.shape
    if len(qs) < 3 or len(ks) != len(qs) or v.dim() != len(qs):
        raise ValueError(f"q, k and v must be [..., heads, tokens, width] of as many axes, got {tuple(qs)}, "
                         f"{tuple(ks)}, {tuple(v.shape)}")
    lead = tuple(qs[:-3])
    h2, nq, d = qs[-3:]
    hk2, nk = ks[-3], ks[-2]
    if h2 % 2 or hk2 % 2:
        raise ValueError(f"q and k hold two maps a head: an even number of heads, got {h2} and {hk2}")
    heads, kv_heads = h2 // 2, hk2 // 2
    _need_shape("k", k, lead + (hk2, nk, d))
    _need_shape("v", v, lead + (kv_heads, nk, 2 * d))
    _need_shape("lambda_vectors", lambda_vectors, (4, heads, d))
    if d not in (32, 64):
        raise ValueError(f"q and k must have a width (head_dim) of 32 or 64, got {d}")
    unit = 4 if dtype is torch.float32 else 8
    items = 1
    for n in lead:
        items *= n
    lam = lambda_vectors
    if not lam.is_contiguous() or lam.data_ptr() & 15:
        lam = lam.clone(memory_format=torch.contiguous_format)
    bp, bst, share = None, (0, 0, 0), 1
    if bias is not None:
        bs = bias.shape
        if not 3 <= len(bs) <= len(qs) or bs[-1] != nk or bs[-2] != nq or bs[-3] != heads:
            raise ValueError(f"bias must be [..., {heads}, {nq}, {nk}], got {tuple(bs)}")
        # planes for the leading items, then axes that share one
        planes = (1,) * (len(qs) - len(bs)) + tuple(bs[:-3])
        axis = len(lead)
        while axis and planes[axis - 1] == 1:
            axis -= 1
            share *= lead[axis]
        if planes[:axis] != lead[:axis]:
            raise ValueError(f"bias must have one plane for each of q's leading axes {lead}, or share one over the last "
                             f"of them, got {tuple(bs[:-3])}")
        bst = bias.stride()
        plane = _folded(bs[:-3], bst[:-3])
        if plane is None or (bst[-1] != 1 and nk > 1) or min(bst) < 0:
            bias = bias.contiguous()
            bst = bias.stride()
            plane = heads * nq * nk
        bp, bst = bias.data_ptr(), (plane, bst[-3], bst[-2])
    m2 = None
    if mask is not None:
        if mask.shape != lead + (nk,):
            try:
                mask = torch.broadcast_to(mask, lead + (nk,))
            except RuntimeError:
                raise ValueError(f"mask of shape {tuple(mask.shape)} does not broadcast to {lead + (nk,)}") from None
        m2 = (mask if mask.dtype is torch.bool else mask.ne(0)).contiguous()
    _dev(q)
    q, qst = _heads(q, unit)
    k, kst = _heads(k, unit)
    v, vst = _heads(v, unit)
    shape = lead + (heads, nq, 2 * d)
    packed = _packed(shape)
    a = _lib.DiffAttentionArgs(
        items, heads, kv_heads, nq, nk, d, share, code, scale, lambda_init, q.data_ptr(), k.data_ptr(), v.data_ptr(), None,
        qst, kst, vst, packed, bp, bst, None if m2 is None else m2.data_ptr(), lam.data_ptr())
    kept = (q, k, v, bias, m2, lam)
    nbytes = _lib.load().fjx_diff_attention_workspace_size(items, heads, kv_heads, nq, nk, d, code)
    strides = [1] * len(shape)
    for i in range(len(shape) - 1, 0, -1):
        strides[i - 1] = strides[i] * shape[i]
    shaped = shape, tuple(strides)
    as_they_lie = all(x is y for x, y in zip(kept, given))
    if as_they_lie:
        _remember(key, (bytes(a), shaped, unit, nbytes))
    return a, kept, shaped, unit, (key if as_they_lie else None, nbytes)


def diff_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    lambda_vectors: torch.Tensor,
    *,
    lambda_init: float,
    scale: float,
    bias: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    return_lse: bool = False,
    out: torch.Tensor | None = None,
):
    """Differential attention (``fjx_diff_attention_fwd``): per head
    ``(softmax(scale q_1 k_1^T + bias) - lambda softmax(scale q_2 k_2^T + bias)) v``
    with ``lambda = exp(a_1 . b_1) - exp(a_2 . b_2) + lambda_init``.

    q ``[..., 2 H, Q, D]`` and k ``[..., 2 Hk, K, D]``, heads 2 h and 2 h + 1
    being the two maps of head h; v ``[..., Hk, K, 2 D]`` (Hk divides H: heads
    may share keys and values); D 32 or 64. Any strides whose rows are whole
    16-byte pieces are taken as they lie, others are copied.
    ``lambda_vectors`` float32 ``[4, H, D]``: a_1, b_1, a_2, b_2. ``bias``
    ``[..., H, Q, K]`` in q's dtype: a plane per leading index of q, or shared
    over the last leading axes (1, or left out): ``[B, 1, H, J, J]`` for the
    rows of a triangle attention. ``mask`` broadcasts to ``[..., K]``: 0 takes
    a key out, whatever it holds. A bias of -inf, or of the dtype's lowest
    value, takes a key out for one query (k and v finite there), any other
    should leave bias / scale within float32's range. A row without keys is
    zeros. ``scale`` in [1e-30, 1e30].

    Returns ``out`` ``[..., H, Q, 2 D]``; with ``return_lse`` also what
    ``diff_attention_backward`` needs to know of the rows. ``out``: write into
    this tensor (its rows whole 16-byte pieces, any order of the other axes),
    which overlaps no input."""
    a, kept, (shape, strides), unit, (_, nbytes) = _diff_attention_args(q, k, v, lambda_vectors, lambda_init, scale, bias, mask)
    if out is None:
        out = torch.empty_strided(shape, strides, dtype=q.dtype, device=q.device)
    else:
        if out.shape != shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError(f"out must be a {q.dtype} tensor of shape {shape} on {q.device}, "
                             f"got {out.dtype} {tuple(out.shape)} on {out.device}")
        if out.data_ptr() in (q.data_ptr(), k.data_ptr(), v.data_ptr()):
            raise ValueError("out must not be q, k or v: other rows' results are taken from them")
        strides = _head_rows(out, unit)
        if strides is None:
            raise ValueError("out must have rows of whole 16-byte pieces, and leading axes that fold into one")
        a.out_strides = strides
    a.out = out.data_ptr()
    lse = None
    if return_lse:
        lse = torch.empty(shape[:-3] + (2 * a.heads, a.nq), dtype=torch.float32, device=q.device)
        a.stats = lse.data_ptr()
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    _launch(_lib.load().fjx_diff_attention_fwd, a, q)
    return (out, lse) if return_lse else out


def diff_attention_backward(
    dout: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    lambda_vectors: torch.Tensor,
    lse: torch.Tensor,
    *,
    lambda_init: float,
    scale: float,
    bias: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    bias_grad: bool = True,
):
    """Gradients of ``diff_attention`` (``fjx_diff_attention_bwd``) at the same
    arguments, ``lse`` being what the forward call returned. Returns ``(dq, dk,
    dv, dbias, dlambda)``: dq, dk, dv and dbias in the dtype and shape of q, k,
    v and bias (dbias None without a bias or with ``bias_grad`` off; of a shared
    plane the sum over the items, of shared heads' k and v the sum over the
    query heads), dlambda float32 ``[4, H, D]``. The same bits each time. Rows
    of the bias are less than 2^23 elements apart."""
    f, kept, (shape, _), unit, (key, _) = _diff_attention_args(q, k, v, lambda_vectors, lambda_init, scale, bias, mask)
    with_bias = bias is not None and bias_grad
    key = None if key is None else (key, _layout(dout, lse), with_bias)
    seen = None if key is None else _BLOCKS.get(key)
    if seen is not None and not dout.data_ptr() & 15:
        block, nbytes = seen
        g = _lib.DiffAttentionBwdArgs.from_buffer_copy(block)
        f.out_strides = g.fwd.out_strides
    else:
        _same_place(q, q.dtype, dout=dout)
        _same_place(q, torch.float32, lse=lse)
        _need_shape("dout", dout, shape)
        _need_shape("lse", lse, shape[:-3] + (2 * f.heads, f.nq))
        given = dout, lse
        dout, f.out_strides = _heads(dout, unit)
        if not lse.is_contiguous():
            lse = lse.contiguous()
        g = _lib.DiffAttentionBwdArgs(f, None, None, None, None, _packed(q.shape), _packed(k.shape), _packed(v.shape), None,
                                      _packed(bias.shape) if with_bias else (0, 0, 0))
        nbytes = _lib.load().fjx_diff_attention_bwd_workspace_size(f.items, f.heads, f.nq, f.nk, f.bias_share, with_bias)
        if key is not None and dout is given[0] and lse is given[1]:
            _remember(key, (bytes(g), nbytes))
    dev = q.device
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
    dlam = torch.empty(lambda_vectors.shape, dtype=torch.float32, device=dev)
    dbias = torch.empty(bias.shape, dtype=bias.dtype, device=dev) if with_bias else None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    f.stats, f.workspace, f.workspace_bytes = lse.data_ptr(), ws.data_ptr(), nbytes
    g.fwd = f
    g.dout, g.dq, g.dk, g.dv, g.dlambda = dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dlam.data_ptr()
    if with_bias:
        g.dbias = dbias.data_ptr()
    _launch(_lib.load().fjx_diff_attention_bwd, g, q)
    return dq, dk, dv, dbias, dlam


_INDEX = {torch.int32: _lib.FJX_INDEX_I32, torch.int64: _lib.FJX_INDEX_I64}


def _packed_rows(t: torch.Tensor, unit: int):
    """Strides {head, token} of [heads, tokens, width] where the kernels can take
    its rows as they lie, None where not."""
    st = _head_rows(t, unit)
    if st is None or (t.shape[1] > 1 and not t.shape[2] <= st[2] < (1 << 24) // t.element_size()):
        return None
    return st[1], st[2]


def _packed_heads(t: torch.Tensor, unit: int):
    """``t`` and its strides, a copy where its rows cannot be taken as they lie."""
    st = _packed_rows(t, unit)
    if st is None:
        t = t.clone(memory_format=torch.contiguous_format)
        st = _packed_rows(t, unit)
    return t, st


def _token_major(heads: int, tokens: int, width: int, like: torch.Tensor) -> torch.Tensor:
    """A new [heads, tokens, width] whose memory has a token's heads side by side,
    as the projections before and behind an attention have them."""
    return torch.empty_strided((heads, tokens, width), (width, heads * width, 1), dtype=like.dtype, device=like.device)


def _packed_attention_args(q, k, v, q_starts, scale, causal, k_starts, k_lengths):
    """The checked argument block that both directions share, the tensors it points
    to, the elements of a 16-byte piece, and (its key, the forward call's workspace)."""
    scale, causal = float(scale), bool(causal)
    key = (_layout(q, k, v, q_starts, k_starts, k_lengths), scale, causal)
    seen = _BLOCKS.get(key)
    if seen is not None:
        block, unit, nbytes = seen
        a = _lib.PackedAttentionArgs.from_buffer_copy(block)
        a.q, a.k, a.v = qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
        if not (qp | kp | vp) & 15:
            a.q_starts = q_starts.data_ptr()
            a.k_starts = a.q_starts if k_starts is None else k_starts.data_ptr()
            if k_lengths is not None:
                a.k_lengths = k_lengths.data_ptr()
            return a, (q, k, v, q_starts, k_starts, k_lengths), unit, (key, nbytes)
    dtype = q.dtype
    code = _code(dtype)
    _same_place(q, dtype, k=k, v=v)
    _same_device(q, q_starts=q_starts, k_starts=k_starts, k_lengths=k_lengths)
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3:
        raise ValueError(f"q, k and v must be [heads, tokens, width], got {tuple(qs)}, {tuple(ks)}, {tuple(v.shape)}")
    heads, tq, d = qs
    kv_heads, tk = ks[:2]
    _need_shape("k", k, (kv_heads, tk, d))
    _need_shape("v", v, (kv_heads, tk, d))
    if d % 8 or not 8 <= d <= 128:
        raise ValueError(f"q, k and v must have a width (head_dim) that is a multiple of 8 up to 128, got {d}")
    if not kv_heads or heads % kv_heads:
        raise ValueError(f"q's heads must be a multiple of k's, got {heads} and {kv_heads}")
    if q_starts.dim() != 1 or q_starts.shape[0] < 2:
        raise ValueError(f"q_starts must hold an offset more than there are sequences, one at least, got {tuple(q_starts.shape)}")
    seqs = q_starts.shape[0] - 1
    if k_starts is None:
        if tk != tq:
            raise ValueError(f"k_starts must be given where k has other tokens than q, got {tk} and {tq}")
    else:
        _need_shape("k_starts", k_starts, (seqs + 1,))
    _need_shape("k_lengths", k_lengths, (seqs,))
    offsets = (q_starts, k_starts, k_lengths)
    for name, t in zip(("q_starts", "k_starts", "k_lengths"), offsets):
        if t is not None and t.dtype not in _INDEX:
            raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
    wide = torch.int64 if any(t is not None and t.dtype is torch.int64 for t in offsets) else torch.int32
    index = _INDEX[wide]
    _dev(q)
    given = (q, k, v, *offsets)
    q_starts, k_starts, k_lengths = (_like(t, wide) for t in offsets)
    unit = 4 if dtype is torch.float32 else 8
    q, qst = _packed_heads(q, unit)
    k, kst = _packed_heads(k, unit)
    v, vst = _packed_heads(v, unit)
    a = _lib.PackedAttentionArgs(
        tq, tk, seqs, heads, kv_heads, d, code, index, causal, 0, scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), None,
        qst, kst, vst, (d, heads * d), q_starts.data_ptr(), (q_starts if k_starts is None else k_starts).data_ptr(),
        _ptr(k_lengths), None, None, (d, heads * d))
    kept = (q, k, v, q_starts, k_starts, k_lengths)
    nbytes = _lib.load().fjx_packed_attention_workspace_size(tq, tk, seqs, heads, kv_heads, d, code)
    as_they_lie = all(x is y for x, y in zip(kept, given))
    if as_they_lie:
        _remember(key, (bytes(a), unit, nbytes))
    return a, kept, unit, (key if as_they_lie else None, nbytes)


def packed_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    q_starts: torch.Tensor,
    *,
    scale: float,
    causal: bool = False,
    k_starts: torch.Tensor | None = None,
    k_lengths: torch.Tensor | None = None,
    return_lse: bool = False,
    out: torch.Tensor | None = None,
):
    """Attention over sequences of different lengths packed one behind the other
    (``fjx_packed_attention_fwd``): ``softmax(scale q k^T) v`` within each.

    q ``[H, Tq, D]``, k and v ``[Hk, Tk, D]`` (Hk divides H: heads may share keys
    and values), D a multiple of 8 up to 128; any strides whose rows are whole
    16-byte pieces are taken as they lie, others are copied. Sequence s has the
    queries ``q_starts[s] .. q_starts[s + 1] - 1`` and, of k and v, the tokens
    ``k_starts[s] .. k_starts[s + 1] - 1`` (left out: those of its queries), with
    ``k_lengths`` only the first ``k_lengths[s]`` of them: a cache with room for
    more, whose unused places may hold anything. The offsets are int32 or int64
    device tensors, from 0 on and not descending (the first counts as 0, whatever it
    holds: a slice of longer offsets goes with its first one subtracted and the
    tokens from there on); they are read on the device, so that a captured call
    takes new lengths at each replay. ``causal``: query i of
    nq sees key j of nk where ``j <= i + nk - nq``: each token those before it, new
    tokens their cache. A row without keys is zeros. k and v are finite. ``scale``
    in [1e-30, 1e30]. Calls of up to 2^28 rows of queries (H Tq) and of keys (Hk Tk),
    H times the offsets up to 2^20, are always taken, larger ones up to 2^23 workgroups.

    Returns ``out`` ``[H, Tq, D]``, a token's heads side by side in memory; rows
    behind the last sequence are zeros. With ``return_lse`` ``(out, lse, rest)``,
    the latter two for ``packed_attention_backward``: what it needs to know of the
    rows, and what the rounding of a bfloat16 output left (None of float32).
    ``out``: write into this tensor (its rows whole 16-byte pieces), which shares
    no memory with an input (refused); its rows behind the last sequence are left as they are."""
    a, kept, unit, (_, nbytes) = _packed_attention_args(q, k, v, q_starts, scale, causal, k_starts, k_lengths)
    if out is None:
        out = _token_major(a.heads, a.tokens_q, a.head_dim, q)
        a.zero_tail = 1
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError(f"out must be a {q.dtype} tensor of shape {tuple(q.shape)} on {q.device}, "
                             f"got {out.dtype} {tuple(out.shape)} on {out.device}")
        strides = _packed_rows(out, unit)
        if strides is None:
            raise ValueError("out must have rows of whole 16-byte pieces that do not overlap")
        a.out_strides = strides
    a.out = out.data_ptr()
    lse = rest = None
    if return_lse:
        lse = torch.empty((a.heads, a.tokens_q, 2), dtype=torch.float32, device=q.device)
        a.lse = lse.data_ptr()
        if q.dtype is torch.bfloat16:
            rest = _token_major(a.heads, a.tokens_q, a.head_dim, q)
            a.rest = rest.data_ptr()
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    _launch(_lib.load().fjx_packed_attention_fwd, a, q)
    return (out, lse, rest) if return_lse else out


def packed_attention_backward(
    dout: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    lse: torch.Tensor,
    rest: torch.Tensor | None,
    q_starts: torch.Tensor,
    *,
    scale: float,
    causal: bool = False,
    k_starts: torch.Tensor | None = None,
    k_lengths: torch.Tensor | None = None,
):
    """Gradients of ``packed_attention`` (``fjx_packed_attention_bwd``) at the same
    arguments; ``out``, ``lse`` and ``rest`` are what the forward call returned.
    Returns ``(dq, dk, dv)`` in the dtype and shape of q, k and v, a token's heads
    side by side in memory; gradients of shared heads are summed over the query
    heads, those of tokens of no sequence and of a cache's unused places are zeros.
    dout is finite; other values than numbers in a row of q may reach the gradients of all
    its sequence's keys. The same bits each time. Without ``rest`` bfloat16 gradients of rows in which
    one key has nearly all the weight lose digits."""
    scale, causal = float(scale), bool(causal)
    key = (_layout(q, k, v, q_starts, k_starts, k_lengths, dout, out, lse, rest), scale, causal)
    seen = _BLOCKS.get(key)
    fits = False
    if seen is not None:
        block, nbytes = seen
        g = _lib.PackedAttentionBwdArgs.from_buffer_copy(block)
        a = g.fwd
        a.q, a.k, a.v, a.out, g.dout = qp, kp, vp, op, dp = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                                             dout.data_ptr())
        if rest is not None:
            a.rest = rp = rest.data_ptr()
            op |= rp
        fits = not (qp | kp | vp | op | dp) & 15
    if fits:
        a.lse, a.q_starts = lse.data_ptr(), q_starts.data_ptr()
        a.k_starts = a.q_starts if k_starts is None else k_starts.data_ptr()
        if k_lengths is not None:
            a.k_lengths = k_lengths.data_ptr()
    else:
        a, kept, unit, (as_they_lie, _) = _packed_attention_args(q, k, v, q_starts, scale, causal, k_starts, k_lengths)
        _same_place(q, q.dtype, dout=dout, out=out, rest=rest)
        _same_place(q, torch.float32, lse=lse)
        _need_shape("dout", dout, q.shape)
        _need_shape("out", out, q.shape)
        _need_shape("rest", rest, q.shape)
        _need_shape("lse", lse, (a.heads, a.tokens_q, 2))
        if rest is not None and q.dtype is not torch.bfloat16:
            raise ValueError("rest is of bfloat16 outputs")
        given = dout, out, lse, rest
        lse = lse.contiguous()
        dout, dst = _packed_heads(dout, unit)
        out, a.out_strides = _packed_heads(out, unit)
        if rest is not None:
            rest, a.rest_strides = _packed_heads(rest, unit)
        by_q, by_k = (a.head_dim, a.heads * a.head_dim), (a.head_dim, a.kv_heads * a.head_dim)
        a.out, a.lse, a.rest = out.data_ptr(), lse.data_ptr(), _ptr(rest)
        g = _lib.PackedAttentionBwdArgs(a, dout.data_ptr(), None, None, None, dst, by_q, by_k, by_k)
        nbytes = _lib.load().fjx_packed_attention_bwd_workspace_size(a.tokens_q, a.tokens_k, a.sequences, a.heads, a.kv_heads,
                                                                     a.head_dim, a.dtype)
        if as_they_lie is not None and all(x is y for x, y in zip((dout, out, lse, rest), given)):
            _remember(key, (bytes(g), nbytes))
        a = g.fwd
    dq, dk, dv = (_token_major(*t.shape, q) for t in (q, k, v))
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    g.dq, g.dk, g.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    _launch(_lib.load().fjx_packed_attention_bwd, g, q)
    return dq, dk, dv


def _side_by_side(shape):
    """Strides of [..., heads, tokens, width] whose memory has a token's heads side
    by side."""
    *lead, heads, tokens, width = shape
    st, step = [width, heads * width, 1], tokens * heads * width
    for n in reversed(lead):
        st.insert(0, step)
        step *= n
    return tuple(st)


def _like_heads(t: torch.Tensor, strides) -> torch.Tensor:
    return torch.empty_strided(t.shape, strides, dtype=t.dtype, device=t.device)


def _rotary_args(q, k, positions, frequencies, q_weight, k_weight, eps, sections, interleaved):
    """The checked argument block that both directions share, the tensors it points
    to, the elements of a 16-byte piece, the strides of outputs like q and k, and its
    key."""
    eps, interleaved = float(eps), bool(interleaved)
    sections = None if sections is None else tuple([int(n) for n in sections])
    key = (_layout(q, k, positions, frequencies, q_weight, k_weight), eps, sections, interleaved, "rotary")
    seen = _BLOCKS.get(key)
    if seen is not None:
        block, unit, like = seen
        a = _lib.HeadNormRotaryArgs.from_buffer_copy(block)
        a.q, a.positions, a.frequencies = p, _, _ = q.data_ptr(), positions.data_ptr(), frequencies.data_ptr()
        if k is not None:
            a.k = kp = k.data_ptr()
            p |= kp
        if q_weight is not None:
            a.q_weight = wp = q_weight.data_ptr()
            p |= wp
        if k_weight is not None:
            a.k_weight = wp = k_weight.data_ptr()
            p |= wp
        if not p & 15:
            return a, (q, k, positions, frequencies, q_weight, k_weight), unit, like, key
    dtype, shape = q.dtype, q.shape
    code = _code(dtype)
    _same_place(q, dtype, k=k, q_weight=q_weight, k_weight=k_weight)
    _same_place(q, torch.float64, frequencies=frequencies)
    _same_device(q, positions=positions)
    if len(shape) < 3:
        raise ValueError(f"q must be [..., heads, tokens, width], got {tuple(shape)}")
    lead, (heads, tokens, d) = tuple(shape[:-3]), shape[-3:]
    kv_heads = 0
    if k is not None:
        kv_heads = k.shape[-3] if k.dim() > 2 else 0
        _need_shape("k", k, lead + (kv_heads, tokens, d))
    elif k_weight is not None:
        raise ValueError("k_weight needs k")
    _need_shape("q_weight", q_weight, (d,))
    _need_shape("k_weight", k_weight, (d,))
    if d % 8 or not 8 <= d <= 256:
        raise ValueError(f"q and k must have a width (head_dim) that is a multiple of 8 up to 256, got {d}")
    if frequencies.dim() != 1 or frequencies.shape[0] % 4 or 2 * frequencies.shape[0] > d:
        raise ValueError(f"frequencies must be a multiple of 4 and at most half of the {d} channels, got {tuple(frequencies.shape)}")
    pairs = frequencies.shape[0]
    sections_ = (pairs,) if sections is None else sections
    if not 1 <= len(sections_) <= 4 or min(sections_) < 0 or sum(sections_) != pairs:
        raise ValueError(f"sections must be 1 to 4 numbers that add up to the {pairs} frequencies, got {sections}")
    index = _INDEX.get(positions.dtype)
    if index is None:
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    axes = len(sections_)
    shared = positions.dim() == 2
    _need_shape("positions", positions, (axes, tokens) if shared else (axes, *lead, tokens))
    _dev(q)
    given = (q, k, positions, frequencies, q_weight, k_weight)
    positions, frequencies = positions.contiguous(), frequencies.contiguous()
    wq, wk = (None if w is None else _aligned(w.contiguous()) for w in (q_weight, k_weight))
    unit = 4 if dtype is torch.float32 else 8
    q, qst = _heads(q, unit)
    k, kst = (None, (0, 0, 0)) if k is None else _heads(k, unit)
    items = 1
    for n in lead:
        items *= n
    a = _lib.HeadNormRotaryArgs(
        items, heads, kv_heads, tokens, d, code, index, interleaved, axes, sections_, eps, q.data_ptr(), _ptr(k), _ptr(wq),
        _ptr(wk), positions.data_ptr(), (positions.stride(0), 0 if shared else tokens), frequencies.data_ptr(), None, None,
        qst, kst, (tokens * heads * d, d, heads * d), (tokens * kv_heads * d, d, kv_heads * d))
    kept = (q, k, positions, frequencies, wq, wk)
    as_they_lie = all(x is y for x, y in zip(kept, given))
    like = _side_by_side(shape), None if k is None else _side_by_side(k.shape)
    if as_they_lie:
        _remember(key, (bytes(a), unit, like))
    return a, kept, unit, like, key if as_they_lie else None


def _aligned(t: torch.Tensor) -> torch.Tensor:
    return t.clone() if t.data_ptr() & 15 else t


def head_norm_rotary(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    sections: tuple[int, ...] | None = None,
    interleaved: bool = False,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
):
    """The root-mean-square norm of each head's queries and keys and their rotation
    by position, in one pass (``fjx_head_norm_rotary_fwd``).

    q ``[..., H, T, D]``, k ``[..., Hk, T, D]`` (or None), D a multiple of 8 up to
    256; any strides whose rows are whole 16-byte pieces are taken as they lie,
    others are copied. ``q_weight`` and ``k_weight`` ``[D]``: ``x / sqrt(mean(x^2) +
    eps) * weight``; None: no norm. ``frequencies`` float64 ``[P]``, in radians a
    position: pair i, the channels (i, i + P) or with ``interleaved`` (2 i, 2 i + 1),
    is turned by position times ``frequencies[i]``, an angle that is taken in 64 bits;
    channels from 2 P on are left (P a multiple of 4, 0 for the norm alone).
    ``positions`` int32 or int64 ``[A, ..., T]``, or ``[A, T]`` for all items alike:
    axis a's for the ``sections[a]`` pairs behind those of the axes before it
    (residue, chain and copy of a token, for instance; up to 4 axes; left out: one).

    Returns ``(q', k')``, a token's heads side by side in memory (k' None without k);
    no tokens or no items are allowed. ``q_out``, ``k_out``: write into these tensors
    (of q's and k's shape, their rows whole 16-byte pieces: places in a cache, for
    one), each of which may be its input, in its very place; they share no other
    memory with an input or each other (refused)."""
    a, kept, unit, like, _ = _rotary_args(q, k, positions, frequencies, q_weight, k_weight, eps, sections, interleaved)
    if q_out is None:
        q_out = _like_heads(q, like[0])
    else:
        a.q_out_strides = _rotary_out("q_out", q_out, q, unit)
    a.q_out = q_out.data_ptr()
    if k is None:
        if k_out is not None:
            raise ValueError("k_out needs k")
    else:
        if k_out is None:
            k_out = _like_heads(k, like[1])
        else:
            a.k_out_strides = _rotary_out("k_out", k_out, k, unit)
        a.k_out = k_out.data_ptr()
    if a.items and a.tokens:
        _launch(_lib.load().fjx_head_norm_rotary_fwd, a, q)
    return q_out, k_out


def _rotary_out(name: str, out: torch.Tensor, x: torch.Tensor, unit: int):
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{name} must be a {x.dtype} tensor of shape {tuple(x.shape)} on {x.device}, "
                         f"got {out.dtype} {tuple(out.shape)} on {out.device}")
    strides = _head_rows(out, unit)
    if strides is None:
        raise ValueError(f"{name} must have rows of whole 16-byte pieces, and leading axes that fold into one")
    return strides


def head_norm_rotary_backward(
    dq: torch.Tensor,
    dk: torch.Tensor | None,
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    sections: tuple[int, ...] | None = None,
    interleaved: bool = False,
):
    """Gradients of ``head_norm_rotary`` (``fjx_head_norm_rotary_bwd``) at the same
    arguments, dq and dk being those of its outputs (dk None without k). Returns
    ``(dx_q, dx_k, dq_weight, dk_weight)``: the inputs' in their dtype and shape, a
    token's heads side by side in memory, the weights' float32 ``[D]``, summed over
    tokens and heads in one order; None for what is not there."""
    eps, interleaved = float(eps), bool(interleaved)
    sections = None if sections is None else tuple([int(n) for n in sections])
    key = (_layout(q, k, positions, frequencies, q_weight, k_weight, dq, dk), eps, sections, interleaved)
    seen = _BLOCKS.get(key)
    fits = False
    if seen is not None:
        block, nbytes, like = seen
        b = _lib.HeadNormRotaryBwdArgs.from_buffer_copy(block)
        a = b.fwd
        a.q, a.q_out = p, yp = q.data_ptr(), dq.data_ptr()
        p |= yp
        if k is not None:
            a.k, a.k_out = kp, yp = k.data_ptr(), dk.data_ptr()
            p |= kp | yp
        if q_weight is not None:
            a.q_weight = wp = q_weight.data_ptr()
            p |= wp
        if k_weight is not None:
            a.k_weight = wp = k_weight.data_ptr()
            p |= wp
        fits = not p & 15
    if fits:
        a.positions, a.frequencies = positions.data_ptr(), frequencies.data_ptr()
    else:
        a, kept, unit, like, as_they_lie = _rotary_args(q, k, positions, frequencies, q_weight, k_weight, eps, sections, interleaved)
        if (dk is None) != (k is None):
            raise ValueError("dk must be given where k is, and only there")
        _same_place(q, q.dtype, dq=dq, dk=dk)
        _need_shape("dq", dq, q.shape)
        if k is not None:
            _need_shape("dk", dk, k.shape)
        given = dq, dk
        dq, a.q_out_strides = _heads(dq, unit)
        a.q_out = dq.data_ptr()
        if dk is not None:
            dk, a.k_out_strides = _heads(dk, unit)
            a.k_out = dk.data_ptr()
        packed = lambda h: (a.tokens * h * a.head_dim, a.head_dim, h * a.head_dim)  # noqa: E731
        b = _lib.HeadNormRotaryBwdArgs(a, None, None, packed(a.heads), packed(a.kv_heads))
        nbytes = 0
        if q_weight is not None or k_weight is not None:
            nbytes = _lib.load().fjx_head_norm_rotary_bwd_workspace_size(a.items, a.heads, a.kv_heads, a.tokens, a.head_dim)
        if as_they_lie is not None and dq is given[0] and dk is given[1]:
            _remember(key, (bytes(b), nbytes, like))
    dev, d = q.device, q.shape[-1]
    gq, gk, dwq, dwk = _like_heads(q, like[0]), None, None, None
    if not (b.fwd.items and b.fwd.tokens):  # no rows: sums of nothing
        return gq, None if k is None else _like_heads(k, like[1]), *(
            None if w is None else torch.zeros(d, dtype=torch.float32, device=dev) for w in (q_weight, k_weight))
    b.dq = gq.data_ptr()
    if k is not None:
        gk = _like_heads(k, like[1])
        b.dk = gk.data_ptr()
    if q_weight is not None:
        dwq = torch.empty(d, dtype=torch.float32, device=dev)
        b.dq_weight = dwq.data_ptr()
    if k_weight is not None:
        dwk = torch.empty(d, dtype=torch.float32, device=dev)
        b.dk_weight = dwk.data_ptr()
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        b.workspace, b.workspace_bytes = ws.data_ptr(), nbytes
    _launch(_lib.load().fjx_head_norm_rotary_bwd, b, q)
    return gq, gk, dwq, dwk


_CODES = {None: (_lib.FJX_CODES_NONE, None), "e4m3": (_lib.FJX_CODES_E4M3, torch.float8_e4m3fn),
          "int8": (_lib.FJX_CODES_INT8, torch.int8)}


def rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    *,
    residual: torch.Tensor | None = None,
    eps: float = 1e-6,
    codes: str | None = None,
    group: int = 0,
    out: torch.Tensor | None = None,
    sum_out: torch.Tensor | None = None,
):
    """Root-mean-square norm over the last axis (``fjx_rms_norm_fwd``):
    ``h / sqrt(mean(h^2) + eps) * weight`` with ``h = x + residual``.

    Returns ``y``, or ``(y, h)`` with a residual (h rounded to x's dtype, y of
    the unrounded sum). ``codes`` ``"e4m3"`` or ``"int8"``: y in 8 bits with a
    float32 scale a row, or every ``group`` channels (32, 64 or 128), and
    ``(codes, scales)`` in y's place: ``(codes, scales)`` or ``(codes, scales,
    h)``; ``y ~ codes * scale``, scales ``[..., 1]`` or ``[..., C / group]``.
    ``out`` (without codes) and ``sum_out``: write y and h into these tensors
    (x's shape and dtype, contiguous); each may be ``x`` or ``residual``."""
    key, eps = None, float(eps)
    if out is None and sum_out is None and (codes is None or isinstance(codes, str)):
        key = (_layout(x, weight, residual), eps, codes, group)
        seen = _BLOCKS.get(key)
        if seen is not None:
            block, scales_shape = seen
            a = _lib.RmsNormArgs.from_buffer_copy(block)
            a.x, a.weight = x.data_ptr(), weight.data_ptr()
            h = scales = None
            if residual is not None:
                h = torch.empty_like(x)
                a.residual, a.sum_out = residual.data_ptr(), h.data_ptr()
            if codes is None:
                y = torch.empty_like(x)
            else:
                y = torch.empty_like(x, dtype=_CODES[codes][1])
                scales = torch.empty(scales_shape, dtype=torch.float32, device=x.device)
                a.scales = scales.data_ptr()
            a.out = y.data_ptr()
            _launch(_lib.load().fjx_rms_norm_fwd, a, x)
            return _norm_result(y, scales, h)
    kind = _CODES.get(codes) if codes is None or isinstance(codes, str) else None
    if kind is None:
        raise ValueError(f"codes must be None, 'e4m3' or 'int8', got {codes!r}")
    dtype, shape = x.dtype, x.shape
    code = _code(dtype)
    _same_place(x, dtype, weight=weight, residual=residual)
    if not shape:
        raise ValueError("x must have a last axis to be normalised over")
    c = shape[-1]
    _need_shape("weight", weight, (c,))
    if residual is not None:
        _need_shape("residual", residual, shape)
    elif sum_out is not None:
        raise ValueError("sum_out needs a residual")
    if group and codes is None:
        raise ValueError("group needs codes")
    _dev(x)
    xf, res = _like(x, dtype), _like(residual, dtype)
    scales = None
    if codes is None:
        y = _out_buffer(out, x, xf)
    else:
        if out is not None:
            raise ValueError("out is for a norm without codes")
        if group < 0 or (group and c % group):
            raise ValueError(f"group must divide the {c} channels, got {group}")
        y = torch.empty(shape, dtype=kind[1], device=x.device)
        scales = torch.empty(shape[:-1] + (c // group if group else 1,), dtype=torch.float32, device=x.device)
    h = None if res is None else _out_buffer(sum_out, x, xf)
    if h is not None and h.data_ptr() == y.data_ptr():
        raise ValueError("out and sum_out must be two buffers")
    w = _like(weight, dtype)
    a = _lib.RmsNormArgs(x.numel() // max(c, 1), c, code, eps, xf.data_ptr(), _ptr(res), w.data_ptr(), _ptr(h), y.data_ptr(),
                         kind[0], group, _ptr(scales))
    if key is not None and xf is x and res is residual and w is weight:
        _remember(key, (bytes(a), None if scales is None else scales.shape))
    _launch(_lib.load().fjx_rms_norm_fwd, a, x)
    return _norm_result(y, scales, h)


def _norm_result(y, scales, h):
    if scales is not None:
        return (y, scales) if h is None else (y, scales, h)
    return y if h is None else (y, h)


def rms_norm_backward(
    dy: torch.Tensor,
    h: torch.Tensor,
    weight: torch.Tensor,
    *,
    dh: torch.Tensor | None = None,
    eps: float = 1e-6,
    out: torch.Tensor | None = None,
):
    """Gradients of ``rms_norm`` at the sum ``h`` it returned (x itself without
    a residual): ``(dx, dweight)`` (``fjx_rms_norm_bwd``). dx is the residual's
    gradient too and includes ``dh``, what reaches h from elsewhere; dweight is
    float32, summed over the rows in one order. ``out``: write dx into this
    tensor, which may be ``dy`` or ``dh``."""
    key, eps = None, float(eps)
    if out is None:
        key = (_layout(dy, h, weight, dh), eps)
        seen = _BLOCKS.get(key)
        if seen is not None:
            block, nbytes, c = seen
            a = _lib.RmsNormBwdArgs.from_buffer_copy(block)
            dx = torch.empty_like(h)
            dw = torch.empty(c, dtype=torch.float32, device=h.device)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
            a.dy, a.h, a.weight, a.dx = dy.data_ptr(), h.data_ptr(), weight.data_ptr(), dx.data_ptr()
            a.dweight, a.workspace = dw.data_ptr(), ws.data_ptr()
            if dh is not None:
                a.dh = dh.data_ptr()
            _launch(_lib.load().fjx_rms_norm_bwd, a, h)
            return dx, dw
    dtype, shape = h.dtype, h.shape
    code = _code(dtype)
    _same_place(h, dtype, dy=dy, weight=weight, dh=dh)
    if not shape:
        raise ValueError("h must have a last axis")
    c = shape[-1]
    _need_shape("weight", weight, (c,))
    _need_shape("dy", dy, shape)
    _need_shape("dh", dh, shape)
    _dev(h)
    hf, dyf, dhf, w = _like(h, dtype), _like(dy, dtype), _like(dh, dtype), _like(weight, dtype)
    if out is not None and out.data_ptr() == h.data_ptr():
        raise ValueError("out must not be h")
    dx = _out_buffer(out, h, hf)
    dw = torch.empty((c,), dtype=torch.float32, device=h.device)
    lib = _lib.load()
    rows = h.numel() // max(c, 1)
    nbytes = lib.fjx_rms_norm_bwd_workspace_size(rows, c)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
    a = _lib.RmsNormBwdArgs(rows, c, code, eps, dyf.data_ptr(), hf.data_ptr(), w.data_ptr(), _ptr(dhf), dx.data_ptr(),
                            dw.data_ptr(), ws.data_ptr(), nbytes)
    if key is not None and hf is h and dyf is dy and dhf is dh and w is weight:
        _remember(key, (bytes(a), nbytes, c))
    _launch(lib.fjx_rms_norm_bwd, a, h)
    return dx, dw


_SHARE = {-3: _lib.FJX_SHARE_N, -2: _lib.FJX_SHARE_M, -1: _lib.FJX_SHARE_C}


def dropout_add(
    x: torch.Tensor,
    *,
    p: float,
    seed: int,
    offset: int = 0,
    step: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    shared: tuple[int, ...] = (),
    out_mask: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``residual + (kept ? x / (1 - p) : 0)``, times ``out_mask != 0`` per
    position when that is given (``fjx_dropout_fwd``); without a residual the
    dropped x alone. The last axis a multiple of 8.

    The mask is drawn anew in every call that needs it and never stored: the
    same ``seed`` (64 bits), ``offset`` (64 bits; one for each use of dropout)
    and shape give the same one. ``shared``: the axes (-3, -2, -1) over which
    one mask entry serves, as the Pairformer drops an update for all rows
    (``(-3,)``) or for all columns (``(-2,)``). ``step``: an int64 tensor of
    one element on x's device, read by the kernel and added to ``offset``: a
    captured call then drops anew at each replay (calls with one seed and one
    step need offsets further apart than the step counts, or the later draws
    what the other drew). ``out``: write into this
    tensor, which may be ``x`` and/or ``residual``."""
    key, p = None, float(p)
    shared = tuple(shared)
    if out_mask is None and step is None and out is None:
        key = (_layout(x, residual), p, shared)
        block = _BLOCKS.get(key)
        if block is not None and 0 <= seed < 2**64 and 0 <= offset < 2**64:
            a = _lib.DropoutArgs.from_buffer_copy(block)
            out = torch.empty_like(x)
            a.seed, a.offset, a.x, a.out = seed, offset, x.data_ptr(), out.data_ptr()
            if residual is not None:
                a.residual = residual.data_ptr()
            _launch(_lib.load().fjx_dropout_fwd, a, x)
            return out
    dtype, shape = x.dtype, x.shape
    code = _code(dtype)
    _same_place(x, dtype, residual=residual)
    dims = len(shape)
    if not dims:
        raise ValueError("x must have a last axis")
    flags = 0
    for axis in shared:
        if axis not in _SHARE or dims < -axis:
            raise ValueError(f"shared must name axes of x among -3, -2 and -1, got {shared!r} for {tuple(shape)}")
        flags |= _SHARE[axis]
    if residual is not None:
        _need_shape("residual", residual, shape)
    if not (0 <= seed < 2**64 and 0 <= offset < 2**64):
        raise ValueError(f"seed and offset must be in [0, 2^64), got {seed} and {offset}")
    if out_mask is not None or step is not None:
        _same_device(x, out_mask=out_mask, step=step)
    if step is not None and (step.dtype is not torch.int64 or step.numel() != 1):
        raise ValueError(f"step must be an int64 tensor of one element, got {step.dtype} {tuple(step.shape)}")
    _dev(x)
    xf, res = _like(x, dtype), _like(residual, dtype)
    om = None if out_mask is None else _rows_of(out_mask, shape[:-1], dtype, "out_mask")
    out = _out_buffer(out, x, xf)
    n, m, c = shape[-3:] if dims > 2 else (1, 1, *shape)[-3:]
    a = _lib.DropoutArgs(x.numel() // max(n * m * c, 1), n, m, c, code, flags, p, seed, offset, _ptr(step), xf.data_ptr(),
                         _ptr(res), _ptr(om), out.data_ptr())
    if key is not None and xf is x and res is residual:
        _remember(key, bytes(a))
    _launch(_lib.load().fjx_dropout_fwd, a, x)
    return out


def dropout_backward(
    dout: torch.Tensor,
    *,
    p: float,
    seed: int,
    offset: int = 0,
    step: torch.Tensor | None = None,
    shared: tuple[int, ...] = (),
    out_mask: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """The gradient of ``dropout_add``'s x: the same mask, drawn again, on the
    output's gradient (the residual's gradient is ``dout`` itself, times
    ``out_mask != 0``). ``step`` must hold what it held in the forward call."""
    return dropout_add(dout, p=p, seed=seed, offset=offset, step=step, shared=shared, out_mask=out_mask, out=out)


def _check_weights(x: torch.Tensor, w) -> None:
    """Every weight contiguous, in ``x``'s dtype and on its (cuda) device."""
    dtype, dev = x.dtype, x.get_device()
    for t in _tensors(w):
        if t is not None and (t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous()):
            name = next(f.name for f in fields(w) if getattr(w, f.name) is t)
            raise ValueError(
                f"weight {name} must be a contiguous {x.dtype} tensor on {x.device}; "
                "pack weights with .to(dtype, device) first"
            )
