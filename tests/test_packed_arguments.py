"""CPU checks of packed attention and of the heads' norm with rotation: what they
refuse, at the Python functions and at the C ABI (fake, never dereferenced pointers),
their struct layouts and workspace sizes, and their compiled kernels' resources."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from foldjax_amd import _lib, kernels
from tests.test_operator_resources import metadata

ROOT = Path(__file__).resolve().parent.parent
FAKE = 0x1000


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_struct_layout_matches_c(tmp_path):
    structs = {
        "fjx_packed_attention_args": _lib.PackedAttentionArgs,
        "fjx_packed_attention_bwd_args": _lib.PackedAttentionBwdArgs,
        "fjx_head_norm_rotary_args": _lib.HeadNormRotaryArgs,
        "fjx_head_norm_rotary_bwd_args": _lib.HeadNormRotaryBwdArgs,
    }
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fjx_tri.h"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join([*lines, "return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT / 'include'}", "-I/opt/rocm/include",
                    str(src), "-o", str(exe)], check=True, capture_output=True, text=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        cname, field, value = line.split()
        cls = structs[cname]
        assert (ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset) == int(value), (cname, field)


def packed(**more):
    a = _lib.PackedAttentionArgs(tokens_q=40, tokens_k=40, sequences=2, heads=4, kv_heads=2, head_dim=32, dtype=1, scale=1.0,
                                 q=FAKE, k=FAKE, v=FAKE, out=FAKE, q_starts=FAKE, k_starts=FAKE)
    for name in ("q_strides", "k_strides", "v_strides", "out_strides", "rest_strides"):
        setattr(a, name, (32, 128))
    for n, v in more.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("more,code,text", [
    ({"sequences": 0}, 1, "sequences"), ({"tokens_q": -1}, 1, "tokens"), ({"tokens_k": -1}, 1, "tokens"), ({"heads": 0}, 1, "heads"),
    ({"dtype": 5}, 1, "dtype"), ({"index_dtype": 2}, 1, "index_dtype"), ({"head_dim": 0}, 2, "head_dim"),
    ({"head_dim": 20}, 2, "head_dim"), ({"head_dim": 136}, 2, "head_dim"), ({"heads": 2048}, 2, "heads"),
    ({"kv_heads": 3}, 1, "divide"), ({"scale": 0.0}, 1, "scale"), ({"scale": float("nan")}, 1, "scale"),
    ({"scale": 1e31}, 1, "scale"), ({"q": None}, 1, "NULL"), ({"v": None}, 1, "NULL"), ({"k_starts": None}, 1, "NULL"),
    ({"q": FAKE + 8}, 1, "16-byte"), ({"lse": FAKE + 4}, 1, "aligned"), ({"q_starts": FAKE + 2}, 1, "aligned"),
    ({"index_dtype": 1, "k_lengths": FAKE + 4}, 1, "aligned"), ({"dtype": 0, "rest": FAKE}, 1, "rest"),
    ({"tokens_q": 1 << 30}, 2, "2\\^31"), ({"tokens_k": 1 << 31}, 2, "2\\^31"), ({"sequences": 1 << 22}, 2, "2\\^22"),
    ({"q_strides": (0, 128)}, 1, "strides"), ({"q_strides": (32, 24)}, 1, "strides"), ({"k_strides": (32, 100)}, 1, "strides"),
    ({"v_strides": (32, 1 << 23)}, 1, "strides"), ({"out_strides": (-32, 128)}, 1, "strides"),
    ({"rest": FAKE, "rest_strides": (32, 0)}, 1, "strides"),
    ({"tokens_q": 1 << 27, "heads": 8, "kv_heads": 8}, 2, "launch"),
])
def test_packed_attention_refusals(lib, more, code, text):
    import re

    a = packed(**more)
    assert lib.fjx_packed_attention_fwd(ctypes.byref(a), None) == code
    assert re.search(text, lib.fjx_last_error().decode()), lib.fjx_last_error()
    b = _lib.PackedAttentionBwdArgs(fwd=a, dout=FAKE, dq=FAKE, dk=FAKE, dv=FAKE)
    for name in ("dout_strides", "dq_strides", "dk_strides", "dv_strides"):
        setattr(b, name, (32, 128))
    if a.lse is None:
        b.fwd.lse = FAKE
    assert lib.fjx_packed_attention_bwd(ctypes.byref(b), None) == code


@pytest.mark.parametrize("more,code,text", [
    ({"dout": None}, 1, "NULL"), ({"dk": None}, 1, "NULL"), ({"dq": FAKE + 4}, 1, "16-byte"),
    ({"dq_strides": (32, 16)}, 1, "strides"), ({"dv_strides": (0, 128)}, 1, "strides"), ({"dout_strides": (33, 128)}, 1, "strides"),
    ({}, 3, "workspace"),
])
def test_packed_attention_gradients_refusals(lib, more, code, text):
    b = _lib.PackedAttentionBwdArgs(fwd=packed(lse=FAKE), dout=FAKE, dq=FAKE, dk=FAKE, dv=FAKE)
    for name in ("dout_strides", "dq_strides", "dk_strides", "dv_strides"):
        setattr(b, name, (32, 128))
    for n, v in more.items():
        setattr(b, n, v)
    assert lib.fjx_packed_attention_bwd(ctypes.byref(b), None) == code
    assert text in lib.fjx_last_error().decode()
    assert lib.fjx_packed_attention_bwd(None, None) == 1


def test_packed_attention_workspace(lib):
    size = lib.fjx_packed_attention_workspace_size
    assert size(0, 10, 1, 4, 2, 32, 1) == 0 and size(8, 10, 0, 4, 2, 32, 1) == 0 and size(8, 10, 1, 4, 3, 32, 1) == 0
    assert size(40, 40, 2, 4, 2, 32, 1) == 0
    need = size(8, 8 * 16384, 8, 8, 2, 128, 1)
    assert need >= 32 * 64 * (128 + 2) * 4  # 32 splits of 64 rows
    a = packed(tokens_q=8, tokens_k=8 * 16384, sequences=8, heads=8, head_dim=128, k_strides=(1 << 22, 128), v_strides=(1 << 22, 128),
               q_strides=(128, 1024), out_strides=(128, 1024))
    for ws, nbytes, code in ((None, need, 3), (FAKE, need - 1, 3), (FAKE + 8, need, 1)):
        a.workspace, a.workspace_bytes = ws, nbytes
        assert lib.fjx_packed_attention_fwd(ctypes.byref(a), None) == code
    assert lib.fjx_packed_attention_fwd(None, None) == 1
    size = lib.fjx_packed_attention_bwd_workspace_size
    assert size(40, 40, 2, 4, 2, 32, 1) >= 4 * 40 * 4 and size(-1, 40, 2, 4, 2, 32, 1) == 0
    # nothing to do is no error
    assert lib.fjx_packed_attention_fwd(ctypes.byref(packed(tokens_q=0, q=None, out=None)), None) == 0


def rotary(**more):
    a = _lib.HeadNormRotaryArgs(items=2, heads=4, kv_heads=2, tokens=8, head_dim=32, dtype=1, axes=2, sections=(8, 8, 0, 0), eps=1e-6,
                                q=FAKE, k=FAKE, q_weight=FAKE, k_weight=FAKE, positions=FAKE, frequencies=FAKE, q_out=FAKE,
                                k_out=FAKE)
    for name in ("q_strides", "k_strides", "q_out_strides", "k_out_strides"):
        setattr(a, name, (1024, 32, 128))
    for n, v in more.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("more,code,text", [
    ({"items": 0}, 1, "items"), ({"tokens": 0}, 1, "tokens"), ({"heads": 0}, 1, "heads"), ({"kv_heads": -1}, 1, "kv_heads"),
    ({"dtype": 3}, 1, "dtype"), ({"index_dtype": 7}, 1, "index_dtype"), ({"head_dim": 28}, 2, "head_dim"),
    ({"head_dim": 264}, 2, "head_dim"), ({"heads": 2000}, 2, "heads"), ({"axes": 0}, 1, "axes"), ({"axes": 5}, 1, "axes"),
    ({"sections": (-4, 8, 0, 0)}, 1, "sections"), ({"sections": (6, 0, 0, 0)}, 2, "pairs"), ({"sections": (12, 8, 0, 0)}, 2, "pairs"),
    ({"q": None}, 1, "NULL"), ({"k_out": None}, 1, "NULL"), ({"positions": None}, 1, "NULL"), ({"frequencies": None}, 1, "NULL"),
    ({"k_weight": FAKE + 2}, 1, "16-byte"), ({"frequencies": FAKE + 4}, 1, "aligned"), ({"positions": FAKE + 2}, 1, "aligned"),
    ({"q_strides": (1024, 33, 128)}, 1, "strides"), ({"items": 1 << 31}, 2, "rows"), ({"q_strides": (-1024, 32, 128)}, 1, "strides"),
])
def test_head_norm_rotary_refusals(lib, more, code, text):
    a = rotary(**more)
    assert lib.fjx_head_norm_rotary_fwd(ctypes.byref(a), None) == code
    assert text in lib.fjx_last_error().decode()
    b = _lib.HeadNormRotaryBwdArgs(a, FAKE, FAKE, (1024, 32, 128), (1024, 32, 128), FAKE, FAKE)
    assert lib.fjx_head_norm_rotary_bwd(ctypes.byref(b), None) == code


def test_head_norm_rotary_gradients_refusals(lib):
    st = (1024, 32, 128)
    for b, code in ((_lib.HeadNormRotaryBwdArgs(rotary(), None, FAKE, st, st, FAKE, FAKE), 1),
                    (_lib.HeadNormRotaryBwdArgs(rotary(), FAKE, None, st, st, FAKE, FAKE), 1),
                    (_lib.HeadNormRotaryBwdArgs(rotary(), FAKE, FAKE, st, st, None, FAKE), 1),
                    (_lib.HeadNormRotaryBwdArgs(rotary(), FAKE, FAKE, (0, 32, 128), st, FAKE, FAKE), 1),
                    (_lib.HeadNormRotaryBwdArgs(rotary(), FAKE, FAKE, st, st, FAKE, FAKE), 3)):
        assert lib.fjx_head_norm_rotary_bwd(ctypes.byref(b), None) == code
    a = rotary()
    a.q_out_strides = (0, 32, 128)
    assert lib.fjx_head_norm_rotary_fwd(ctypes.byref(a), None) == 1  # an output's items fall together
    assert lib.fjx_head_norm_rotary_fwd(None, None) == 1 and lib.fjx_head_norm_rotary_bwd(None, None) == 1
    size = lib.fjx_head_norm_rotary_bwd_workspace_size
    assert size(0, 4, 2, 8, 32) == 0 and size(2, 4, 2, 8, 30) == 0 and size(2, 4, 2, 8, 32) >= 2 * 32 * 4


def tensors(h=4, kv=2, tq=10, tk=10, d=32, dtype=torch.bfloat16):
    return torch.zeros(h, tq, d, dtype=dtype), torch.zeros(kv, tk, d, dtype=dtype), torch.zeros(kv, tk, d, dtype=dtype)


I32 = torch.tensor([0, 4, 10], dtype=torch.int32)


@pytest.mark.parametrize("change,text", [
    ({"q": torch.zeros(4, 10, 32, dtype=torch.float16)}, "float32 or bfloat16"), ({"k": torch.zeros(2, 10, 32)}, "k must be"),
    ({"q": torch.zeros(10, 32, dtype=torch.bfloat16)}, "heads, tokens, width"), ({"v": torch.zeros(2, 10, 64, dtype=torch.bfloat16)}, "v must"),
    ({"k": torch.zeros(2, 11, 32, dtype=torch.bfloat16), "v": torch.zeros(2, 11, 32, dtype=torch.bfloat16)}, "k_starts must be given"),
    ({"k": torch.zeros(3, 10, 32, dtype=torch.bfloat16), "v": torch.zeros(3, 10, 32, dtype=torch.bfloat16)}, "multiple of k's"),
    ({"q_starts": torch.tensor([0])}, "q_starts"), ({"q_starts": I32.float()}, "int32 or int64"), ({"q_starts": I32[None]}, "q_starts"),
    ({"k_starts": I32[:2]}, "k_starts"), ({"k_starts": I32.short()}, "k_starts must be int32"), ({"k_lengths": I32}, "k_lengths"),
    ({"k_lengths": I32[:2].double()}, "k_lengths must be int32"), ({}, "device tensors"),
])
def test_packed_attention_names_what_is_wrong(change, text):
    q, k, v = tensors()
    a = {"q": q, "k": k, "v": v, "q_starts": I32, **change}
    more = {n: a.pop(n) for n in ("k_starts", "k_lengths") if n in a}
    with pytest.raises(ValueError, match=text):
        kernels.packed_attention(*a.values(), scale=1.0, **more)
    lse = torch.zeros(4, 10, 2)
    with pytest.raises(ValueError, match=text):
        kernels.packed_attention_backward(q, a["q"], a["k"], a["v"], q, lse, None, a["q_starts"], scale=1.0, **more)


@pytest.mark.parametrize("d", [0, 4, 20, 36, 136, 256])
def test_packed_attention_head_dim(d):
    q, k, v = tensors(d=d)
    with pytest.raises(ValueError, match=f"head_dim.*{d}"):
        kernels.packed_attention(q, k, v, I32, scale=1.0)


Q, K = torch.zeros(2, 4, 8, 32), torch.zeros(2, 2, 8, 32)
POS, FR = torch.zeros(1, 8, dtype=torch.int32), torch.ones(16, dtype=torch.float64)


@pytest.mark.parametrize("args,more,text", [
    ((Q.half(), K.half(), POS, FR), {}, "float32 or bfloat16"), ((Q, K.bfloat16(), POS, FR), {}, "k must be"),
    ((Q[0, 0], None, POS, FR), {}, "heads, tokens, width"), ((Q, K[:1], POS, FR), {}, "k must have shape"),
    ((Q, K, POS, FR.float()), {}, "frequencies must be"), ((Q, K, POS, FR[:6]), {}, "multiple of 4"),
    ((Q, K, POS, torch.ones(20, dtype=torch.float64)), {}, "at most half"), ((Q, K, POS.float(), FR), {}, "positions must be int32"),
    ((Q, K, POS[:, :7], FR), {}, "positions must have shape"), ((Q, K, POS, FR), {"sections": (8, 8)}, "positions must have shape"),
    ((Q, K, POS, FR), {"sections": (8, 4)}, "add up"), ((Q, K, POS, FR), {"sections": ()}, "add up"),
    ((Q, K, POS, FR), {"sections": (4, 4, 4, 2, 2)}, "add up"), ((Q, K, POS, FR), {"sections": (-4, 20)}, "add up"),
    ((Q, K, POS, FR), {"q_weight": torch.ones(16)}, "q_weight"), ((Q, K, POS, FR), {"k_weight": torch.ones(32).bfloat16()}, "k_weight"),
    ((Q, None, POS, FR), {"k_weight": torch.ones(32)}, "needs k"), ((torch.zeros(1, 8, 36), None, POS, FR), {}, "head_dim"),
    ((Q, K, POS, FR), {}, "device tensors"),
])
def test_head_norm_rotary_names_what_is_wrong(args, more, text):
    with pytest.raises(ValueError, match=text):
        kernels.head_norm_rotary(*args, **more)
    with pytest.raises(ValueError, match=text):
        kernels.head_norm_rotary_backward(args[0], args[1], *args, **more)


SOURCES = ["fjx_packed.hip", "fjx_packed_bwd.hip", "fjx_headnorm.hip"]


@pytest.mark.parametrize("src", SOURCES)
def test_no_scratch_and_no_spills(src):
    found = metadata(src)
    assert found
    for name, m in found.items():
        assert m["private_segment_fixed_size"] == 0 and m["vgpr_spill_count"] == 0 and m["sgpr_spill_count"] == 0, (name, m)


@pytest.mark.parametrize("more", [
    {"tokens_q": 1 << 61}, {"tokens_q": (1 << 29) - 64}, {"tokens_k": (1 << 31) - 512}, {"tokens_k": (1 << 31) - 1},
    {"sequences": (1 << 22) - 1, "tokens_q": (3 << 27)},
], ids=str)
def test_row_numbers_fit_32_bits(lib, more):
    """Rows are numbered in 32 bits, up to the end of a tile of 128 behind each sequence."""
    for call, a in ((lib.fjx_packed_attention_fwd, packed(**more)),
                    (lib.fjx_packed_attention_bwd, _lib.PackedAttentionBwdArgs(fwd=packed(**more)))):
        assert call(ctypes.byref(a), None) == 2
        assert "2^31" in lib.fjx_last_error().decode()
