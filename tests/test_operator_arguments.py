"""CPU checks of differential attention, RMS norm and dropout: what they refuse,
at the Python functions and at the C ABI (fake, never dereferenced pointers), their
struct layouts and workspace sizes, and the generator's known answers."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from foldjax_amd import _lib, kernels
from tests.philox import block

ROOT = Path(__file__).resolve().parent.parent
FAKE = 0x1000


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_struct_layout_matches_c(tmp_path):
    structs = {
        "fjx_diff_attention_args": _lib.DiffAttentionArgs,
        "fjx_diff_attention_bwd_args": _lib.DiffAttentionBwdArgs,
        "fjx_rms_norm_args": _lib.RmsNormArgs,
        "fjx_rms_norm_bwd_args": _lib.RmsNormBwdArgs,
        "fjx_dropout_args": _lib.DropoutArgs,
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


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_known_answers(counter, key, want):
    assert tuple(int(x) for x in block(np.array(counter, np.uint64), key)) == want


def diff(**more):
    a = _lib.DiffAttentionArgs(items=2, heads=4, kv_heads=2, nq=8, nk=16, head_dim=32, bias_share=1, dtype=1, scale=1.0,
                               q=FAKE, k=FAKE, v=FAKE, out=FAKE, lambda_vectors=FAKE)
    a.q_strides = _lib._i64x3(8 * 8 * 32, 8 * 32, 32)
    a.k_strides = _lib._i64x3(4 * 16 * 32, 16 * 32, 32)
    a.v_strides = _lib._i64x3(2 * 16 * 64, 16 * 64, 64)
    a.out_strides = _lib._i64x3(4 * 8 * 64, 8 * 64, 64)
    for name, value in more.items():
        setattr(a, name, _lib._i64x3(*value) if name.endswith("strides") else value)
    return a


DIFF_BAD = [
    (dict(items=0), "INVALID", "must be >= 1"), (dict(nq=0), "INVALID", "must be >= 1"), (dict(nk=0), "INVALID", ">= 1"),
    (dict(dtype=5), "INVALID", "dtype"), (dict(head_dim=48), "UNSUPPORTED", "head_dim"),
    (dict(heads=2048, kv_heads=2), "UNSUPPORTED", "heads"), (dict(kv_heads=3), "INVALID", "divide"),
    (dict(q=None), "INVALID", "NULL"), (dict(lambda_vectors=None), "INVALID", "NULL"), (dict(out=None), "INVALID", "NULL"),
    (dict(k=FAKE + 8), "INVALID", "16-byte"), (dict(q_strides=(2048, 256, 33)), "INVALID", "strides"),
    (dict(k_strides=(2048, 512, -32)), "INVALID", "strides"), (dict(out_strides=(0, 512, 64)), "INVALID", "strides"),
    (dict(bias=FAKE, bias_share=3), "INVALID", "bias_share"), (dict(bias=FAKE, bias_share=0), "INVALID", "bias_share"),
    (dict(bias=FAKE + 1), "INVALID", "bias"), (dict(bias=FAKE, bias_strides=(8, -1, 1)), "INVALID", "bias strides"),
    (dict(nk=2**31), "UNSUPPORTED", "2^31"), (dict(items=2**28), "UNSUPPORTED", "one launch"),
]


@pytest.mark.parametrize("more,code,text", DIFF_BAD, ids=lambda v: str(v)[:40])
def test_diff_attention_refusals(lib, more, code, text):
    want = getattr(_lib, f"FJX_ERR_{code}")
    assert lib.fjx_diff_attention_fwd(ctypes.byref(diff(**more)), None) == want
    assert text in lib.fjx_last_error().decode()
    b = _lib.DiffAttentionBwdArgs(fwd=diff(**{"out": None, "stats": FAKE, **{k: v for k, v in more.items() if k != "out"}}),
                                  dout=None if "out" in more else FAKE, dq=FAKE, dk=FAKE, dv=FAKE, dlambda=FAKE)
    b.dq_strides, b.dk_strides, b.dv_strides = b.fwd.q_strides, b.fwd.k_strides, b.fwd.v_strides
    if "out_strides" not in more:  # an input there: any stride will do
        assert lib.fjx_diff_attention_bwd(ctypes.byref(b), None) == want
        assert text in lib.fjx_last_error().decode()


def test_diff_attention_workspaces(lib):
    size = lib.fjx_diff_attention_workspace_size
    assert size(1, 6, 6, 37, 37, 32, 1) == 0  # one block of keys
    assert size(499, 2, 2, 499, 499, 32, 1) == 0  # rows enough without a split
    assert size(8, 8, 2, 1, 16384, 64, 1) >= 2 * 8 * 8 * 2 * (128 + 2) * 4  # two splits at least
    assert size(1, 6, 4, 37, 37, 32, 1) == 0 and size(1, 6, 6, 0, 37, 32, 1) == 0
    few = diff(items=1, heads=2, kv_heads=2, nq=1, nk=8192)
    assert lib.fjx_diff_attention_fwd(ctypes.byref(few), None) == _lib.FJX_ERR_WORKSPACE
    few.workspace, few.workspace_bytes = FAKE + 4, 1 << 40
    assert lib.fjx_diff_attention_fwd(ctypes.byref(few), None) == _lib.FJX_ERR_INVALID
    bwd = lib.fjx_diff_attention_bwd_workspace_size
    assert bwd(4, 6, 100, 100, 1, 1) == bwd(4, 6, 100, 100, 1, 0) >= 4 * 12 * 100 * 4
    assert bwd(64, 2, 100, 90, 64, 1) >= bwd(64, 2, 100, 90, 64, 0) + 2 * 100 * 90 * 4
    assert bwd(64, 2, 100, 90, 63, 1) == 0
    b = _lib.DiffAttentionBwdArgs(fwd=diff(stats=FAKE, out=None), dout=FAKE, dq=FAKE, dk=FAKE, dv=FAKE, dlambda=FAKE)
    b.dq_strides, b.dk_strides, b.dv_strides = b.fwd.q_strides, b.fwd.k_strides, b.fwd.v_strides
    call = lambda: lib.fjx_diff_attention_bwd(ctypes.byref(b), None)  # noqa: E731
    assert call() == _lib.FJX_ERR_WORKSPACE
    b.dbias = FAKE  # without a bias
    assert call() == _lib.FJX_ERR_INVALID
    b.dbias, b.dq_strides = None, _lib._i64x3(0, 256, 32)
    assert call() == _lib.FJX_ERR_INVALID
    b.dq_strides, b.fwd.stats = b.fwd.q_strides, None
    assert call() == _lib.FJX_ERR_INVALID
    assert lib.fjx_diff_attention_bwd(None, None) == lib.fjx_diff_attention_fwd(None, None) == _lib.FJX_ERR_INVALID


def test_backward_bias_rows_within_32_bits(lib):
    """The kernels address a tile's rows of the bias with 32 bits."""
    for bias_row, dbias_row, nq, code in ((2**23, 16, 8, "UNSUPPORTED"), (16, 2**23, 8, "UNSUPPORTED"),
                                          (2**23 - 1, 2**23 - 1, 8, "WORKSPACE"), (2**23, 2**23, 1, "WORKSPACE")):
        b = _lib.DiffAttentionBwdArgs(fwd=diff(nq=nq, stats=FAKE, out=None, bias=FAKE, bias_strides=(8, 8, bias_row)), dout=FAKE,
                                      dq=FAKE, dk=FAKE, dv=FAKE, dlambda=FAKE, dbias=FAKE)
        b.dq_strides, b.dk_strides, b.dv_strides = b.fwd.q_strides, b.fwd.k_strides, b.fwd.v_strides
        b.dbias_strides = _lib._i64x3(8, 8, dbias_row)
        assert lib.fjx_diff_attention_bwd(ctypes.byref(b), None) == getattr(_lib, f"FJX_ERR_{code}"), (bias_row, dbias_row)
        assert "2^23" in lib.fjx_last_error().decode() or code == "WORKSPACE"


def test_rms_norm_refusals(lib):
    ok = dict(rows=4, c=128, dtype=1, eps=1e-6, x=FAKE, weight=FAKE, out=2 * FAKE)
    for more, code in ((dict(rows=0), "INVALID"), (dict(c=12), "UNSUPPORTED"), (dict(c=8200), "UNSUPPORTED"),
                       (dict(dtype=7), "INVALID"), (dict(x=None), "INVALID"), (dict(out=FAKE + 8), "INVALID"),
                       (dict(codes=3), "INVALID"), (dict(codes=1), "INVALID"),  # no scales
                       (dict(codes=1, scales=FAKE, group=48), "UNSUPPORTED"),
                       (dict(codes=1, scales=FAKE, group=64, c=96), "UNSUPPORTED"),
                       (dict(codes=1, scales=FAKE, out=FAKE), "INVALID"), (dict(sum_out=2 * FAKE), "INVALID")):
        a = _lib.RmsNormArgs(**{**ok, **more})
        assert lib.fjx_rms_norm_fwd(ctypes.byref(a), None) == getattr(_lib, f"FJX_ERR_{code}"), more
    ok = dict(rows=4, c=128, dtype=1, eps=1e-6, dy=FAKE, h=FAKE, weight=FAKE, dx=FAKE, dweight=FAKE)
    for more, code in ((dict(rows=0), "INVALID"), (dict(c=12), "UNSUPPORTED"), (dict(h=None), "INVALID"),
                       (dict(dx=FAKE + 4), "INVALID"), ({}, "WORKSPACE")):
        a = _lib.RmsNormBwdArgs(**{**ok, **more})
        assert lib.fjx_rms_norm_bwd(ctypes.byref(a), None) == getattr(_lib, f"FJX_ERR_{code}"), more
    assert lib.fjx_rms_norm_bwd_workspace_size(0, 128) == lib.fjx_rms_norm_bwd_workspace_size(5, 12) == 0
    assert lib.fjx_rms_norm_bwd_workspace_size(5, 128) >= 128 * 4
    assert lib.fjx_rms_norm_fwd(None, None) == lib.fjx_rms_norm_bwd(None, None) == _lib.FJX_ERR_INVALID


def test_dropout_refusals(lib):
    ok = dict(batch=1, n=2, m=3, c=16, dtype=0, p=0.5, x=FAKE, out=FAKE)
    for more, code in ((dict(n=0), "INVALID"), (dict(c=12), "UNSUPPORTED"), (dict(c=0), "UNSUPPORTED"),
                       (dict(p=1.0), "INVALID"), (dict(p=-0.1), "INVALID"), (dict(p=float("nan")), "INVALID"),
                       (dict(shared=8), "INVALID"), (dict(x=None), "INVALID"), (dict(residual=FAKE + 4), "INVALID"),
                       (dict(step=FAKE + 4), "INVALID"), (dict(batch=2**48), "UNSUPPORTED"), (dict(dtype=9), "INVALID")):
        a = _lib.DropoutArgs(**{**ok, **more})
        assert lib.fjx_dropout_fwd(ctypes.byref(a), None) == getattr(_lib, f"FJX_ERR_{code}"), more
    assert lib.fjx_dropout_fwd(None, None) == _lib.FJX_ERR_INVALID


def cpu_attn(**more):
    bf = torch.bfloat16
    t = dict(q=torch.zeros(2, 3, 4, 8, 32, dtype=bf), k=torch.zeros(2, 3, 2, 9, 32, dtype=bf),
             v=torch.zeros(2, 3, 1, 9, 64, dtype=bf), lam=torch.zeros(4, 2, 32), bias=None, mask=None)
    t.update(more)
    return lambda: kernels.diff_attention(t["q"], t["k"], t["v"], t["lam"], lambda_init=0.5, scale=1.0, bias=t["bias"],
                                          mask=t["mask"])


def test_python_functions_refuse_by_name():
    z = lambda *s, **k: torch.zeros(*s, **{"dtype": torch.bfloat16, **k})  # noqa: E731
    for more, text in ((dict(q=z(2, 3, 3, 8, 32)), "even"), (dict(k=z(2, 3, 2, 9, 64)), "k must"),
                       (dict(v=z(2, 3, 2, 9, 64)), "v must"), (dict(k=z(2, 9, 32)), "as many axes"),
                       (dict(lam=torch.zeros(4, 4, 32)), "lambda_vectors"), (dict(lam=z(4, 2, 32)), "lambda_vectors"),
                       (dict(v=z(2, 3, 1, 9, 64, dtype=torch.float32)), "v must be"), (dict(q=z(2, 3, 4, 8, 32).half()), "float32 or bfloat16"),
                       (dict(bias=z(3, 8, 9)), "bias must be"), (dict(bias=z(1, 3, 2, 8, 9)), "one plane for each"),
                       (dict(bias=z(2, 2, 2, 8, 9)), "one plane for each"), (dict(bias=z(2, 1, 2, 8, 9).float()), "bias must be"),
                       (dict(mask=torch.ones(3, 2, 9)), "broadcast"), (dict(bias=z(2, 1, 2, 8, 9)), "device tensors"),
                       ({}, "device tensors")):
        with pytest.raises(ValueError, match=text):
            cpu_attn(**more)()
    x, w = z(4, 128), z(128)
    for call, text in (
        (lambda: kernels.rms_norm(x, w, codes="fp4"), "codes"), (lambda: kernels.rms_norm(x, z(64)), "weight"),
        (lambda: kernels.rms_norm(x, w.float()), "weight"), (lambda: kernels.rms_norm(x, w, residual=z(3, 128)), "residual"),
        (lambda: kernels.rms_norm(x, w, group=32), "group needs"), (lambda: kernels.rms_norm(x, w, sum_out=x), "sum_out"),
        (lambda: kernels.rms_norm(x, w), "device tensors"), (lambda: kernels.rms_norm_backward(z(3, 128), x, w), "dy"),
        (lambda: kernels.rms_norm_backward(x, x, w, dh=x.float()), "dh"),
        (lambda: kernels.dropout_add(x, p=0.1, seed=-1), "seed"), (lambda: kernels.dropout_add(x, p=0.1, seed=0, offset=2**64), "offset"),
        (lambda: kernels.dropout_add(x, p=0.1, seed=0, shared=(-3,)), "shared"),
        (lambda: kernels.dropout_add(x, p=0.1, seed=0, shared=(0,)), "shared"),
        (lambda: kernels.dropout_add(x, p=0.1, seed=0, step=torch.zeros(2, dtype=torch.int64)), "step"),
        (lambda: kernels.dropout_add(x, p=0.1, seed=0, residual=z(4, 64)), "residual"),
        (lambda: kernels.dropout_add(x, p=0.1, seed=0), "device tensors"),
    ):
        with pytest.raises(ValueError, match=text):
            call()
