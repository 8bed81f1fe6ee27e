"""The heads' norm with rotation without tokens or items, as packed attention takes it."""

from __future__ import annotations

import pytest
import torch

from foldjax_amd import kernels
from tests.gpu_util import say
from tests.test_gpu_head_norm_rotary import DTYPES, freqs, gen, heads, places, weights
from tests.test_gpu_packed_attention import ints

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("lead,tokens", [((), 0), ((3,), 0), ((0,), 7), ((2, 0), 1), ((0,), 0)])
@pytest.mark.parametrize("keys", [True, False], ids=["keys", "alone"])
def test_without_rows(lead, tokens, keys, dtype):
    """Outputs and gradients of the inputs' shapes; the weights' gradients are zeros."""
    say(f"rotary without rows {lead} {tokens} {keys} {dtype}")
    g = gen(1)
    q = heads(g, lead, 4, tokens, 32, dtype)
    k = heads(g, lead, 2, tokens, 32, dtype) if keys else None
    wq, wk = weights(g, 32, dtype)
    fr = freqs(16)
    for pos in (places(1, tokens, lead), places(1, tokens)):
        more = {"q_weight": wq, "k_weight": wk if keys else None}
        for _ in range(2):  # also of a layout that was seen
            y, yk = kernels.head_norm_rotary(q, k, pos, fr, **more)
            dq, dk, dwq, dwk = kernels.head_norm_rotary_backward(y, yk, q, k, pos, fr, **more)
            assert y.shape == dq.shape == q.shape and y.dtype == dq.dtype == dtype and (dwq == 0).all() and dwq.shape == (32,)
            if keys:
                assert yk.shape == dk.shape == k.shape and (dwk == 0).all() and dwk.shape == (32,)
            else:
                assert yk is None and dk is None and dwk is None
    assert kernels.head_norm_rotary(q, k, pos, fr, q_out=q, k_out=k, **more)[0] is q
    none = kernels.head_norm_rotary_backward(y, yk, q, k, pos, fr)
    assert none[2] is None and none[3] is None


@DTYPES
def test_attention_without_tokens(dtype):
    """Both operators of a sublayer, one after the other, on sequences of no tokens."""
    say(f"rotary and attention without tokens {dtype}")
    g = gen(2)
    q, k, v = (heads(g, (), n, 0, 64, dtype) for n in (8, 2, 2))
    wq, wk = weights(g, 64, dtype)
    pos, fr, st = places(1, 0), freqs(32), ints([0, 0, 0])
    qr, kr = kernels.head_norm_rotary(q, k, pos, fr, q_weight=wq, k_weight=wk)
    out, lse, rest = kernels.packed_attention(qr, kr, v, st, scale=0.125, return_lse=True)
    dq, dk, dv = kernels.packed_attention_backward(out, qr, kr, v, out, lse, rest, st, scale=0.125)
    dx, dxk, dwq, dwk = kernels.head_norm_rotary_backward(dq, dk, q, k, pos, fr, q_weight=wq, k_weight=wk)
    assert dx.shape == q.shape and dxk.shape == dv.shape == k.shape and (dwq == 0).all() and (dwk == 0).all()


def test_refusals_without_rows():
    say("rotary refusals without rows")
    q = torch.zeros(4, 0, 36, device="cuda")
    pos = places(1, 0)
    with pytest.raises(ValueError, match="head_dim"):
        kernels.head_norm_rotary(q, None, pos, freqs(16))
    with pytest.raises(ValueError, match="positions must have shape"):
        kernels.head_norm_rotary(q[..., :32], None, places(1, 3), freqs(16))
    with pytest.raises(ValueError, match="q_out must be"):
        kernels.head_norm_rotary(q[..., :32], None, pos, freqs(16), q_out=torch.zeros(4, 1, 32, device="cuda"))
