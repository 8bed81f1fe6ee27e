"""Where the heads' norm with rotation writes, on the GPU: queries and keys that share a
buffer, in place, and the outputs that it refuses."""

from __future__ import annotations

import pytest
import torch

from foldjax_amd import kernels
from tests.gpu_util import say
from tests.test_gpu_head_norm_rotary import DTYPES, freqs, gen, places, weights

pytestmark = pytest.mark.gpu


def views(g, form, tokens, h, kv, d, dtype):
    """(buffer, queries, keys, values) of one projection's output."""
    n = h + 2 * kv
    if form == "tokens":
        x = torch.randn(tokens, n, d, generator=g, device="cuda").to(dtype)
        t = x.transpose(0, 1)
    else:
        x = torch.randn(n, tokens, d, generator=g, device="cuda").to(dtype)
        t = x
    return x, t[:h], t[h:h + kv], t[h + kv:]


@DTYPES
@pytest.mark.parametrize("form", ["tokens", "heads"])
@pytest.mark.parametrize("tokens", [1, 9, 600, 5000])
def test_in_place_of_a_shared_projection(tokens, form, dtype):
    say(f"rotary shared buffer {tokens} {form} {dtype}")
    h, kv, d = 8, 2, 128
    x, q, k, v = views(gen(tokens), form, tokens, h, kv, d, dtype)
    wq, wk = weights(gen(1), d, dtype)
    pos, fr = places(1, tokens), freqs(64)
    more = {"q_weight": wq, "k_weight": wk}
    want = kernels.head_norm_rotary(q.clone(), k.clone(), pos, fr, **more)
    values = v.clone()
    got = kernels.head_norm_rotary(q, k, pos, fr, q_out=q, k_out=k, **more)
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, values)


@DTYPES
def test_keys_that_are_heads_of_the_queries(dtype):
    """Read by both, written to neither: as from two buffers. Keys into the values' place."""
    say(f"rotary keys of the queries {dtype}")
    x, q, k, v = views(gen(2), "tokens", 9, 8, 2, 128, dtype)
    wq, wk = weights(gen(3), 128, dtype)
    pos, fr = places(1, 9), freqs(64)
    more = {"q_weight": wq, "k_weight": wk}
    want = kernels.head_norm_rotary(q.clone(), q[2:4].clone(), pos, fr, **more)
    got = kernels.head_norm_rotary(q, q[2:4], pos, fr, k_out=v, **more)
    assert torch.equal(got[0], want[0]) and got[1] is v and torch.equal(v, want[1])


@DTYPES
def test_outputs_over_other_inputs_are_refused(dtype):
    say(f"rotary refused places {dtype}")
    x, q, k, v = views(gen(4), "tokens", 9, 8, 2, 128, dtype)
    wq, wk = weights(gen(5), 128, dtype)
    pos, fr = places(1, 9), freqs(64)
    more = {"q_weight": wq, "k_weight": wk}
    before = x.clone()
    room = torch.zeros(12, 10, 128, dtype=dtype, device="cuda")
    same = torch.zeros(9, 8, 128, dtype=dtype, device="cuda").transpose(0, 1)
    for keys, outs in ((q[:2], {"k_out": q[:2]}), (q[2:4], {"k_out": q[2:4]}), (q, {"k_out": q}), (q, {"q_out": q}),
                       (k, {"k_out": q[6:]}), (k, {"q_out": x.transpose(0, 1)[2:10]}),
                       (k, {"q_out": room[:8, 1:], "k_out": room[7:9, 1:]}), (k, {"q_out": same, "k_out": same[3:5]})):
        with pytest.raises(ValueError, match="two buffers"):
            kernels.head_norm_rotary(q, keys, pos, fr, **outs, **more)
    tokens = torch.zeros(8, 10, 128, dtype=dtype, device="cuda")
    with pytest.raises(ValueError, match="two buffers"):  # a token on from its input
        kernels.head_norm_rotary(tokens[:, :9], None, pos, fr, q_weight=wq, q_out=tokens[:, 1:])
    assert torch.equal(x, before) and (room == 0).all() and (same == 0).all() and (tokens == 0).all()
