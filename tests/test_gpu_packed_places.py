"""Where packed attention writes, on the GPU: an output beside queries, keys and values
in one buffer, and the outputs that it refuses."""

from __future__ import annotations

import pytest
import torch

from foldjax_amd import kernels
from tests.gpu_util import say
from tests.test_gpu_packed_attention import ints, starts
from tests.test_gpu_packed_paths import DTYPES

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("form", ["tokens", "heads"])
def test_out_beside_its_inputs(form, dtype):
    say(f"packed one buffer {form} {dtype}")
    lens, h, kv, d = [40, 0, 25], 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(41)
    n = 2 * (h + kv)
    x = torch.randn(*((65, n) if form == "tokens" else (n, 65)), d, generator=g, device="cuda").to(dtype)
    t = x.transpose(0, 1) if form == "tokens" else x
    q, k, v, out = t[:h], t[h:h + kv], t[h + kv:h + 2 * kv], t[h + 2 * kv:]
    st, more = ints(starts(lens)), {"scale": 0.125, "causal": True}
    want, before = kernels.packed_attention(q, k, v, st, **more), t[:h + 2 * kv].clone()
    assert kernels.packed_attention(q, k, v, st, out=out, **more) is out
    assert torch.equal(out, want) and torch.equal(t[:h + 2 * kv], before)
    for over in (q, t[1:1 + h], t[h - 1:2 * h - 1], t[h + kv:2 * h + kv]):
        with pytest.raises(ValueError, match="out must not overlap"):
            kernels.packed_attention(q, k, v, st, out=over, **more)
    room = torch.zeros(h, 66, d, dtype=dtype, device="cuda")
    with pytest.raises(ValueError, match="out must not overlap"):  # a token on from the queries
        kernels.packed_attention(room[:, :65], k, v, st, out=room[:, 1:], **more)
    assert torch.equal(t[:h + 2 * kv], before) and (room == 0).all()
