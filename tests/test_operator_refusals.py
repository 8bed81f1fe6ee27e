"""CPU check: what differential attention refuses by name before anything is
copied or launched."""

from __future__ import annotations

import pytest
import torch

from foldjax_amd import kernels


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d", [1, 16, 20, 36, 48, 128])
def test_head_dim(d, dtype):
    q, k = torch.zeros(2, 4, 8, d, dtype=dtype), torch.zeros(2, 2, 9, d, dtype=dtype)
    v, lam = torch.zeros(2, 1, 9, 2 * d, dtype=dtype), torch.zeros(4, 2, d)
    for call in (kernels.diff_attention, lambda *a, **m: kernels.diff_attention_backward(
            torch.zeros(2, 2, 8, 2 * d, dtype=dtype), *a, torch.zeros(2, 4, 8), **m)):
        with pytest.raises(ValueError, match=f"head_dim.*{d}"):
            call(q, k, v, lam, lambda_init=0.5, scale=1.0)
