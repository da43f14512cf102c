"""Refusals of the paged-cache operators that need no GPU."""
import math

import pytest
import torch

import rocm_attn_b200


@pytest.mark.parametrize("scale", [0.0, -0.125, -1.0, math.inf, -math.inf, math.nan, 1e-60, 1e39])
def test_scale_must_be_positive_and_finite(scale):
    # such a scale was taken as "not given"; it is refused before anything else of the call is looked at
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    q = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="scale must be"):
        rocm_attn_b200.attn_decode(q, k, k, t, n, scale=scale)
    for good in (None, 1e-30, 0.125, 3):
        with pytest.raises(RuntimeError, match="CUDA"):
            rocm_attn_b200.attn_decode(q, k, k, t, n, scale=good)
