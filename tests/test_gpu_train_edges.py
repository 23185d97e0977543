"""Calls of layer norm, rotary positions and cross attention at the edges of what their documentation allows, on the GPU."""
import math

import pytest
import torch

from detectorfreesfm_amd import ops
from test_gpu_cross_attention import TYPES

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_gradient_of_no_query_heads_is_zero(built_lib):
    """dk and dv are sums over the query heads: of none, zeros, whatever the allocator's memory held before."""
    for t in TYPES:
        q, k = torch.empty((2, 3, 0, 32), dtype=t, device=DEV), torch.randn((2, 5, 2, 32), device=DEV).to(t)
        out, lse = ops.cross_attention(q, k, k)
        assert out.shape == q.shape and lse.shape == (2, 0, 3)
        junk = [torch.full_like(k, math.nan) for _ in range(8)]
        del junk
        dq, dk, dv = ops.cross_attention_backward(q, q, k, k, out, lse)
        assert dq.shape == q.shape and dk.shape == k.shape and dv.shape == k.shape
        assert bool((dk == 0).all()) and bool((dv == 0).all())
