"""Attention over an e4m3 cache with numbers far apart: queries near the largest ones and keys as small, whose scores
are ordinary, and values that differ by as much as the documentation allows."""

from __future__ import annotations

import pytest
import torch
from paged_oracle import Problem, check_attention

from ako_b200 import paged_attention_cuda_sm100

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 4, 8, 100], ids=["8rows", "16rows", "32rows", "many"])
@pytest.mark.parametrize("power", [118, -90])
def test_queries_and_keys_of_opposite_size(cuda_device, new, power) -> None:
    p = Problem(torch.bfloat16, True, 8, 2, 128, 16, [(new, 300), (new, new)], True, 71, cuda_device)
    p.q = (p.q.double() * 2.0**power).to(torch.bfloat16)
    p.caches["k_scale"] *= 2.0**-power
    for b in range(2):
        p.k[b] *= 2.0**-power
    check_attention(p, paged_attention_cuda_sm100(p.q.to(cuda_device), p.kv(), p.batch(new)))


@pytest.mark.parametrize("new", [1, 4, 8, 100], ids=["8rows", "16rows", "32rows", "many"])
@pytest.mark.parametrize("low,high", [(-50, 50), (-99, 0), (-30, 70)])
def test_value_scales_as_far_apart_as_is_stated(cuda_device, new, low, high) -> None:
    """Every third key's values 2^100 times the others': all keys' weights count in the sum."""
    p = Problem(torch.bfloat16, True, 8, 2, 128, 16, [(new, 300), (new, new + 2)], True, 72, cuda_device)
    for b, (_, kv) in enumerate(p.lengths):
        for j in range(kv):
            f = 2.0 ** (high if j % 3 == 2 else low + 1)
            p.caches["v_scale"][int(p.table[b, j // 16]), :, j % 16] *= f
            p.v[b][j] *= f
            p.v_scale[b][j] *= f
    check_attention(p, paged_attention_cuda_sm100(p.q.to(cuda_device), p.kv(), p.batch(new)))
