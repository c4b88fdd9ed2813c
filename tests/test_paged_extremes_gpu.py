"""Attention over an e4m3 cache with queries near the largest numbers and keys as small: their scores are ordinary."""

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
