"""Waits of attention on the tensor cores that run out in the middle of their work (measurement build, limits of a few
polls): copies and products that are under way then are waited for before the kernel ends, so that what runs next is
as if nothing had happened."""

from __future__ import annotations

import pytest
import torch
from paged_oracle import Problem, check_attention

from ako_b200 import _native, paged_attention_cuda_sm100

pytestmark = pytest.mark.gpu

KINDS = [(torch.bfloat16, False, 16), (torch.bfloat16, False, 7), (torch.float16, True, 16)]
IDS = ["boxes", "copies", "e4m3"]
POLLS = [0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 64, 256]


def _limited(p: Problem, q, polls: int) -> tuple[torch.Tensor, int]:
    """The outputs under a limit of `polls` polls a wait, and whether a wait ran out."""
    lib = _native.active()
    try:
        lib.ako_b200_measure_set_wait_polls(polls)
        out = paged_attention_cuda_sm100(q, p.kv(), p.batch())
    finally:
        lib.ako_b200_measure_set_wait_polls(1 << 24)
    torch.cuda.synchronize()
    return out, _native.take_device_status()


def _problem(kind, device) -> Problem:
    dtype, quantised, page = kind
    return Problem(dtype, quantised, 8, 2, 128, page, [(300, 1500), (190, 190), (70, 900), (1, 40)], True, 41, device)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_calls_after_a_wait_that_ran_out_midway(cuda_device, kind) -> None:
    with _native.measurement():
        p = _problem(kind, cuda_device)
        q = p.q.to(cuda_device)
        want = paged_attention_cuda_sm100(q, p.kv(), p.batch())
        check_attention(p, want)
        for polls in POLLS:
            _limited(p, q, polls)
            assert torch.equal(paged_attention_cuda_sm100(q, p.kv(), p.batch()), want)
    assert _native.take_device_status() == 0


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_rows_are_right_or_nan_when_a_wait_runs_out_midway(cuda_device, kind) -> None:
    """Never sums that lack a tile: a row is what it always is, or NaN and the expiry is on record."""
    with _native.measurement():
        p = _problem(kind, cuda_device)
        q = p.q.to(cuda_device)
        want = paged_attention_cuda_sm100(q, p.kv(), p.batch())
        for polls in POLLS:
            out, expired = _limited(p, q, polls)
            nan = out.isnan().all(-1)
            assert bool(((out == want).all(-1) | nan).all()), f"{polls} polls"
            assert expired or not bool(nan.any()), f"{polls} polls"
    assert _native.take_device_status() == 0
