"""Calls of the paged cache that are refused on the CPU, before a launch: at the C ABI with addresses that are never
dereferenced, and in Python."""

from __future__ import annotations

import pytest
from test_paged import E4M3_CODE, P, cache, lib, read, seqs, write  # noqa: F401


@pytest.mark.parametrize("stride", ["page", "head", "slot"])
@pytest.mark.parametrize("tensor", ["k", "v", "ks", "vs"])
def test_a_cache_that_repeats_its_elements_is_not_written(lib, tensor, stride) -> None:  # noqa: F811
    scales = dict(dtype=E4M3_CODE, k_scale=P, v_scale=P, ks_stride_page=16, ks_stride_head=8, ks_stride_slot=1,
                  vs_stride_page=16, vs_stride_head=8, vs_stride_slot=1) if tensor in ("ks", "vs") else {}
    assert write(lib, cache(**{**scales, f"{tensor}_stride_{stride}": 0}), seqs()) == 1
    assert b"repeats its elements" in lib.ako_b200_last_error()
    # nothing to write, or an axis of one element, whose stride plays no part
    assert write(lib, cache(**{**scales, f"{tensor}_stride_{stride}": 0}), seqs(), tokens=0, q_len=0) == 0
    one = {"page": {"num_pages": 1}, "head": {"kv_heads": 1}, "slot": {"page_size": 1}}[stride]
    assert write(lib, cache(**{**scales, **one, f"{tensor}_stride_{stride}": 0}), seqs(), k=None) == 1
    assert b"null pointer" in lib.ako_b200_last_error()
    # reading such a cache is allowed: the next refusal is another's
    assert read(lib, cache(**{**scales, f"{tensor}_stride_{stride}": 0}), seqs(), k=None) == 1
    assert b"k_out or v_out is a null pointer" in lib.ako_b200_last_error()
