"""Calls of the paged cache that are refused on the CPU, before a launch: at the C ABI with addresses that are never
dereferenced, and in Python."""

from __future__ import annotations

import pytest
import torch
from test_paged import E4M3_CODE, P, cache, lib, read, seqs, write  # noqa: F401
from test_paged_decoder import SMALL

from ako_b200.decoder import ModelConfig, PagedKVCache


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


@pytest.mark.parametrize("what,words", [
    ({"page_size": 0}, "page_size must be >= 1"), ({"page_size": -16}, "page_size must be >= 1"),
    ({"max_len": 0}, "max_len"), ({"batch": 0}, "batch"), ({"kv_dtype": torch.float32}, "kept as"),
    ({"kv_dtype": torch.float16}, "kept as"), ({"window": -1}, "window"), ({"sinks": -1}, "sinks")])
def test_a_paged_cache_of_the_decoder_that_could_not_be_used(what, words) -> None:
    """Refused when it is made, and not as a division by zero or at the first step."""
    made = {"batch": 2, "max_len": 16, "device": "cpu", "dtype": torch.bfloat16, **what}
    with pytest.raises(ValueError, match=words):
        PagedKVCache(ModelConfig(**SMALL), **made)
