"""The paged-cache operators without a GPU: what they refuse, at the C ABI and in Python, before any launch; and the
oracle's quantiser against torch's e4m3."""

from __future__ import annotations

import ctypes

import pytest
import torch
from paged_oracle import E4M3, Problem, attend, quantise, sees

from ako_b200 import _native, kv_cache_read_cuda_sm100, kv_cache_write_cuda_sm100, paged, paged_attention_cuda_sm100

P = 256  # an aligned address, never dereferenced: every call below fails or has nothing to do before a launch
BF16, F32, E4M3_CODE = 2, 0, 3


def cache(**kw) -> _native.PagedKVStruct:
    c = _native.PagedKVStruct(P, P, None, None, *([1024, 512, 64] * 2), *([0] * 6), 10, 2, 8, 64, BF16)
    for name, x in kw.items():
        setattr(c, name, x)
    return c


def seqs(**kw) -> _native.PagedBatchStruct:
    b = _native.PagedBatchStruct(P, P, None, 4, 3, 4, 1)
    for name, x in kw.items():
        setattr(b, name, x)
    return b


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        from ako_b200.build import build

        build()
    return _native.lib()


def write(lib, c, b, *, k=P, v=P, tokens=6, q_len=2, dtype=BF16, stride=128):
    return lib.ako_b200_kv_cache_write(k, 256, stride, 64, v, 256, 128, 64, c, b, tokens, q_len, dtype, None)


def read(lib, c, b, *, start=0, length=5, k=P, stride=64, dtype=BF16):
    return lib.ako_b200_kv_cache_read(c, b, start, length, k, 640, 320, stride, P, 640, 320, 64, dtype, None)


def attention(lib, c, b, *, q=P, out=P, tokens=6, q_len=2, heads=4, scale=0.1, window=0, sinks=0, work=P, size=1 << 40,
              dtype=BF16, stride=256):
    return lib.ako_b200_paged_attention(q, 512, stride, 64, c, b, tokens, q_len, heads, scale, window, sinks, out, 512,
                                        256, 64, work, size, dtype, None)


@pytest.mark.parametrize("call", [write, read, attention], ids=["write", "read", "attention"])
def test_caches_and_batches_that_every_call_refuses(lib, call) -> None:
    def refused(c, b, words, status=1, **kw):
        assert call(lib, c, b, **kw) == status
        assert words in lib.ako_b200_last_error(), lib.ako_b200_last_error()

    refused(None, seqs(), b"cache is a null pointer")
    refused(cache(), None, b"batch is a null pointer")
    refused(cache(k=None), seqs(), b"null pointer")
    refused(cache(v=P + 8), seqs(), b"16 bytes")
    refused(cache(k_stride_slot=60), seqs(), b"16 bytes")
    refused(cache(dtype=7), seqs(), b"dtype", 2)
    refused(cache(dtype=1), seqs(), b"differs")
    refused(cache(dtype=E4M3_CODE), seqs(), b"k_scale")
    refused(cache(head_dim=60), seqs(), b"head_dim")
    refused(cache(head_dim=136), seqs(), b"head_dim")
    refused(cache(head_dim=72, dtype=E4M3_CODE, k_scale=P, v_scale=P), seqs(), b"multiple of 16")
    for name in ("num_pages", "kv_heads", "page_size"):
        refused(cache(**{name: 0}), seqs(), b">= 1")
    refused(cache(num_pages=1 << 31), seqs(), b">= 1")
    refused(cache(), seqs(batch=-1), b"batch")
    refused(cache(), seqs(batch=65536), b"batch")
    refused(cache(), seqs(kv_lens=None), b"null pointer")
    refused(cache(), seqs(page_table=None), b"null pointer")
    refused(cache(), seqs(page_table_stride=3), b"page_table_stride")
    refused(cache(), seqs(max_pages=1 << 28), b"max_pages")
    refused(cache(), seqs(), b"dtype", 2, dtype=9)


def test_write_refusals(lib) -> None:
    for kw, words in (({"k": None}, b"null pointer"), ({"k": P + 2}, b"16 bytes"), ({"stride": 130}, b"16 bytes"),
                      ({"tokens": 5}, b"batch * q_len"), ({"tokens": -6, "q_len": -2}, b"tokens"),
                      ({"dtype": F32}, b"differs")):
        assert write(lib, cache(), seqs(), **kw) == 1
        assert words in lib.ako_b200_last_error()
    assert write(lib, cache(), seqs(cu_seqlens=P), tokens=1 << 31) == 1
    assert write(lib, cache(), seqs(cu_seqlens=P), tokens=1 << 30) == 1
    assert b"kv_heads" in lib.ako_b200_last_error()
    assert write(lib, cache(), seqs(), tokens=0, q_len=0) == 0
    assert write(lib, cache(), seqs(batch=0), tokens=0, q_len=2) == 0
    assert write(lib, cache(), seqs(max_pages=0, page_table=None)) == 0


def test_read_refusals(lib) -> None:
    for kw, words in (({"start": -1}, b"start"), ({"length": -1}, b"start"), ({"length": 1 << 31}, b"start"),
                      ({"length": 1 << 30}, b"batch * kv_heads"), ({"k": None}, b"null"), ({"k": P + 4}, b"16 bytes"),
                      ({"stride": 66}, b"16 bytes"), ({"dtype": F32}, b"differs")):
        assert read(lib, cache(), seqs(), **kw) == 1
        assert words in lib.ako_b200_last_error()
    assert read(lib, cache(), seqs(), length=0) == 0
    assert read(lib, cache(), seqs(batch=0)) == 0


def test_attention_refusals(lib) -> None:
    for kw, words in (({"heads": 3}, b"multiple of kv_heads"), ({"heads": 0}, b"multiple of kv_heads"),
                      ({"window": -1}, b"window"), ({"sinks": -1}, b"sinks"), ({"scale": float("nan")}, b"scale"),
                      ({"scale": float("inf")}, b"scale"), ({"scale": 1e39}, b"scale"), ({"q": None}, b"null"), ({"out": None}, b"null"),
                      ({"q": P + 8}, b"16 bytes"), ({"stride": 252}, b"16 bytes"), ({"work": None}, b"workspace"),
                      ({"work": P + 8}, b"workspace"), ({"size": 100}, b"workspace")):
        assert attention(lib, cache(), seqs(), **kw) == 1
        assert words in lib.ako_b200_last_error(), kw
    assert attention(lib, cache(dtype=F32), seqs(), dtype=F32) == 2
    assert b"fp16 or bf16" in lib.ako_b200_last_error()
    assert attention(lib, cache(), seqs(cu_seqlens=P), tokens=1 << 30) == 1
    assert b"q_heads" in lib.ako_b200_last_error()
    assert attention(lib, cache(), seqs(), tokens=0, q_len=0) == 0
    assert attention(lib, cache(), seqs(batch=0), tokens=0) == 0


def _plan(lib, c, b, tokens, q_len, heads):
    out = [ctypes.c_int(), ctypes.c_int(), ctypes.c_int(), ctypes.c_int64()]
    assert lib.ako_b200_paged_attention_plan(c, b, tokens, q_len, heads, BF16, *map(ctypes.byref, out)) == 0
    return tuple(x.value for x in out)


def test_plan_goes_by_the_rows_of_a_sequence(lib) -> None:
    assert _plan(lib, cache(), seqs(), 3, 1, 16)[:2] == (0, 8)
    assert _plan(lib, cache(), seqs(), 3, 1, 20)[:2] == (0, 16)
    assert _plan(lib, cache(), seqs(), 6, 2, 32)[:2] == (0, 32)
    assert _plan(lib, cache(), seqs(), 6, 2, 34)[:2] == (1, 256)
    assert _plan(lib, cache(), seqs(cu_seqlens=P, max_q_len=5), 30, 0, 14)[:2] == (1, 256)
    packed = seqs(cu_seqlens=P, max_q_len=4)
    assert _plan(lib, cache(), packed, 30, 0, 4)[:2] == (0, 8)
    kernel, rows, ctas, size = _plan(lib, cache(), seqs(), 3, 1, 16)
    assert size == ctas * (16 + 2 * rows * (2 + 64) * 4)
    assert lib.ako_b200_paged_attention_plan(cache(), seqs(), 3, 1, 16, BF16, None, None, None, None) == 1


def test_wrappers_refuse_cpu_tensors() -> None:
    k = torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="requires a CUDA tensor"):
        paged.PagedKV(k, k)
    with pytest.raises(ValueError, match="requires a CUDA tensor"):
        paged.PagedBatch(torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="requires a CUDA tensor"):
        kv_cache_write_cuda_sm100(k, k, None, None)
    with pytest.raises(ValueError, match="expected a PagedKV"):
        kv_cache_read_cuda_sm100(None, None, 0, 1)
    with pytest.raises(ValueError, match="requires a CUDA tensor"):
        paged_attention_cuda_sm100(k, None, None)


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU, so that the checks behind that one run here."""

    @property
    def is_cuda(self) -> bool:
        return True


def gpu(*shape, dtype=torch.bfloat16) -> torch.Tensor:
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnGpu)


def test_wrapper_checks() -> None:
    for bad in (lambda: paged.PagedKV(gpu(4, 2, 8, 64), gpu(4, 2, 8, 32)), lambda: paged.PagedKV(gpu(2, 8, 64), gpu(2, 8, 64)),
                lambda: paged.PagedKV(gpu(4, 2, 8, 64), gpu(4, 2, 8, 64, dtype=torch.float16)),
                lambda: paged.PagedKV(gpu(4, 2, 8, 60), gpu(4, 2, 8, 60)),
                lambda: paged.PagedKV(gpu(4, 2, 8, 256), gpu(4, 2, 8, 256)),
                lambda: paged.PagedKV(gpu(4, 2, 8, 128)[..., ::2], gpu(4, 2, 8, 64)),
                lambda: paged.PagedKV(gpu(4, 2, 8, 64, dtype=torch.int8), gpu(4, 2, 8, 64, dtype=torch.int8)),
                lambda: paged.PagedKV(gpu(4, 2, 8, 64), gpu(4, 2, 8, 64), gpu(4, 2, 8), gpu(4, 2, 8)),
                lambda: paged.PagedKV(gpu(4, 2, 8, 64, dtype=E4M3), gpu(4, 2, 8, 64, dtype=E4M3)),
                lambda: paged.PagedKV(gpu(4, 2, 8, 64, dtype=E4M3), gpu(4, 2, 8, 64, dtype=E4M3), gpu(4, 2, 8), gpu(4, 2, 8))):
        with pytest.raises(ValueError, match="PagedKV"):
            bad()
    i32 = torch.int32
    for bad in (lambda: paged.PagedBatch(gpu(3, 4, dtype=torch.int64), gpu(3, dtype=i32)),
                lambda: paged.PagedBatch(gpu(3, 4, dtype=i32).T, gpu(4, dtype=i32)),
                lambda: paged.PagedBatch(gpu(3, 4, dtype=i32), gpu(2, dtype=i32)),
                lambda: paged.PagedBatch(gpu(3, 4, dtype=i32), gpu(3, dtype=i32), cu_seqlens=gpu(3, dtype=i32)),
                lambda: paged.PagedBatch(gpu(3, 4, dtype=i32), gpu(3, dtype=i32), max_q_len=4),
                lambda: paged.PagedBatch(gpu(3, 4, dtype=i32), gpu(6, dtype=i32)[::2])):
        with pytest.raises(ValueError, match="PagedBatch"):
            bad()
    kv = paged.PagedKV(gpu(4, 2, 8, 64), gpu(4, 2, 8, 64))
    flat, ragged = (paged.PagedBatch(gpu(3, 4, dtype=i32), gpu(3, dtype=i32), cu_seqlens=cu)
                    for cu in (None, gpu(4, dtype=i32)))
    for bad in (lambda: kv_cache_write_cuda_sm100(gpu(3, 2, 2, 64), gpu(3, 2, 2, 32), kv, flat),
                lambda: kv_cache_write_cuda_sm100(gpu(2, 2, 2, 64), gpu(2, 2, 2, 64), kv, flat),
                lambda: kv_cache_write_cuda_sm100(gpu(3, 2, 3, 64), gpu(3, 2, 3, 64), kv, flat),
                lambda: kv_cache_write_cuda_sm100(gpu(3, 2, 2, 64), gpu(3, 2, 2, 64), kv, ragged),
                lambda: kv_cache_write_cuda_sm100(gpu(3, 2, 2, 64, dtype=torch.float16),
                                                  gpu(3, 2, 2, 64, dtype=torch.float16), kv, flat),
                lambda: kv_cache_read_cuda_sm100(kv, flat, -1, 4), lambda: kv_cache_read_cuda_sm100(kv, flat, 0, -4),
                lambda: kv_cache_read_cuda_sm100(kv, flat, 1 << 31, 4), lambda: kv_cache_read_cuda_sm100(kv, flat, 0, 1 << 64),
                lambda: kv_cache_read_cuda_sm100(kv, flat, 0, 4, dtype=torch.float16),
                lambda: kv_cache_read_cuda_sm100(kv, flat, 0, 4, out=(gpu(3, 2, 4, 64), gpu(3, 1, 4, 64).expand(3, 2, 4, 64))),
                lambda: paged_attention_cuda_sm100(gpu(3, 2, 4, 64), kv, flat, out=gpu(1, 2, 4, 64).expand(3, 2, 4, 64)),
                lambda: kv_cache_read_cuda_sm100(kv, flat, 0, 4, out=(gpu(3, 2, 4, 64), gpu(3, 2, 5, 64))),
                lambda: paged_attention_cuda_sm100(gpu(3, 2, 3, 64), kv, flat),
                lambda: paged_attention_cuda_sm100(gpu(3, 2, 0, 64), kv, flat),
                lambda: paged_attention_cuda_sm100(gpu(3, 2, 64), kv, flat),
                lambda: paged_attention_cuda_sm100(gpu(3, 2, 4, 64, dtype=torch.float32), kv, flat),
                lambda: paged_attention_cuda_sm100(gpu(3, 2, 4, 64), kv, flat, window=-1),
                lambda: paged_attention_cuda_sm100(gpu(3, 2, 4, 64), kv, flat, scale=float("nan")),
                lambda: paged_attention_cuda_sm100(gpu(3, 2, 4, 64), kv, flat, out=gpu(3, 2, 4, 32))):
        with pytest.raises(ValueError, match="cuda_sm100"):
            bad()


def test_oracle_quantiser_is_torchs_rounding() -> None:
    x = torch.randn(2000, 32, generator=torch.Generator().manual_seed(0)) * torch.exp2(torch.arange(2000) % 60 - 30.0)[:, None]
    y, s = quantise(x)
    assert torch.equal((x.double() / s[:, None]).float().to(E4M3).double(), y)
    top = x.abs().amax(-1).double()
    assert bool((top / s <= 448).all()) and bool((top / (s / 2) > 448).all())


def test_oracle_attention_is_a_softmax() -> None:
    p = Problem(torch.bfloat16, False, 4, 2, 16, 4, [(3, 10)], True, 1)
    out, bound = attend(p.q, p.k[0], p.v[0], p.v_scale[0], sees(3, 10, 0, 0), 0.25, torch.bfloat16, False)
    k, v = (t[0].repeat_interleave(2, 1).transpose(0, 1) for t in (p.k, p.v))
    want = torch.nn.functional.scaled_dot_product_attention(
        p.q.double().transpose(0, 1), k, v, attn_mask=sees(3, 10, 0, 0), scale=0.25).transpose(0, 1)
    torch.testing.assert_close(out, want, atol=1e-12, rtol=1e-12)
    assert bool((bound > 0).all()) and float(bound.max()) < 0.1
