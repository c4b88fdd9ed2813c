"""Paged key/value cache: writing, reading back, and attention over it.

The reference keeps one dense cache per layer and concatenates it at every
step (``ako/models/decoder.py:84-93``); it has no counterpart of these
operators, so they are not candidates of its dispatcher, and writing a cache
in place could not be one. They are called directly:

============================  ==========================================  =======================
op                            call                                        returns
============================  ==========================================  =======================
kv_cache_write                ``fn(k, v, cache, batch)``                  nothing; the cache holds k, v
kv_cache_read                 ``fn(cache, batch, start, length)``         dense ``(k, v)``
paged_attention               ``fn(q, cache, batch)``                     tensor like ``q``
============================  ==========================================  =======================

A :class:`PagedKV` is one layer's cache, a :class:`PagedBatch` says which
sequences a step runs and where their tokens lie; both check their tensors
once, keep them, and are passed to every call, so that a step of many layers
checks its page table once. Their contents may change in place between calls
and between replays of a captured graph.

Errors and streams are those of :mod:`ako_b200.kernels`: bad arguments raise
``ValueError`` (CPU tensors included), a failed launch ``RuntimeError``; every
call runs on the current stream of the tensors' device and can be captured.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from ako_b200 import _native
from ako_b200.kernels import _DTYPE_CODE, _DeviceGuard, _dtype_code, _require_cuda, _stream

#: Element type of a quantised cache (one fp32 scale per token and head).
E4M3 = torch.float8_e4m3fn
_E4M3_CODE = 3
#: Widest head the operators take.
MAX_HEAD_DIM = 128
#: Above every position and number of tokens.
_ENDLESS = (1 << 31) - 1


def _strides(t: torch.Tensor) -> tuple[int, ...]:
    """Strides, with those of axes of one element (which never matter) as 0."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride(), t.shape))


def _overlaps(t: torch.Tensor) -> bool:
    """Whether an output repeats its elements along an axis, so that which row is left there would be chance."""
    return any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape))


def _vectors(t: torch.Tensor) -> torch.Tensor:
    """``t`` with a contiguous last axis and all else on 16-byte boundaries, copied only if it is not so."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():  # rows of whole vectors, one behind the other
            return t
        each = 16 // t.element_size()
        if t.stride(-1) == 1 and all(s % each == 0 for s in _strides(t)[:-1]):
            return t
    out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
    return out.copy_(t)


class PagedKV:
    """One layer's paged cache.

    ``k`` and ``v``: ``(num_pages, kv_heads, page_size, head_dim)`` tensors of
    float32, float16, bfloat16 or, quantised, float8_e4m3fn, with a contiguous
    last axis and otherwise free strides (a cache laid out ``(num_pages,
    page_size, kv_heads, head_dim)`` is passed as its ``transpose(1, 2)``),
    all on 16-byte boundaries. ``k_scale`` and ``v_scale``: float32
    ``(num_pages, kv_heads, page_size)``, for a quantised cache only; a cached
    value stands for ``element * scale``, scales being positive. Attention takes
    a value's scale below 2^-100 for that, and those of the keys that a row sees
    should lie within 2^100 of one another: past 2^126 a key of the smaller ones
    is lost from the row's sum of weights. ``head_dim`` is a multiple of 8 (16
    when quantised) up to 128; attention takes float16 and bfloat16 queries.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None) -> None:
        fn = "PagedKV"
        _require_cuda(k, fn)
        if k.ndim != 4 or v.shape != k.shape:
            raise ValueError(f"{fn}: expected k and v of shape (num_pages, kv_heads, page_size, head_dim), "
                             f"got {tuple(k.shape)} and {tuple(v.shape)}")
        if v.dtype != k.dtype or v.device != k.device:
            raise ValueError(f"{fn}: v must match k in dtype and device")
        self.quantised = k.dtype == E4M3
        code = _E4M3_CODE if self.quantised else _dtype_code(k, "or float8_e4m3fn caches", fn)
        pages, heads, page_size, dim = k.shape
        if min(k.shape) < 1 or dim % (16 if self.quantised else 8) or dim > MAX_HEAD_DIM:
            raise ValueError(f"{fn}: head_dim must be a multiple of {16 if self.quantised else 8} up to {MAX_HEAD_DIM} "
                             f"and no axis empty, got {tuple(k.shape)}")
        for name, t in (("k", k), ("v", v)):
            if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s * t.element_size() % 16 for s in _strides(t)[:-1]):
                raise ValueError(f"{fn}: {name} needs a contiguous last axis and 16-byte aligned rows")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if (t is not None) != self.quantised:
                raise ValueError(f"{fn}: a float8_e4m3fn cache needs {name}" if self.quantised else
                                 f"{fn}: only a float8_e4m3fn cache takes {name}")
            if t is not None and (t.shape != k.shape[:3] or t.dtype != torch.float32 or t.device != k.device):
                raise ValueError(f"{fn}: {name} must be float32 {tuple(k.shape[:3])} on {k.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.dtype = k.device, k.dtype
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, page_size, dim
        scales = [(t.data_ptr(), _strides(t)) if t is not None else (None, (0, 0, 0)) for t in (k_scale, v_scale)]
        self._c = _native.PagedKVStruct(
            k.data_ptr(), v.data_ptr(), scales[0][0], scales[1][0], *_strides(k)[:3], *_strides(v)[:3],
            *scales[0][1], *scales[1][1], pages, heads, page_size, dim, code)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, page_size: int, head_dim: int, *, dtype: torch.dtype,
              device: torch.device | str = "cuda") -> "PagedKV":
        """A new cache of ``dtype`` (float8_e4m3fn for a quantised one), its contents undefined."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype != E4M3:
            return cls(k, v)
        return cls(k, v, *(torch.empty(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))


class PagedBatch:
    """The sequences of a step.

    ``page_table``: int32 ``(batch, max_pages)``, the pages of each sequence in
    order; ``kv_lens``: int32 ``(batch,)``, its tokens in the cache with the
    step's new ones. The new tokens are a sequence's last positions. Tensors of
    new tokens are ``(batch, q_len, heads, head_dim)``, every sequence having
    the same number, or, with ``cu_seqlens`` (int32 ``(batch + 1,)``),
    ``(tokens, heads, head_dim)`` in which sequence ``b`` owns the rows
    ``cu_seqlens[b]`` up to ``cu_seqlens[b + 1]``. ``max_q_len``: most new
    tokens of a sequence where ``cu_seqlens`` is given, for attention's choice of
    a kernel only. Without it that takes all of the call's tokens for those of
    one sequence, and a step of single tokens runs on the kernel for chunks: 69
    us in place of 47 for 32 sequences of 1500 to 2176 tokens (32 heads of 128, 8
    kv heads, bfloat16), 141 in place of 38 with an e4m3 cache.

    No call reads these tensors on the host. What they say is clamped to what
    there is: lengths to the table and to the tokens given; a page number
    outside the cache is a page that is not there, not written, read as zeros
    and seen by no token. New tokens of a length past the table that the table
    has no place for are not written. Rows behind ``cu_seqlens[-1]`` are left
    as they are.
    """

    def __init__(self, page_table: torch.Tensor, kv_lens: torch.Tensor, *, cu_seqlens: torch.Tensor | None = None,
                 max_q_len: int | None = None) -> None:
        fn = "PagedBatch"
        _require_cuda(page_table, fn)
        if page_table.ndim != 2 or page_table.dtype != torch.int32:
            raise ValueError(f"{fn}: page_table must be int32 (batch, max_pages), got {page_table.dtype} "
                             f"{tuple(page_table.shape)}")
        batch, pages = page_table.shape
        if pages > 1 and page_table.stride(1) != 1 or batch > 1 and page_table.stride(0) < pages:
            raise ValueError(f"{fn}: page_table needs contiguous rows")
        for name, t, n in (("kv_lens", kv_lens, batch), ("cu_seqlens", cu_seqlens, batch + 1)):
            if t is None and name == "cu_seqlens":
                continue
            if t.shape != (n,) or t.dtype != torch.int32 or t.device != page_table.device:
                raise ValueError(f"{fn}: {name} must be int32 ({n},) on {page_table.device}")
            if n > 1 and t.stride(0) != 1:
                raise ValueError(f"{fn}: {name} must be contiguous")
        if max_q_len is not None and (cu_seqlens is None or max_q_len < 1):
            raise ValueError(f"{fn}: max_q_len is a positive number given with cu_seqlens")
        self.page_table, self.kv_lens, self.cu_seqlens, self.max_q_len = page_table, kv_lens, cu_seqlens, max_q_len
        self.device, self.batch, self.max_pages = page_table.device, batch, pages
        self._most = _ENDLESS if max_q_len is None else min(max_q_len, _ENDLESS)
        self._c = _native.PagedBatchStruct(
            page_table.data_ptr(), kv_lens.data_ptr(), None if cu_seqlens is None else cu_seqlens.data_ptr(),
            page_table.stride(0) if batch > 1 else pages, batch, pages, self._most)
        self._ref = ctypes.byref(self._c)


def _check(cache: PagedKV, batch: PagedBatch, fn: str) -> None:
    if not isinstance(cache, PagedKV) or not isinstance(batch, PagedBatch):
        raise ValueError(f"{fn}: expected a PagedKV and a PagedBatch")
    if cache.device != batch.device:
        raise ValueError(f"{fn}: the cache is on {cache.device}, the batch on {batch.device}")


def _new_tokens(t: torch.Tensor, name: str, heads: int | None, cache: PagedKV, batch: PagedBatch,
                fn: str) -> tuple[torch.Tensor, int, int, tuple[int, int, int]]:
    """Checks a tensor of new tokens; returns it in 16-byte vectors, with (tokens, q_len, strides over batch, tokens
    and heads)."""
    shape = t.shape
    dims = 4 if batch.cu_seqlens is None else 3
    if (len(shape) != dims or shape[-1] != cache.head_dim or (heads is not None and shape[-2] != heads)
            or (dims == 4 and shape[0] != batch.batch)):
        want = f"({batch.batch}, q_len" if dims == 4 else "(tokens"
        raise ValueError(f"{fn}: expected {name} of shape {want}, {heads or 'heads'}, {cache.head_dim}), "
                         f"got {tuple(shape)}")
    if t.device != cache.device:
        raise ValueError(f"{fn}: {name} is on {t.device}, the cache on {cache.device}")
    if not cache.quantised and t.dtype != cache.dtype:
        raise ValueError(f"{fn}: {name} is {t.dtype}, the cache {cache.dtype}")
    t = _vectors(t)
    s = t.stride()
    if dims == 4:
        return t, shape[0] * shape[1], shape[1], (s[0], s[1], s[2])
    return t, shape[0], 0, (0, s[0], s[1])


def kv_cache_write_cuda_sm100(k: torch.Tensor, v: torch.Tensor, cache: PagedKV, batch: PagedBatch) -> None:
    """Store the new tokens' keys and values in the cache, in place.

    ``k`` and ``v``: ``(batch, q_len, kv_heads, head_dim)``, or ``(tokens,
    kv_heads, head_dim)`` with ``cu_seqlens``; strided views (the k and v parts
    of a packed projection) are read in place. Their dtype is the cache's, or
    any of the three activation dtypes for a quantised cache, which takes
    ``round(x / s)`` under the least power of two ``s`` that keeps the token's
    values of a head within e4m3's 448, and stores ``s`` with it. Tokens of one
    call must not share a slot; a cache expanded along an axis is refused.
    """
    fn = "kv_cache_write_cuda_sm100"
    _require_cuda(k, fn)
    _check(cache, batch, fn)
    code = _dtype_code(k, "k", fn)
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{fn}: v {tuple(v.shape)} {v.dtype} must match k {tuple(k.shape)} {k.dtype}")
    k, tokens, q_len, ks = _new_tokens(k, "k", cache.kv_heads, cache, batch, fn)
    v, _, _, vs = _new_tokens(v, "v", cache.kv_heads, cache, batch, fn)
    with _DeviceGuard(k.device):
        status = _native.active().ako_b200_kv_cache_write(
            k.data_ptr(), *ks, v.data_ptr(), *vs, cache._ref, batch._ref, tokens, q_len, code, _stream(k.device))
    if status:
        _native.raise_for_status(status, fn)


def kv_cache_read_cuda_sm100(
    cache: PagedKV, batch: PagedBatch, start: int, length: int, *, dtype: torch.dtype | None = None,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Positions ``start .. start + length - 1`` of every sequence as dense ``(k, v)``.

    Returns tensors of shape ``(batch, kv_heads, length, head_dim)``, zero
    behind a sequence's last position, in the cache's dtype, or for a quantised
    cache in ``dtype`` (one of the three activation dtypes), each value rounded
    once. ``out``: a pair of such tensors to write to, with a contiguous last
    axis, 16-byte aligned rows and otherwise free strides.
    """
    fn = "kv_cache_read_cuda_sm100"
    _check(cache, batch, fn)
    if dtype is None:
        dtype = out[0].dtype if out is not None else cache.dtype
    code = _DTYPE_CODE.get(dtype)
    if code is None:
        raise ValueError(f"{fn}: a quantised cache is read as float32/float16/bfloat16, got dtype {dtype}")
    if not cache.quantised and dtype != cache.dtype:
        raise ValueError(f"{fn}: a {cache.dtype} cache is read as such, got dtype {dtype}")
    if not (0 <= start <= _ENDLESS and 0 <= length <= _ENDLESS):
        raise ValueError(f"{fn}: start and length must be within 0 .. 2^31 - 1, got {start} and {length}")
    shape = (batch.batch, cache.kv_heads, length, cache.head_dim)
    if out is None:
        k = torch.empty(shape, dtype=dtype, device=cache.device)
        v = torch.empty(shape, dtype=dtype, device=cache.device)
    else:
        k, v = out
        for name, t in (("k", k), ("v", v)):
            if t.shape != shape or t.dtype != dtype or t.device != cache.device or t.stride(-1) != 1 or _overlaps(t):
                raise ValueError(f"{fn}: the output for {name} must be {dtype} {shape} on {cache.device} with a "
                                 f"contiguous last axis and no axis expanded")
    with _DeviceGuard(cache.device):
        status = _native.active().ako_b200_kv_cache_read(
            cache._ref, batch._ref, start, length, k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], code,
            _stream(cache.device))
    if status:
        _native.raise_for_status(status, fn)
    return k, v


#: Rows from which on the kernel, and with it the workspace, is always the same.
_MANY_ROWS = 1024


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(dtype: torch.dtype, dim: int, device: torch.device, code: int, rows: int) -> int:
    """Workspace of a call whose longest sequence has ``rows`` rows (new tokens times q heads per kv head): the rows,
    the types and the head's width alone decide it, so one token of a cache with one head stands for them."""
    p = 256  # an aligned address, never read
    quantised = dtype == E4M3
    kv = _native.PagedKVStruct(p, p, p if quantised else None, p if quantised else None, *([0] * 12), 1, 1, 16, dim,
                               _E4M3_CODE if quantised else _DTYPE_CODE[dtype])
    seqs = _native.PagedBatchStruct(p, p, None, 1, 1, 1, 1)
    kernel, tile, ctas, size = ctypes.c_int(), ctypes.c_int(), ctypes.c_int(), ctypes.c_int64()
    with _DeviceGuard(device):
        status = _native.active().ako_b200_paged_attention_plan(
            ctypes.byref(kv), ctypes.byref(seqs), 1, 1, rows, code, ctypes.byref(kernel), ctypes.byref(tile),
            ctypes.byref(ctas), ctypes.byref(size))
    _native.raise_for_status(status, "paged_attention_cuda_sm100")
    return size.value


def paged_attention_cuda_sm100(
    q: torch.Tensor, cache: PagedKV, batch: PagedBatch, *, scale: float | None = None, window: int = 0,
    sinks: int = 0, out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention of the new tokens over the cache, which already holds their keys and values.

    ``q``: ``(batch, q_len, q_heads, head_dim)``, or ``(tokens, q_heads,
    head_dim)`` with ``cu_seqlens``, float16 or bfloat16 (the cache's dtype
    unless it is quantised); ``q_heads`` is a multiple of the cache's
    ``kv_heads``, and head ``h`` attends to kv head ``h // (q_heads //
    kv_heads)``. ``scale`` defaults to ``head_dim ** -0.5``. With ``window`` w
    above 0 the token at position p sees the positions ``p - w + 1 .. p`` and,
    below them, the first ``sinks`` ones; pages that are neither may have been
    given away, their table entries set to -1. A row that sees nothing, or
    nothing with a score above minus infinity, is zero.

    Values that are infinite or NaN reach the rows that see them and no others.
    ``out``: where to write, with a contiguous last axis and 16-byte aligned
    rows; rows behind ``cu_seqlens[-1]`` are left as they are, which in a new
    output is undefined.
    """
    fn = "paged_attention_cuda_sm100"
    _require_cuda(q, fn)
    _check(cache, batch, fn)
    code = _DTYPE_CODE.get(q.dtype, 0)
    if code == 0:
        raise ValueError(f"{fn} supports float16/bfloat16 q, got {q.dtype}")
    q, tokens, q_len, qs = _new_tokens(q, "q", None, cache, batch, fn)
    heads = q.shape[-2]
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"{fn}: {heads} q heads are not a multiple of the cache's {cache.kv_heads} kv heads")
    if window < 0 or sinks < 0:
        raise ValueError(f"{fn}: window and sinks must be >= 0, got {window} and {sinks}")
    window, sinks = min(window, _ENDLESS), min(sinks, _ENDLESS)  # one that reaches behind every position is none
    if scale is None:
        scale = cache.head_dim ** -0.5
    elif not math.isfinite(scale):
        raise ValueError(f"{fn}: scale must be finite, got {scale}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(-1) != 1
          or _overlaps(out)):
        raise ValueError(f"{fn}: out must match q in shape, dtype and device and have a contiguous last axis and no "
                         f"axis expanded")
    os = out.stride()
    os = (os[0], os[1], os[2]) if batch.cu_seqlens is None else (0, os[0], os[1])
    most = q_len if batch.cu_seqlens is None else min(batch._most, tokens)
    rows = min(max(most, 1) * (heads // cache.kv_heads), _MANY_ROWS)
    size = _workspace_bytes(cache.dtype, cache.head_dim, cache.device, code, rows)
    work = torch.empty(size, dtype=torch.uint8, device=q.device)
    with _DeviceGuard(q.device):
        status = _native.active().ako_b200_paged_attention(
            q.data_ptr(), *qs, cache._ref, batch._ref, tokens, q_len, heads, scale, window, sinks,
            out.data_ptr(), *os, work.data_ptr(), size, code, _stream(q.device))
    if status:
        _native.raise_for_status(status, fn)
    return out


__all__ = ["E4M3", "MAX_HEAD_DIM", "PagedBatch", "PagedKV", "kv_cache_read_cuda_sm100", "kv_cache_write_cuda_sm100",
           "paged_attention_cuda_sm100"]
