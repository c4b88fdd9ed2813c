"""The paged-cache kernels on a GPU against definitions in 64 bits.

Unused places of every cache hold NaN, pages lie in any order, and table entries behind a sequence's pages are -1."""

from __future__ import annotations

import math

import pytest
import torch
from paged_oracle import E4M3, HALF_STEP, Problem, attend, check_attention, quantise, sees

from ako_b200 import (PagedBatch, PagedKV, kv_cache_read_cuda_sm100, kv_cache_write_cuda_sm100,
                      paged_attention_cuda_sm100)

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
RAGGED = [(1, 1), (3, 70), (17, 17), (0, 40), (2, 129), (5, 64)]


def _bits(t: torch.Tensor) -> torch.Tensor:
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


# ------------------------------------------------------------------- write
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("quantised", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("dim,heads,page,packed,slots_first", [
    (128, 8, 16, True, False), (128, 2, 1, False, True), (80, 3, 7, True, True), (16, 1, 64, False, False),
    (64, 4, 32, True, False), (112, 5, 8, False, True)])
def test_write(cuda_device, dtype, quantised, dim, heads, page, packed, slots_first) -> None:
    lengths = RAGGED if packed else [(3, 3), (3, 50), (3, 65), (3, 2)]
    p = Problem(dtype, quantised, heads, heads, dim, page, lengths, packed, 3, cuda_device, slots_first)
    cache = p.kv()
    before = {n: None if t is None else t.clone() for n, t in p.caches.items()}
    kv_cache_write_cuda_sm100(p.k_new.to(cuda_device), p.v_new.to(cuda_device), cache, p.batch())
    for name, new in (("k", p.k_new), ("v", p.v_new)):
        want = before[name].cpu().clone()
        scale = before[name + "_scale"].cpu().clone() if quantised else None
        for b, (n, kv) in enumerate(lengths):
            rows = p.rows(new, b)
            if quantised:
                x, s = quantise(rows)
            for i in range(n):
                j = kv - n + i
                if j < 0:
                    continue
                at = int(p.table[b, j // page]), slice(None), j % page
                if quantised:
                    want.view(torch.uint8)[at] = x[i].float().to(E4M3).view(torch.uint8)
                    scale[at] = s[i].float()
                else:
                    want[at] = rows[i]
        assert torch.equal(_bits(p.caches[name].cpu()), _bits(want))
        if quantised:
            assert torch.equal(_bits(p.caches[name + "_scale"].cpu()), _bits(scale))


def test_write_every_e4m3_rounding(cuda_device) -> None:
    """Every finite bf16 value, in rows of sixteen consecutive ones and in rows next to 448 times a power of two; rows
    of zeros, infinities and NaN."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(torch.int16)
    x = bits.view(BF16)
    x = x[torch.isfinite(x)].clone()
    rows = torch.cat([x[: x.numel() // 16 * 16].view(-1, 16), x[torch.randperm(
        x.numel(), generator=torch.Generator().manual_seed(1))[: 16 * 2000]].view(-1, 16)])
    extra = torch.zeros(6, 16, dtype=BF16)
    extra[1, 3], extra[2, 5], extra[3, 7] = math.inf, -math.inf, math.nan
    extra[4] = 448.0
    extra[5], extra[5, 0] = 1e-30, 450.0
    extra[2, 0] = 3.0
    rows = torch.cat([rows, extra])
    n = len(rows)
    cache = PagedKV.empty(-(-n // 64), 1, 64, 16, dtype=E4M3, device=cuda_device)
    batch = PagedBatch(torch.arange(cache.num_pages, dtype=torch.int32, device=cuda_device)[None],
                       torch.tensor([n], dtype=torch.int32, device=cuda_device))
    k = rows.view(1, n, 1, 16).to(cuda_device)
    kv_cache_write_cuda_sm100(k, k, cache, batch)
    want, scale = quantise(rows)
    got = cache.k.float().cpu().view(-1, 16)[:n].double()
    assert torch.equal(cache.k_scale.cpu().view(-1)[:n].double(), scale)
    assert torch.equal(torch.nan_to_num(got, nan=9e9), torch.nan_to_num(want, nan=9e9))
    assert torch.equal(_bits(cache.k.cpu())[:, 0].reshape(-1, 16)[:n], _bits(cache.v.cpu())[:, 0].reshape(-1, 16)[:n])


def test_write_skips_what_is_not_there(cuda_device) -> None:
    """Pages outside the cache, lengths that pass the table or do not reach, offsets that pass the tokens, and rows
    behind the last sequence."""
    p = Problem(BF16, False, 2, 2, 64, 8, [(4, 20), (4, 30), (4, 9)], True, 5, cuda_device)
    p.table[0, 2] = 1000
    p.table[1, 3] = -7
    p.kv_lens[2] = 10_000  # past the table's four pages
    p.cu[3] = 11  # the last row belongs to nobody
    before = p.caches["k"].clone()
    kv_cache_write_cuda_sm100(p.k_new.to(cuda_device), p.v_new.to(cuda_device), p.kv(), p.batch())
    want = before.cpu().clone()
    for j, i in ((16, 0), (17, 1), (18, 2), (19, 3)):
        assert int(p.table[0, j // 8]) == 1000, i
    for i in range(4):  # sequence 1 holds positions 26 .. 29, page 3: not there
        assert (26 + i) // 8 == 3
    for i in range(3):  # clamped to 32 positions: 29 .. 31 in page 3, which is -1
        assert int(p.table[2, (29 + i) // 8]) == -1
    assert torch.equal(_bits(p.caches["k"].cpu()), _bits(want))


# -------------------------------------------------------------------- read
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("quantised", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("dim,heads,page,start,length,slots_first", [
    (128, 8, 16, 0, 129, False), (80, 3, 7, 5, 61, True), (16, 1, 64, 0, 1, False), (64, 4, 1, 128, 200, False),
    (112, 2, 8, 3, 1000, True)])
def test_read(cuda_device, dtype, quantised, dim, heads, page, start, length, slots_first) -> None:
    p = Problem(dtype, quantised, heads, heads, dim, page, RAGGED, True, 7, cuda_device, slots_first)
    got = kv_cache_read_cuda_sm100(p.kv(), p.batch(), start, length, dtype=dtype)
    for out, rows in zip(got, (p.k, p.v)):
        want = torch.zeros(len(RAGGED), heads, length, dim, dtype=torch.float64)
        for b, (_, kv) in enumerate(RAGGED):
            n = max(0, min(length, kv - start))
            want[b, :, :n] = rows[b][start:start + n].transpose(0, 1)
        assert out.dtype == dtype
        assert torch.equal(out.cpu(), want.to(dtype))  # element * scale fits every activation type exactly, or rounds once


def test_read_into_strided_outputs(cuda_device) -> None:
    p = Problem(F16, True, 2, 2, 64, 16, [(1, 33), (1, 5)], True, 8, cuda_device)
    k = torch.full((2, 40, 2, 64), 7.0, dtype=F16, device=cuda_device)
    v = torch.full((2, 2, 48, 64), 7.0, dtype=F16, device=cuda_device)
    out = (k.transpose(1, 2)[:, :, 2:38], v[:, :, :36])
    got = kv_cache_read_cuda_sm100(p.kv(), p.batch(), 0, 36, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    ref = kv_cache_read_cuda_sm100(p.kv(), p.batch(), 0, 36, dtype=F16)
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
    assert bool((k[:, :2] == 7).all()) and bool((k[:, 38:] == 7).all()) and bool((v[:, :, 36:] == 7).all())


def test_read_of_pages_that_are_not_there(cuda_device) -> None:
    p = Problem(BF16, False, 1, 1, 32, 4, [(1, 12)], True, 9, cuda_device)
    p.table[0, 1] = p.num_pages
    k, _ = kv_cache_read_cuda_sm100(p.kv(), p.batch(), 0, 12)
    assert bool((k[0, 0, 4:8] == 0).all())
    assert torch.equal(k[0, 0, :4].cpu().double(), p.k[0][:4, 0]) and torch.equal(k[0, 0, 8:].cpu().double(), p.k[0][8:, 0])


# --------------------------------------------------------------- attention
CACHES = [(BF16, False), (F16, False), (BF16, True), (F16, True)]
CACHE_IDS = ["bf16", "f16", "bf16-e4m3", "f16-e4m3"]


def _run(p: Problem, max_q_len=None, **kw) -> torch.Tensor:
    return paged_attention_cuda_sm100(p.q.to(p.device), p.kv(), p.batch(max_q_len), **kw)


@pytest.mark.parametrize("dtype,quantised", CACHES, ids=CACHE_IDS)
@pytest.mark.parametrize("heads,dim,page", [((8, 8), 128, 16), ((8, 2), 128, 1), ((5, 1), 64, 64), ((16, 1), 80, 7),
                                            ((12, 2), 32, 8), ((40, 2), 96, 16), ((2, 2), 16, 128)])
def test_attention_single_tokens(cuda_device, dtype, quantised, heads, dim, page) -> None:
    p = Problem(dtype, quantised, *heads, dim, page, [(1, n) for n in (1, 2, 63, 64, 65, 300, 17)], False, 11, cuda_device)
    check_attention(p, _run(p))


@pytest.mark.parametrize("dtype,quantised", CACHES, ids=CACHE_IDS)
@pytest.mark.parametrize("heads,dim,page,lengths", [
    ((8, 2), 128, 16, RAGGED),
    ((4, 4), 64, 5, [(33, 33), (1, 200), (64, 190), (100, 100)]),
    ((6, 2), 112, 32, [(129, 300), (1, 1), (7, 7)]),
    ((16, 2), 128, 64, [(2, 9), (70, 500)]),
    ((1, 1), 48, 16, [(300, 301)]),
])
def test_attention_chunks(cuda_device, dtype, quantised, heads, dim, page, lengths) -> None:
    p = Problem(dtype, quantised, *heads, dim, page, lengths, True, 12, cuda_device, slots_first=page == 5)
    check_attention(p, _run(p))
    check_attention(p, _run(p, max_q_len=max(n for n, _ in lengths)))


@pytest.mark.parametrize("dtype,quantised", [(BF16, False), (F16, True)], ids=["bf16", "f16-e4m3"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (63, 1), (64, 100), (100, 0), (1000, 3), (5, 7)])
def test_attention_window_and_sinks(cuda_device, dtype, quantised, window, sinks) -> None:
    p = Problem(dtype, quantised, 4, 2, 64, 16, [(1, 500), (1, 3), (40, 333), (130, 130), (1, 64), (9, 700)], True, 13,
                cuda_device)
    check_attention(p, _run(p, window=window, sinks=sinks), window=window, sinks=sinks)
    single = Problem(dtype, quantised, 4, 2, 64, 16, [(1, n) for n in (500, 3, 64, 65, 1000)], False, 13, cuda_device)
    check_attention(single, _run(single, window=window, sinks=sinks), window=window, sinks=sinks)


def test_attention_with_pages_given_away(cuda_device) -> None:
    """Pages behind the window and past the sinks may be -1 or hold anything, NaN too."""
    p = Problem(BF16, False, 4, 2, 64, 16, [(1, 500), (20, 400)], True, 14, cuda_device)
    want = _run(p, window=50, sinks=3)
    first = [500 - 1 - 50 + 1, 400 - 20 - 50 + 1]
    for b in range(2):
        for i in range(1, first[b] // 16):
            p.caches["k"][int(p.table[b, i])] = math.nan
            p.caches["v"][int(p.table[b, i])] = math.inf
            p.table[b, i] = -1 if i % 2 else 10_000
    assert torch.equal(_run(p, window=50, sinks=3), want)
    check_attention(p, want, window=50, sinks=3)


@pytest.mark.parametrize("more", [0, 150], ids=["few", "many"])
@pytest.mark.parametrize("quantised", [False, True], ids=["same", "e4m3"])
def test_attention_rows_without_keys_are_zero(cuda_device, quantised, more) -> None:
    """More new tokens than cached ones, no cached ones, no new ones, and only pages that are not there."""
    n = 5 + more
    p = Problem(BF16, quantised, 4, 2, 64, 16, [(n, n), (3, 3), (0, 9), (2, 10)], True, 15, cuda_device)
    p.kv_lens[0] = 2  # all rows but two before the first position
    p.kv_lens[1] = 0
    p.table[3, 0] = -1
    out = _run(p).cpu()
    assert bool((out[: n - 2] == 0).all()) and bool((out[n:] == 0).all())
    want, bound = attend(p.q[n - 2:n], p.k[0][:2], p.v[0][:2], p.v_scale[0][:2], sees(2, 2, 0, 0), 64**-0.5, BF16, quantised)
    assert bool(((out[n - 2:n].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("new", [2, 100], ids=["few", "many"])
def test_attention_clamps_what_it_is_told(cuda_device, new) -> None:
    """Lengths past the table, negative ones and offsets past the tokens: what there is is attended, nothing else is
    touched."""
    p = Problem(BF16, False, 4, 2, 64, 16, [(new, 160), (new, 160), (new, 160), (new, 160)], True, 27, cuda_device)
    want = _run(p)
    p.kv_lens[0] = 2_000_000_000  # the table holds 160 positions
    p.kv_lens[1] = -5
    p.cu[4] = 1_000_000
    out = torch.full((4 * new + 3, 4, 64), 9.0, dtype=BF16, device=cuda_device)
    q = torch.cat([p.q.to(cuda_device), torch.zeros(3, 4, 64, dtype=BF16, device=cuda_device)])
    p.cu[3] = 2 * new  # the third sequence has no new tokens, the fourth all the others
    paged_attention_cuda_sm100(q, p.kv(), p.batch(), out=out)
    assert torch.equal(out[:new], want[:new])
    assert bool((out[new:2 * new] == 0).all())
    assert torch.isfinite(out).all() and not bool((out[2 * new:] == 9).all(-1).any())
    p.cu[:] = torch.tensor([4 * new, 3, -9, 2 * new, 2 * new])  # in no order
    out.fill_(9.0)
    paged_attention_cuda_sm100(q, p.kv(), p.batch(), out=out)
    assert bool((out[2 * new:] == 9).all())


def test_max_q_len_chooses_a_kernel_and_bounds_nothing(cuda_device) -> None:
    p = Problem(BF16, False, 8, 2, 64, 16, [(70, 300), (1, 40), (9, 9)], True, 28, cuda_device)
    check_attention(p, _run(p, max_q_len=1))
    check_attention(p, _run(p, max_q_len=1000))


@pytest.mark.parametrize("quantised", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("new", [1, 4, 40])
def test_attention_nonfinite_values_stay_with_the_rows_that_see_them(cuda_device, quantised, new) -> None:
    p = Problem(F16, quantised, 4, 2, 64, 16, [(new, 90), (new, 70)], True, 16, cuda_device)
    odd = [(80, 3, math.nan)] if quantised else [(80, 3, math.nan), (75, 9, math.inf), (88, 9, -math.inf), (70, 1, math.inf)]
    for j, d, x in odd:
        at = int(p.table[0, j // 16]), 1, j % 16, d
        if quantised:
            p.caches["v"].view(torch.uint8)[at] = 0x7F
        else:
            p.caches["v"][at] = x
        p.v[0][j, 1, d] = x
    at = int(p.table[1, 4]), 0, 69 - 64  # the last key of the second sequence: only its last row sees it
    if quantised:
        p.caches["k"].view(torch.uint8)[at][7] = 0x7F
    else:
        p.caches["k"][at][7] = math.nan
    out = _run(p)
    second = p.rows(out, 1).cpu()
    assert bool(second[-1, :2].isnan().all()) and bool(torch.isfinite(second[:-1]).all())
    p.lengths = p.lengths[:1]
    p.cu = p.cu[:2]
    check_attention(p, out)


@pytest.mark.parametrize("new", [1, 40], ids=["few", "many"])
def test_attention_rows_whose_scores_are_all_minus_infinity_are_zero(cuda_device, new) -> None:
    """Of the first sequence's rows only the last key is infinite, of the second's all are."""
    p = Problem(BF16, False, 4, 2, 64, 16, [(new, new), (new, new)], True, 17, cuda_device)
    p.q[..., 0] = -1.0
    for j in range(new):
        for b in range(2):
            p.caches["k"][int(p.table[b, j // 16]), :, j % 16] = 0.0
            p.caches["k"][int(p.table[b, j // 16]), :, j % 16, 0] = math.inf if b == 1 or j == new - 1 else 0.0
    # infinity times the other columns' zeros of k is none: a score is that of column 0
    out = _run(p)
    assert bool((p.rows(out, 1) == 0).all())
    first = p.rows(out, 0)
    assert bool(torch.isfinite(first).all())
    if new > 1:  # the last row: the mean of the values before its own
        want = p.v[0][: new - 1].mean(0).repeat_interleave(2, 0)
        bound = (2 * HALF_STEP[BF16] + 2.0**-20) * p.v[0].abs().amax()
        assert bool(((first[-1].double().cpu() - want).abs() <= bound).all())


def test_windows_that_reach_behind_everything_are_none(cuda_device) -> None:
    p = Problem(BF16, False, 4, 2, 64, 16, [(40, 90), (1, 70)], True, 18, cuda_device)
    want = _run(p)
    for window, sinks in ((1 << 31, 0), (1 << 70, 5), (90, 1 << 70), ((1 << 64) + 5, 0)):
        assert torch.equal(_run(p, window=window, sinks=sinks), want)


def test_attention_large_scores_and_scales(cuda_device) -> None:
    """Scores of hundreds (weights of all but one key underflow), a negative scale, and keys' and values' scales far
    apart."""
    p = Problem(F16, False, 4, 2, 64, 16, [(3, 150), (1, 400)], True, 17, cuda_device, spread=20.0)
    for scale in (1.0, -0.25, 0.0, 1e-60):
        check_attention(p, _run(p, scale=scale), scale=scale)
    p = Problem(F16, False, 4, 2, 64, 16, [(60, 150), (33, 400)], True, 17, cuda_device, spread=20.0)
    for scale in (1.0, -0.25, 0.0, 1e-60):
        check_attention(p, _run(p, scale=scale), scale=scale)
    for lengths in ([(3, 150), (1, 400)], [(60, 150), (33, 400)]):
        p = Problem(BF16, True, 4, 2, 64, 16, lengths, True, 18, cuda_device)
        for b, (_, kv) in enumerate(p.lengths):
            for j in range(kv):
                f = 2.0 ** ((j * 7) % 40 - 20)
                at = int(p.table[b, j // 16]), slice(None), j % 16
                p.caches["v_scale"][at] *= f
                p.v[b][j] *= f
                p.v_scale[b][j] *= f
        check_attention(p, _run(p))


def test_attention_of_strided_queries_into_strided_outputs(cuda_device) -> None:
    p = Problem(BF16, False, 4, 2, 64, 16, [(3, 50), (3, 60)], False, 19, cuda_device)
    want = _run(p)
    packed = torch.randn(2, 3, 9, 64, device=cuda_device).to(BF16)
    packed[:, :, 2:6] = p.q.to(cuda_device)
    out = torch.full((2, 5, 8, 64), 3.0, dtype=BF16, device=cuda_device)
    view = out[:, 1:4, ::2]
    assert paged_attention_cuda_sm100(packed[:, :, 2:6], p.kv(), p.batch(), out=view) is view
    assert torch.equal(view, want)
    assert bool((out[:, 0] == 3).all()) and bool((out[:, 4] == 3).all()) and bool((out[:, :, 1::2] == 3).all())
    odd = torch.randn(2, 3, 4, 68, device=cuda_device).to(BF16)  # rows that are not on 16-byte boundaries
    odd[..., :64] = p.q.to(cuda_device)
    assert torch.equal(paged_attention_cuda_sm100(odd[..., :64], p.kv(), p.batch()), want)


@pytest.mark.parametrize("new", [3, 90], ids=["few", "many"])
def test_rows_behind_the_last_sequence_are_left(cuda_device, new) -> None:
    p = Problem(BF16, False, 4, 2, 64, 16, [(new, 100), (2, 60)], True, 20, cuda_device)
    want = _run(p)
    q = torch.cat([p.q.to(cuda_device), torch.full((4, 4, 64), math.nan, dtype=BF16, device=cuda_device)])
    out = torch.full_like(q, 5.0)
    paged_attention_cuda_sm100(q, p.kv(), p.batch(), out=out)
    assert torch.equal(out[: new + 2], want) and bool((out[new + 2:] == 5).all())


def test_many_sequences(cuda_device) -> None:
    """More sequences than a CTA has threads, of very different lengths, some without new tokens."""
    lengths = [(1 if b % 7 else 0, 1 + (b * 37) % 90) for b in range(700)]
    lengths[333] = (1, 3000)
    p = Problem(BF16, True, 4, 2, 32, 16, lengths, True, 21, cuda_device)
    check_attention(p, _run(p, max_q_len=1))
    kv_cache_write_cuda_sm100(p.k_new.to(cuda_device), p.v_new.to(cuda_device), p.kv(), p.batch())
    k, _ = kv_cache_read_cuda_sm100(p.kv(), p.batch(), 0, 3000, dtype=BF16)
    for b in (1, 333, 698):
        x, s = quantise(p.rows(p.k_new, b))
        assert torch.equal(k[b, :, lengths[b][1] - 1].cpu().double(), (x * s[..., None])[0])


def test_nothing_to_do(cuda_device) -> None:
    cache = PagedKV.empty(2, 2, 16, 64, dtype=BF16, device=cuda_device)
    none = PagedBatch(torch.zeros(0, 3, dtype=torch.int32, device=cuda_device),
                      torch.zeros(0, dtype=torch.int32, device=cuda_device))
    x = torch.zeros(0, 1, 2, 64, dtype=BF16, device=cuda_device)
    kv_cache_write_cuda_sm100(x, x, cache, none)
    assert paged_attention_cuda_sm100(x, cache, none).shape == x.shape
    assert kv_cache_read_cuda_sm100(cache, none, 0, 5)[0].shape == (0, 2, 5, 64)
    one = PagedBatch(torch.zeros(1, 3, dtype=torch.int32, device=cuda_device),
                     torch.zeros(1, dtype=torch.int32, device=cuda_device))
    x = torch.zeros(1, 0, 2, 64, dtype=BF16, device=cuda_device)
    kv_cache_write_cuda_sm100(x, x, cache, one)
    assert paged_attention_cuda_sm100(x, cache, one).shape == x.shape
    assert kv_cache_read_cuda_sm100(cache, one, 0, 0)[0].shape == (1, 2, 0, 64)
    bare = PagedBatch(torch.zeros(1, 0, dtype=torch.int32, device=cuda_device),
                      torch.ones(1, dtype=torch.int32, device=cuda_device))
    q = torch.ones(1, 1, 2, 64, dtype=BF16, device=cuda_device)
    kv_cache_write_cuda_sm100(q, q, cache, bare)
    assert bool((paged_attention_cuda_sm100(q, cache, bare) == 0).all())
    assert bool((kv_cache_read_cuda_sm100(cache, bare, 0, 2)[0] == 0).all())


@pytest.mark.parametrize("new", [1, 40], ids=["few", "many"])
def test_offsets_beyond_32_bits(cuda_device, new) -> None:
    """A cache of 2^32 + elements: its last pages lie behind 2^31 elements and 2^32 bytes."""
    pages, heads, page, dim = 33_000, 8, 64, 128  # 2.16e9 elements, 4.3 GB each in bf16
    k = torch.empty(pages, heads, page, dim, dtype=BF16, device=cuda_device)
    cache = PagedKV(k, torch.empty_like(k))
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device=cuda_device)
    batch = PagedBatch(table, torch.tensor([150], dtype=torch.int32, device=cuda_device))
    g = torch.Generator().manual_seed(2)
    new_k, new_v = (torch.randn(1, 150, heads, dim, generator=g).to(BF16) for _ in range(2))
    kv_cache_write_cuda_sm100(new_k.to(cuda_device), new_v.to(cuda_device), cache, batch)
    got_k, got_v = kv_cache_read_cuda_sm100(cache, batch, 0, 150)
    assert torch.equal(got_k[0].transpose(0, 1).cpu(), new_k[0]) and torch.equal(got_v[0].transpose(0, 1).cpu(), new_v[0])
    assert torch.equal(k[pages - 2, :, 21].cpu(), new_k[0, 149])
    q = torch.randn(1, new, heads, dim, generator=g).to(BF16)
    out = paged_attention_cuda_sm100(q.to(cuda_device), cache, batch)
    want, bound = attend(q[0], new_k[0].double(), new_v[0].double(), torch.ones(150, heads, dtype=torch.float64),
                         sees(new, 150, 0, 0), dim**-0.5, BF16, False)
    assert bool(((out[0].cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("quantised", [False, True], ids=["same", "e4m3"])
def test_steps_of_a_server(cuda_device, quantised) -> None:
    """Prompts of different lengths in chunks, then single tokens, all written, attended and at the end read back."""
    g = torch.Generator().manual_seed(23)
    heads, kv_heads, dim, page, total = 8, 2, 64, 16, [75, 9, 130]
    steps = [[40, 9, 64], [35, 0, 65], [0, 0, 1]]
    total = [sum(s[b] for s in steps) for b in range(3)]
    cache = PagedKV.empty(40, kv_heads, page, dim, dtype=E4M3 if quantised else BF16, device=cuda_device)
    table = torch.randperm(40, generator=g)[:33].view(3, 11).to(torch.int32).to(cuda_device)
    k, v = ([torch.randn(n, kv_heads, dim, generator=g).to(BF16) for n in total] for _ in range(2))
    q = [torch.randn(n, heads, dim, generator=g).to(BF16) for n in total]
    if quantised:
        held = [[quantise(x) for x in t] for t in (k, v)]
        held = [[(x * s[..., None], s) for x, s in t] for t in held]
    else:
        held = [[(x.double(), torch.ones(x.shape[:2], dtype=torch.float64)) for x in t] for t in (k, v)]
    done = [0, 0, 0]
    for step in steps:
        rows = lambda t: torch.cat([t[b][done[b]:done[b] + n] for b, n in enumerate(step)]).to(cuda_device)  # noqa: E731,B023
        cu = torch.tensor([0, step[0], step[0] + step[1], sum(step)], dtype=torch.int32, device=cuda_device)
        lens = torch.tensor([d + n for d, n in zip(done, step)], dtype=torch.int32, device=cuda_device)
        batch = PagedBatch(table, lens, cu_seqlens=cu, max_q_len=max(step))
        kv_cache_write_cuda_sm100(rows(k), rows(v), cache, batch)
        out = paged_attention_cuda_sm100(rows(q), cache, batch).cpu()
        for b, n in enumerate(step):
            end = done[b] + n
            want, bound = attend(q[b][done[b]:end], held[0][b][0][:end], held[1][b][0][:end], held[1][b][1][:end],
                                 sees(n, end, 0, 0), dim**-0.5, BF16, quantised)
            assert bool(((out[cu[b]:cu[b + 1]].double() - want).abs() <= bound).all())
            done[b] = end
    got = kv_cache_read_cuda_sm100(cache, batch, 0, max(total), dtype=BF16)
    for out, t in zip(got, held):
        for b in range(3):
            assert torch.equal(out[b, :, :total[b]].transpose(0, 1).cpu().double(), t[b][0])
            assert bool((out[b, :, total[b]:] == 0).all())


def test_graph_replay_on_new_contents_and_streams(cuda_device) -> None:
    """Write and attention captured once and replayed as the sequences grow; two graphs on two streams at once."""
    g = torch.Generator(device=cuda_device).manual_seed(3)
    caches, batches, qs, ks, outs, graphs = [], [], [], [], [], []
    for i in range(2):
        cache = PagedKV.empty(24, 2, 16, 64, dtype=BF16, device=cuda_device)
        cache.k.normal_(generator=g)
        cache.v.normal_(generator=g)
        table = torch.randperm(24, generator=g, device=cuda_device).to(torch.int32).view(4, 6)
        lens = torch.tensor([5, 60, 33, 17], dtype=torch.int32, device=cuda_device)
        caches.append(cache)
        batches.append(PagedBatch(table, lens))
        qs.append(torch.randn(4, 1, 8, 64, generator=g, device=cuda_device).to(BF16))
        ks.append(torch.randn(4, 1, 2, 64, generator=g, device=cuda_device).to(BF16))
        kv_cache_write_cuda_sm100(ks[i], ks[i], cache, batches[i])
        paged_attention_cuda_sm100(qs[i], cache, batches[i])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lens.add_(1)
            kv_cache_write_cuda_sm100(ks[i], ks[i], cache, batches[i])
            outs.append(paged_attention_cuda_sm100(qs[i], cache, batches[i]))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for step in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                qs[i].normal_(generator=None)
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert batches[i].kv_lens.tolist() == [6 + step, 61 + step, 34 + step, 18 + step]
            assert torch.equal(outs[i], paged_attention_cuda_sm100(qs[i], caches[i], batches[i]))
            k, _ = kv_cache_read_cuda_sm100(caches[i], batches[i], 0, 96)
            for b, n in enumerate(batches[i].kv_lens.tolist()):
                assert torch.equal(k[b, :, n - 1], ks[i][b, 0])


def test_graph_of_chunks_replayed_on_new_lengths(cuda_device) -> None:
    """Chunks on the tensor cores, captured without a call before, replayed with other lengths and another split of
    the tokens among the sequences."""
    p = Problem(BF16, False, 8, 2, 128, 32, [(50, 300), (40, 90), (6, 500)], True, 29, cuda_device)
    q, cache, batch = p.q.to(cuda_device), p.kv(), p.batch()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = paged_attention_cuda_sm100(q, cache, batch)
    graph.replay()
    check_attention(p, out)
    other = [(10, 200), (80, 80), (6, 450)]
    batch.kv_lens.copy_(torch.tensor([kv for _, kv in other]))
    batch.cu_seqlens.copy_(torch.tensor([0, 10, 90, 96]))
    graph.replay()
    p.cu, p.lengths = torch.tensor([0, 10, 90, 96]), other
    for b, (_, kv) in enumerate(other):
        p.k[b], p.v[b], p.v_scale[b] = p.k[b][:kv], p.v[b][:kv], p.v_scale[b][:kv]
    check_attention(p, out)


def test_same_bits_twice_and_on_another_stream(cuda_device) -> None:
    p = Problem(BF16, True, 8, 2, 128, 16, [(1, 900), (30, 600), (1, 5)], True, 25, cuda_device)
    first = _run(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _run(p)
    side.synchronize()
    assert torch.equal(first, second)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_on_a_device_that_is_not_current(cuda_device) -> None:
    other = torch.device("cuda", 1)
    p = Problem(BF16, False, 4, 2, 64, 16, [(1, 90), (3, 40)], True, 26, other)
    check_attention(p, _run(p))


def test_half_steps() -> None:
    assert all(HALF_STEP[t] == torch.finfo(t).eps / 2 for t in HALF_STEP)


def test_expired_wait_is_reported_and_never_silent(cuda_device) -> None:
    """Attention on the tensor cores with a wait limit of 0 polls (measurement build): every wait gives up at once, the
    rows become NaN, the expiry is recorded, and calls are refused until it is taken."""
    from ako_b200 import _native

    with _native.measurement() as lib:
        try:
            p = Problem(BF16, False, 8, 2, 128, 16, [(70, 300), (90, 90), (1, 40)], True, 30, cuda_device)
            assert lib.ako_b200_measure_set_wait_polls(0) == 1 << 24
            out = _run(p)
            lib.ako_b200_measure_set_wait_polls(1 << 24)
            torch.cuda.synchronize()
            assert bool(out.isnan().all())
            with pytest.raises(RuntimeError, match="bounded wait"):
                _run(p)
            with pytest.raises(RuntimeError, match="bounded wait"):
                kv_cache_read_cuda_sm100(p.kv(), p.batch(), 0, 8)
            assert _native.take_device_status() == 1
            assert _native.take_device_status() == 0
            check_attention(p, _run(p))
        finally:
            lib.ako_b200_measure_set_wait_polls(1 << 24)
    assert _native.take_device_status() == 0
