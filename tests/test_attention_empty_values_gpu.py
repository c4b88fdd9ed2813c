"""Attention over an e4m3 cache some of whose value rows are all zero: such a row takes a share of the weights, however
large, and must cost the other keys' weights no bits, whatever its scale says.

The bound is made of what the definition has, weights p and values v, and not of the scales that a cache happens to
hold. With u the output type's half step it is, for an output o of a row,

    u |o| + (2^-11 + 2 e) sum p|v| + 2^-25 J sum |c| + 2^-25 (fp16 outputs, below which their steps are 2^-24)

where each weight is rounded to fp16 once (2^-11), and below 2^-14 of the largest contribution J to steps of 2^-24 of
it, times its value's element c = 448 v / max|v| at most: J is the largest p max|v| / 224, an element of each row that
is not zero being above 224. e is what 32 bits and the hardware's exponential and logarithm move a weight by: (dim + 4)
2^-24 of the score's sum |q k|, four roundings of the score and of the scale's logarithm, 2^-20 for the two functions,
and n 2^-23 for the sums over n keys.
"""

from __future__ import annotations

import math

import pytest
import torch
from paged_oracle import HALF_STEP, Problem, sees

from ako_b200 import kv_cache_write_cuda_sm100, paged_attention_cuda_sm100

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _pull(p: Problem, keys, bits: float, scale: float = 1.0, negative: bool = False) -> None:
    """Makes `keys` of every sequence take `bits` powers of two more than a score of zero from every row, and their
    values zero under the stored `scale`. Column 0 of the other keys is zero, that of q is one."""
    p.q[..., 0] = 1.0
    for b, (_, kv) in enumerate(p.lengths):
        p.k[b][..., 0] = 0.0
        for j in range(kv):
            at = int(p.table[b, j // p.page_size]), slice(None), j % p.page_size
            elements = p.caches["k"].view(torch.uint8)
            elements[at + (0,)] = 0
            if j not in keys:
                continue
            elements[at] = 0
            elements[at + (0,)] = 0x7E  # 448
            by = bits * math.log(2.0) * math.sqrt(p.dim) / 448
            p.caches["k_scale"][at] = by
            p.k[b][j] = 0.0
            p.k[b][j, :, 0] = 448 * float(torch.tensor(by))
            p.caches["v"].view(torch.uint8)[at] = 0x80 if negative else 0
            p.caches["v_scale"][at] = scale
            p.v[b][j] = 0.0


def _spread(p: Problem, f: float) -> None:
    """All values times f, a power of two, by their scales."""
    p.caches["v_scale"] *= f
    for b in range(len(p.lengths)):
        p.v[b] *= f


def _expect(p: Problem, b: int) -> tuple[torch.Tensor, torch.Tensor]:
    n, kv = p.lengths[b]
    ok = sees(n, kv, 0, 0)
    q = p.rows(p.q, b).double()
    out = torch.zeros_like(q)
    bound = torch.zeros_like(q)
    group, scale, u = p.q_heads // p.kv_heads, p.dim**-0.5, HALF_STEP[p.dtype]
    for h in range(p.q_heads):
        k, v = p.k[b][:, h // group], p.v[b][:, h // group]
        s = (q[:, h] @ k.T * scale).masked_fill(~ok, -math.inf)
        w = torch.softmax(s, -1)
        largest = v.abs().amax(-1)
        size = (q[:, h].abs() @ k.abs().T * scale).masked_fill(~ok, 0.0)
        logs = torch.log2(largest.clamp(min=1e-300) / 448).abs() * (largest > 0)
        e = ((p.dim + 4) * 2.0**-24 * size + 4 * 2.0**-24 * (s.masked_fill(~ok, 0.0).abs() + logs)).amax(-1, keepdim=True)
        e = e + 2.0**-20 + kv * 2.0**-23
        joint = (w * largest).amax(-1, keepdim=True) / 224
        elements = 448 * v.abs() / torch.where(largest > 0, largest, 1.0)[:, None]
        out[:, h] = w @ v
        bound[:, h] = (u * out[:, h].abs() + (2.0**-11 + 2 * e) * (w @ v.abs())
                       + 2.0**-25 * joint * (ok.double() @ elements) + (2.0**-25 if p.dtype == F16 else 0.0))
    return out, bound


def _check(p: Problem, got: torch.Tensor) -> None:
    got = got.cpu()
    for b in range(len(p.lengths)):
        want, bound = _expect(p, b)
        # the bound notices an answer that is lost: in most places the right one is far above it
        assert float((want.abs() > 4 * bound).double().mean()) > 0.5
        over = (p.rows(got, b).double() - want).abs() / bound
        assert float(over.max()) <= 1.0, f"sequence {b}: {float(over.max()):.2f} of the bound"


CASES = [(BF16, 10, 1.0), (BF16, 20, 2.0**-10), (BF16, 36, 2.0**-7), (BF16, 14, 2.0**-40), (F16, 6, 1.0), (F16, 10, 2.0**3)]


@pytest.mark.parametrize("dtype,bits,f", CASES)
@pytest.mark.parametrize("new", [1, 2, 7, 90], ids=["8rows", "8rows-2", "32rows", "many"])
@pytest.mark.parametrize("heads,dim", [((8, 2), 128), ((4, 1), 64)])
def test_a_first_key_without_values(cuda_device, dtype, bits, f, new, heads, dim) -> None:
    """The key that a model attends to when it attends to nothing, with the scale of 1 that a cache write gives it."""
    p = Problem(dtype, True, *heads, dim, 16, [(new, 400), (new, new + 1), (new, 1100)], True, 51, cuda_device)
    _spread(p, f)
    _pull(p, {0}, bits)
    _check(p, paged_attention_cuda_sm100(p.q.to(cuda_device), p.kv(), p.batch(new)))


@pytest.mark.parametrize("new", [1, 90], ids=["few", "many"])
@pytest.mark.parametrize("where", ["last", "fifths", "tile", "all-but-one"])
@pytest.mark.parametrize("scale", [1.0, 2.0**-20, 2.0**60, 0.37])
def test_keys_without_values_in_other_places(cuda_device, new, where, scale) -> None:
    """Under any scale, of either sign of zero; whole tiles of them, and all keys but one."""
    kv = 700
    keys = {"last": {kv - new}, "fifths": set(range(0, kv, 5)), "tile": set(range(120, 400)),
            "all-but-one": set(range(1, kv))}[where]
    p = Problem(BF16, True, 8, 2, 128, 16, [(new, kv)], True, 52, cuda_device)
    _spread(p, 2.0**-7)
    _pull(p, keys, 9.0, scale, negative=scale == 0.37)
    _check(p, paged_attention_cuda_sm100(p.q.to(cuda_device), p.kv(), p.batch(new)))


@pytest.mark.parametrize("new", [1, 90], ids=["few", "many"])
def test_nothing_but_keys_without_values_is_zero(cuda_device, new) -> None:
    p = Problem(BF16, True, 8, 2, 128, 16, [(new, 300)], True, 53, cuda_device)
    _pull(p, set(range(300)), 12.0)
    assert bool((paged_attention_cuda_sm100(p.q.to(cuda_device), p.kv(), p.batch(new)) == 0).all())


@pytest.mark.parametrize("new", [1, 90], ids=["few", "many"])
def test_a_written_row_of_zeros(cuda_device, new) -> None:
    """The same through the write: the first token's values are zeros, the others' about 1e-3."""
    kv = 500
    p = Problem(BF16, True, 8, 2, 128, 16, [(kv, kv)], True, 54, cuda_device)
    v_new = (p.v_new * 1e-3).to(BF16)
    k_new = p.k_new / 3
    v_new[0] = 0
    k_new[..., 0] = 0
    k_new[0] = 0
    k_new[0, :, 0] = 14 * math.log(2.0) * math.sqrt(p.dim)
    kv_cache_write_cuda_sm100(k_new.to(cuda_device), v_new.to(cuda_device), p.kv(), p.batch())
    for name, into in (("k", p.k), ("v", p.v)):
        for j in range(kv):
            at = int(p.table[0, j // 16]), slice(None), j % 16
            into[0][j] = p.caches[name][at].double().cpu() * p.caches[name + "_scale"][at].double().cpu()[:, None]
    p.q[..., 0] = 1.0
    p.q = p.q[kv - new:]
    p.lengths = [(new, kv)]
    p.cu = torch.tensor([0, new], dtype=torch.int32)
    _check(p, paged_attention_cuda_sm100(p.q.to(cuda_device), p.kv(), p.batch(new)))
