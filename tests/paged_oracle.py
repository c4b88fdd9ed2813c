"""Paged-cache operators in 64 bits, and the bounds their kernels are held to."""

from __future__ import annotations

import math
import random
from dataclasses import dataclass, field

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn
#: Half a step of each type, relative to the value: what one rounding may be off by.
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Elements (as float64) and scales of rows ``x`` (..., head_dim) by the definition: the least power of two s,
    at least 2^-126, with max|x| / s <= 448 over finite values, and x / s on e4m3's grid (4 significant bits, least
    step 2^-9), ties to even, infinities at 448."""
    x = x.double().numpy()
    top = np.where(np.isfinite(x), np.abs(x), 0.0).max(-1)
    s = np.exp2(np.clip(np.ceil(np.log2(np.where(top > 0, top, 448.0) / 448.0)), -126, None))
    s = np.where(top / s > 448.0, 2 * s, s)  # log2's own rounding
    s = np.where((top > 0) & (top / (s / 2) <= 448.0) & (s > 2.0**-126), s / 2, s)
    y = x / s[..., None]
    with np.errstate(invalid="ignore"):
        mag = np.where(np.isfinite(y) & (y != 0), np.abs(y), 1.0)
        step = np.exp2(np.maximum(np.floor(np.log2(mag)), -6) - 3)
        y = np.clip(np.where(np.isfinite(y), np.rint(y / step) * step, y), -448.0, 448.0)
    return torch.from_numpy(y), torch.from_numpy(s)


@dataclass
class Problem:
    """Sequences with their keys and values in a paged cache whose unused places hold NaN."""

    dtype: torch.dtype
    quantised: bool
    q_heads: int
    kv_heads: int
    dim: int
    page_size: int
    lengths: list[tuple[int, int]]  # (new, cached with the new ones)
    packed: bool
    seed: int = 0
    device: torch.device | str = "cpu"
    slots_first: bool = False  # the cache laid out (pages, page_size, heads, dim)
    spare_pages: int = 2
    table_width: int | None = None
    spread: float = 1.0
    k: list[torch.Tensor] = field(default_factory=list)  # per sequence (kv, heads, dim), float64
    v: list[torch.Tensor] = field(default_factory=list)
    v_scale: list[torch.Tensor] = field(default_factory=list)  # (kv, heads)

    def __post_init__(self) -> None:
        g = torch.Generator().manual_seed(self.seed)
        rnd = random.Random(self.seed)
        pages = [-(-kv // self.page_size) for _, kv in self.lengths]
        width = max([1, *pages]) if self.table_width is None else self.table_width
        self.num_pages = sum(pages) + self.spare_pages
        free = list(range(self.num_pages))
        rnd.shuffle(free)
        table = torch.full((len(pages), width), -1, dtype=torch.int32)
        for b, n in enumerate(pages):
            for i in range(n):
                table[b, i] = free.pop()
        self.table = table
        self.kv_lens = torch.tensor([kv for _, kv in self.lengths], dtype=torch.int32)
        self.cu = torch.tensor([0, *np.cumsum([q for q, _ in self.lengths])], dtype=torch.int32)
        shape = (self.num_pages, self.kv_heads, self.page_size, self.dim)
        held = E4M3 if self.quantised else self.dtype
        self.caches = {}
        for name in ("k", "v"):
            x = torch.full(shape, math.nan)
            scale = torch.full(shape[:3], math.nan)
            for b, (_, kv) in enumerate(self.lengths):
                rows = (torch.randn(kv, self.kv_heads, self.dim, generator=g) * self.spread).to(self.dtype)
                if self.quantised:
                    rows, s = quantise(rows)
                else:
                    rows, s = rows.double(), torch.ones(kv, self.kv_heads, dtype=torch.float64)
                getattr(self, name).append(rows * s[..., None])
                if name == "v":
                    self.v_scale.append(s)
                for j in range(kv):
                    p, o = int(table[b, j // self.page_size]), j % self.page_size
                    x[p, :, o], scale[p, :, o] = rows[j].float(), s[j].float()
            x = x.to(held)
            if self.slots_first:
                x = x.transpose(1, 2).contiguous().transpose(1, 2)
            self.caches[name] = x.to(self.device) if not self.slots_first else (
                x.transpose(1, 2).to(self.device).transpose(1, 2))
            self.caches[name + "_scale"] = scale.to(self.device) if self.quantised else None
        new = sum(q for q, _ in self.lengths)
        if self.packed:
            lead = (new,)
        else:
            lead = (len(self.lengths), self.lengths[0][0] if self.lengths else 1)
        self.q = torch.randn(*lead, self.q_heads, self.dim, generator=g).to(self.dtype)
        self.k_new = (torch.randn(*lead, self.kv_heads, self.dim, generator=g) * 3).to(self.dtype)
        self.v_new = torch.randn(*lead, self.kv_heads, self.dim, generator=g).to(self.dtype)

    def kv(self):
        from ako_b200 import PagedKV

        return PagedKV(self.caches["k"], self.caches["v"], self.caches["k_scale"], self.caches["v_scale"])

    def batch(self, max_q_len: int | None = None):
        from ako_b200 import PagedBatch

        d = self.device
        if not self.packed:
            return PagedBatch(self.table.to(d), self.kv_lens.to(d))
        return PagedBatch(self.table.to(d), self.kv_lens.to(d), cu_seqlens=self.cu.to(d), max_q_len=max_q_len)

    def rows(self, t: torch.Tensor, b: int) -> torch.Tensor:
        """Sequence b's new tokens of a tensor of them."""
        return t[self.cu[b]:self.cu[b + 1]] if self.packed else t[b]


def sees(q: int, kv: int, window: int, sinks: int) -> torch.Tensor:
    """(q, kv) truth values: which keys each new token sees."""
    p = torch.arange(kv - q, kv)[:, None]
    j = torch.arange(kv)[None]
    ok = j <= p
    if window:
        ok &= (j > p - window) | (j < sinks)
    return ok


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, v_scale: torch.Tensor, ok: torch.Tensor,
           scale: float, dtype: torch.dtype, quantised: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """One sequence's outputs (q, q_heads, dim) in 64 bits, and how far a kernel may be from each.

    With u the half step of the 16-bit types: the output is rounded once (u |o|). Each weight is rounded once to
    the second product's type: bf16 and fp16 as the activations, or for an e4m3 cache fp16 or bf16, whose larger
    half step counts here, u_w sum p|v|; in fp16 weights below 2^-14 of the largest are off by up to 2^-25 of it,
    times their values' elements. A score is a sum of dim products in fp32, in any order, and scaled in three more
    roundings: off by at most (dim + 4) 2^-24 scale sum|q k| + 4 2^-24 |s|; with the hardware's exponential and
    logarithm (2^-20 together for arguments up to 2^7) that moves each weight, and with them sum p|v| and the sum of
    weights, by that much relatively; fp32 sums over n keys add n 2^-24 twice.
    """
    heads, groups = q.shape[1], q.shape[1] // k.shape[1]
    q = q.double()
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros_like(out)
    u = HALF_STEP[dtype]
    u_w = max(u, HALF_STEP[torch.float16]) if quantised else u
    for h in range(heads):
        kk, vv, vs = k[:, h // groups], v[:, h // groups], v_scale[:, h // groups]
        s = (q[:, h] @ kk.T * scale).masked_fill(~ok, -math.inf)
        size = q[:, h].abs() @ kk.abs().T * abs(scale)
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
        w = torch.where(ok, w, 0.0)
        total = w.sum(-1, keepdim=True)
        p = w / torch.where(total > 0, total, 1.0)
        seen_v = torch.where(torch.isfinite(vv), vv, 0.0)
        o = p @ seen_v
        # infinities and NaN, through the keys that a row sees
        for bad in (vv == math.inf, vv == -math.inf, vv.isnan()):
            hit = ok.double() @ bad.double() > 0
            o = torch.where(hit, o + (math.inf if bad is not None and vv[bad].numel() and (vv[bad] == math.inf).all()
                                      else -math.inf if vv[bad].numel() and (vv[bad] == -math.inf).all() else math.nan), o)
        n = kk.shape[0]
        e = torch.where(ok, (kk.shape[1] + 4) * 2.0**-24 * size + 4 * 2.0**-24 * s.abs().masked_fill(~ok, 0), 0.0)
        e = (e.amax(-1, keepdim=True) if n else torch.zeros(len(q), 1)) + 2.0**-20 + n * 2.0**-23
        mass = p @ seen_v.abs()
        elements = seen_v.abs() / torch.where(vs > 0, vs, 1.0)[:, None]
        joint = (p * vs[None]).amax(-1, keepdim=True) if n else torch.zeros(len(q), 1)
        small = 2.0**-25 * joint * (ok.double() @ elements)
        out[:, h] = o
        bound[:, h] = u * o.abs() + (u_w + 2 * e) * mass + small + 2.0**-25 * o.abs() + 2.0**-26
    return out, bound


def check_attention(p: Problem, got: torch.Tensor, *, scale: float | None = None, window: int = 0,
                    sinks: int = 0) -> None:
    got = got.cpu()
    scale = p.dim**-0.5 if scale is None else scale
    for b, (n, kv) in enumerate(p.lengths):
        want, bound = attend(p.rows(p.q, b), p.k[b], p.v[b], p.v_scale[b], sees(n, kv, window, sinks), scale, p.dtype,
                             p.quantised)
        have = p.rows(got, b).double()
        fine = torch.isfinite(want)
        same = (have[~fine] == want[~fine]) | (have[~fine].isnan() & want[~fine].isnan())
        assert bool(same.all()), f"sequence {b}: infinities and NaN differ"
        over = ((have - want).abs() / bound)[fine]
        assert not over.numel() or float(over.max()) <= 1.0, (
            f"sequence {b} of {p.lengths}: error {float(over.max()):.3f} of its bound at "
            f"{np.unravel_index(int(((have - want).abs() / bound).nan_to_num(0).argmax()), have.shape)}")
