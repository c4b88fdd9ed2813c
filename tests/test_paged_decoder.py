"""The decoder on a paged cache. The RoPE tables are set here, so that nothing needs the reference package."""

from __future__ import annotations

import math

import pytest
import torch

from ako_b200.decoder import GraphDecoder, ModelConfig, PagedKVCache, build_decoder
from ako_b200.paged import E4M3

SMALL = dict(hidden_dim=256, n_layers=2, n_heads=8, n_kv_heads=2, intermediate_dim=512, max_seq_len=160, vocab_size=97)


def _tables(m, device) -> None:
    cfg = m.cfg
    f = cfg.rope_base ** (-torch.arange(0, cfg.head_dim, 2, dtype=torch.float64) / cfg.head_dim)
    a = torch.arange(cfg.max_seq_len, dtype=torch.float64)[:, None] * f
    m._tables = (a.cos().float().to(device), a.sin().float().to(device))


def _model(device, **kw):
    m = build_decoder(ModelConfig(**SMALL), device=device, dtype=torch.bfloat16, seed=3, **kw)
    _tables(m, device)
    return m


def test_paged_cache_refusals() -> None:
    m = build_decoder(ModelConfig(**SMALL), backend="torch", device="cpu", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="backend='b200'"):
        m.new_paged_cache(2)
    with pytest.raises(ValueError, match="float16/bfloat16"):
        PagedKVCache(ModelConfig(**SMALL), 1, 16, device="cpu", dtype=torch.float32)


def _plain_hidden(m, ids, window=0, sinks=0):
    """Final hidden states of the same weights in fp64, with dense masked attention."""
    cfg = m.cfg
    w = {n: p.double() for n, p in m.named_parameters()}
    cos, sin = (t.double()[: ids.shape[1], None] for t in m._tables)

    def norm(x, g):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + cfg.eps) * g

    def rope(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    n = ids.shape[1]
    p, j = torch.arange(n, device=ids.device)[:, None], torch.arange(n, device=ids.device)[None]
    hide = j > p
    if window:
        hide |= (j + window <= p) & (j >= sinks)
    x = w["embed.weight"][ids]
    for i in range(cfg.n_layers):
        g = lambda name: w[f"layers.{i}.{name}"]  # noqa: E731,B023
        h = norm(x, g("input_norm_weight")) @ g("qkv_proj.weight").T
        q, k, v = h.split([cfg.n_heads * cfg.head_dim] + [cfg.n_kv_heads * cfg.head_dim] * 2, -1)
        q, k, v = (t.view(*ids.shape, -1, cfg.head_dim) for t in (q, k, v))
        q, k = rope(q), rope(k)
        k, v = (t.repeat_interleave(cfg.n_heads // cfg.n_kv_heads, 2) for t in (k, v))
        s = torch.einsum("bphd,bjhd->bhpj", q, k) / math.sqrt(cfg.head_dim)
        a = torch.softmax(s.masked_fill(hide, -math.inf), -1)
        x = x + torch.einsum("bhpj,bjhd->bphd", a, v).flatten(2) @ g("o_proj.weight").T
        gate, up = (norm(x, g("post_attention_norm_weight")) @ g("gate_up_proj.weight").T).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ g("down_proj.weight").T
    return norm(x, w["final_norm_weight"])


@pytest.mark.gpu
@pytest.mark.parametrize("kv_dtype,window,sinks", [(None, 0, 0), (None, 20, 3), (E4M3, 0, 0)])
def test_chunks_and_steps_against_fp64(cuda_device, kv_dtype, window, sinks) -> None:
    """Chunks of 40, 1, 37 and 2 tokens. Hidden states have unit mean square; bf16 rounds each of about ten
    intermediate results per layer by at most 2^-8, e4m3 keys and values by at most 2^-4, both mostly averaged out:
    the mean square error stays below (2 layers x 10 x 2^-8)^2, the bound if they all added up, and for e4m3 below
    its 2^-4 squared on top."""
    m = _model(cuda_device)
    ids = torch.randint(0, 97, (3, 80), generator=torch.Generator().manual_seed(1)).to(cuda_device)
    with torch.inference_mode():
        cache = m.new_paged_cache(3, 100, page_size=16, kv_dtype=kv_dtype, window=window, sinks=sinks)
        at, out = 0, []
        for n in (40, 1, 37, 2):
            out.append(m.hidden(ids[:, at:at + n], cache))
            at += n
        assert cache.length == 80
        want = _plain_hidden(m, ids, window, sinks)
    err = float((torch.cat(out, 1).double() - want).square().mean().sqrt())
    bound = 2 * 10 * 2.0**-8
    assert err <= (bound if kv_dtype is None else math.hypot(bound, 2.0**-4)), err
    with pytest.raises(ValueError, match="KV cache holds 100"):
        m.hidden(ids[:, :21], cache)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_dtype", [None, E4M3])
def test_graph_decoding_on_pages_equals_eager(cuda_device, kv_dtype) -> None:
    m = _model(cuda_device)
    ids = torch.randint(0, 97, (3, 20), generator=torch.Generator().manual_seed(2)).to(cuda_device)
    with torch.inference_mode():
        cache = m.new_paged_cache(3, 32, page_size=8, kv_dtype=kv_dtype)
        m.hidden(ids, cache)
        tok, eager = ids[:, -1:].clone(), []
        for _ in range(6):
            tok = m(tok, cache).argmax(-1, keepdim=True)
            eager.append(tok)
        cache.length = 20
        gd = GraphDecoder(m, cache, ids[:, -1:], 6)
        assert torch.equal(gd.run(ids[:, -1:]), torch.cat(eager, 1))
        assert torch.equal(gd.run(ids[:, -1:]), torch.cat(eager, 1))
