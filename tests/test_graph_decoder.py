"""Graph decoding up to a cache's last position, and what it refuses beyond it."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
from test_paged_decoder import SMALL, _model, _tables

from ako_b200.decoder import GraphDecoder, KVCache, ModelConfig, build_decoder
from ako_b200.paged import E4M3


@pytest.mark.parametrize("length,max_len,steps,words", [
    (20, 32, 13, "KV cache holds 32 positions, asked for 33"), (32, 32, 1, "KV cache holds 32"),
    (0, 8, 9, "KV cache holds 8"), (150, 200, 11, "the model has 160 positions, asked for 161"),
    (20, 32, 0, "steps must be >= 1"), (20, 32, -1, "steps must be >= 1")])
def test_graph_decoder_refuses_steps_that_do_not_fit(length, max_len, steps, words) -> None:
    model = SimpleNamespace(cfg=ModelConfig(**SMALL))
    first = torch.zeros(2, 1, dtype=torch.int64)
    paged = SimpleNamespace(length=length, max_len=max_len)  # what a paged cache says of itself; its own needs a GPU
    dense = KVCache(model.cfg, 2, max_len, device="cpu", dtype=torch.bfloat16)
    dense.length = length
    for cache in (paged, dense):
        with pytest.raises(ValueError, match=words):
            GraphDecoder(model, cache, first, steps)
    if steps > 1:
        GraphDecoder(model, SimpleNamespace(length=length, max_len=length + 1), first, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["dense", "paged", "paged-e4m3"])
@pytest.mark.parametrize("start,steps", [(26, 6), (31, 1), (154, 6)])
def test_graph_decoding_up_to_the_last_position(cuda_device, kind, start, steps) -> None:
    """The cache's end is that of a page, at (154, 6) that of the model's positions too. Tokens are the eager path's,
    and what was cached before is left as it was, by the warm-up before the capture too."""
    if kind == "dense":  # eager and graph steps call different attentions of torch there: equal tokens need 32 bits
        m = build_decoder(ModelConfig(**SMALL), device=cuda_device, dtype=torch.float32, seed=5)
        _tables(m, cuda_device)
    else:
        m = _model(cuda_device)
    ids = torch.randint(0, 97, (3, start), generator=torch.Generator().manual_seed(7)).to(cuda_device)
    with torch.inference_mode():
        if kind == "dense":
            cache = m.new_cache(3, start + steps)
        else:
            cache = m.new_paged_cache(3, start + steps, page_size=8, kv_dtype=E4M3 if kind == "paged-e4m3" else None)
        m.hidden(ids, cache)

        def held() -> list[torch.Tensor]:
            """The prompt's keys and values, as they are stored."""
            out = []
            for layer in range(2):
                if kind == "dense":
                    out += [t[layer][:, :, :start] for t in (cache.k, cache.v)]
                    continue
                pages = (start + steps) // 8
                for t in (cache.layers[layer].k, cache.layers[layer].v):
                    t = t.view(torch.uint8).unflatten(0, (3, pages)).transpose(2, 3).flatten(1, 2)
                    out.append(t[:, :start])
            return [t.clone() for t in out]

        before = held()
        tok, eager = ids[:, -1:].clone(), []
        for _ in range(steps):
            tok = m(tok, cache).argmax(-1, keepdim=True)
            eager.append(tok)
        with pytest.raises(ValueError, match="KV cache holds"):
            m(tok, cache)
        cache.length = start
        gd = GraphDecoder(m, cache, ids[:, -1:], steps)
        assert torch.equal(gd.run(ids[:, -1:]), torch.cat(eager, 1))
        assert torch.equal(gd.run(ids[:, -1:]), torch.cat(eager, 1))
        assert all(torch.equal(a, b) for a, b in zip(held(), before))
        with pytest.raises(ValueError, match="KV cache holds"):
            GraphDecoder(m, cache, ids[:, -1:], steps + 1)
