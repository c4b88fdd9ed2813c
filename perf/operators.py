"""Cases of the paged-cache operators: writing new keys and values into a paged cache, reading them back, and attention
of new tokens over it.

A case says which operator runs (``op``), the element type of the activations (``dtype``), how the cache holds its
values (``cache``: ``same`` as the activations, or ``e4m3`` with one power-of-two scale per token and head), the head
layout and the page size, and how many sequences there are, with how many new (``q_min .. q_max``) and cached
(``kv_min .. kv_max``, new ones included) tokens. ``mix`` seeds the lengths, so that a case is always the same work;
the values and the order of the pages come from the seed that ``prepare`` is given.
"""

import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


def _case(name, op, dtype, cache, heads, dim, page, batch, q, kv, window=0, sinks=0, mix=1):
    return {"name": name, "op": op, "dtype": dtype, "cache": cache, "q_heads": heads[0], "kv_heads": heads[1],
            "head_dim": dim, "page_size": page, "batch": batch, "q_min": q[0], "q_max": q[1], "kv_min": kv[0],
            "kv_max": kv[1], "window": window, "sinks": sinks, "mix": mix}


def listed():
    return [
        # one decoding step of 32 sequences writes its new token's keys and values: the smallest write
        _case("write_step_e4m3", "write", "bfloat16", "e4m3", (32, 8), 128, 16, 32, (1, 1), (1, 2048)),
        # ragged prompts written as they are
        _case("write_prompts_bf16", "write", "bfloat16", "same", (32, 8), 128, 64, 8, (777, 2048), (777, 2100)),
        # ragged prompts of a model without shared heads, quantised as they are written
        _case("write_prompts_f16_e4m3", "write", "float16", "e4m3", (32, 32), 64, 32, 6, (901, 4099), (901, 4099)),
        # four short sequences read back, to be handed to code that wants a dense cache
        _case("read_short_e4m3", "read", "bfloat16", "e4m3", (32, 8), 128, 16, 4, (1, 1), (130, 517)),
        # eight long sequences read back
        _case("read_long_e4m3", "read", "bfloat16", "e4m3", (32, 8), 128, 64, 8, (1, 1), (8000, 16384)),
        # one sequence's decoding step on a short context: latency
        _case("decode_one", "attend", "bfloat16", "same", (32, 8), 128, 16, 1, (1, 1), (777, 777)),
        # the decoder's decoding step: 32 sequences, contexts of about 2048 tokens
        _case("decode_batch", "attend", "bfloat16", "same", (32, 8), 128, 64, 32, (1, 1), (1500, 2176)),
        # long contexts of very different lengths in a quantised cache
        _case("decode_long_e4m3", "attend", "bfloat16", "e4m3", (32, 8), 128, 64, 16, (1, 1), (2000, 65536)),
        # a decoding step under a sliding window with four first tokens that stay visible
        _case("decode_window_f16", "attend", "float16", "same", (16, 4), 64, 32, 64, (1, 1), (3, 16384), 1024, 4),
        # one step of a server that mixes decoding sequences with chunks of prompts, on a quantised cache
        _case("mixed_chunks_e4m3", "attend", "bfloat16", "e4m3", (32, 8), 128, 16, 12, (1, 317), (1, 4000), 0, 0, 3),
        # a chunk of 2048 new tokens on a context of 16384
        _case("chunk_long", "attend", "bfloat16", "same", (32, 8), 128, 64, 1, (2048, 2048), (18432, 18432)),
        # the decoder's prompts, into an empty cache
        _case("prompt_batch", "attend", "bfloat16", "same", (32, 8), 128, 64, 8, (2048, 2048), (2048, 2048)),
    ]


def _lengths(case):
    """New and cached tokens of each sequence: the first has the most of both, the others' lengths are spread evenly
    over their logarithm where the range spans more than a factor of ten, and over the range otherwise."""
    r = random.Random(case["mix"])

    def pick(lo, hi):
        if hi <= 10 * lo:
            return r.randint(lo, hi)
        return min(hi, int(math.exp(r.uniform(math.log(lo), math.log(hi + 1)))))

    got = [(case["q_max"], max(case["q_max"], case["kv_max"]))]
    for _ in range(case["batch"] - 1):
        q = pick(case["q_min"], case["q_max"])
        got.append((q, max(q, pick(case["kv_min"], case["kv_max"]))))
    return got


def _seen(q, kv, window, sinks):
    """Pairs of a new token and a key that it sees, and keys that any of the new tokens sees."""
    p = np.arange(kv - q, kv, dtype=np.int64)
    if not window:
        return int((p + 1).sum()), kv
    near = np.minimum(p + 1, window)
    first = np.minimum(sinks, p + 1 - near)
    start = max(0, kv - q + 1 - window)
    return int((near + first).sum()), kv - start + min(sinks, start)


def work(case):
    bytes_in = 2
    held = 1 if case["cache"] == "e4m3" else bytes_in
    scale = 8 if case["cache"] == "e4m3" else 0  # a key's and a value's scale
    d, hq, hk = case["head_dim"], case["q_heads"], case["kv_heads"]
    lengths = _lengths(case)
    new = sum(q for q, _ in lengths)
    if case["op"] == "write":
        return {"bytes": new * hk * (2 * d * (bytes_in + held) + scale), "flops": 0}
    if case["op"] == "read":
        rows = sum(kv for _, kv in lengths)
        dense = case["batch"] * max(kv for _, kv in lengths)
        return {"bytes": hk * (rows * (2 * d * held + scale) + dense * 2 * d * bytes_in), "flops": 0}
    seen = [_seen(q, kv, case["window"], case["sinks"]) for q, kv in lengths]
    return {"bytes": 2 * new * hq * d * bytes_in + sum(k for _, k in seen) * hk * (2 * d * held + scale),
            "flops": 4 * d * hq * sum(pairs for pairs, _ in seen)}


def _dense(case):
    """Values of the padded arrays that the plain form makes."""
    q, kv = case["q_max"], max(case["q_max"], case["kv_max"])
    rows = case["batch"] * kv * case["kv_heads"] * case["head_dim"]
    return max(rows, case["batch"] * case["q_heads"] * q * kv if case["op"] == "attend" else 0)


def draw(rng):
    def log(lo, hi):
        return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))

    op = rng.choice(["write", "read", "attend", "attend", "attend"])
    most = [work(c) for c in listed() if c["op"] == op]
    most = {k: max(w[k] for w in most) for k in ("bytes", "flops")}
    while True:
        kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
        q_heads = kv_heads * rng.choice([1, 2, 4, 5, 8, 16])
        dim = rng.choice([32, 64, 80, 96, 128, 128])
        page = rng.choice([8, 16, 16, 32, 64, 128])
        batch = log(1, 64)
        most_kv = 65536 if op != "write" else 8192
        kv = (log(1, most_kv), log(1, most_kv))
        q = (1, 1)
        if op == "write" or (op == "attend" and rng.random() < 0.6):
            q = (log(1, 4096), log(1, 4096))
        q, kv = (min(q), max(q)), (min(kv), max(kv))
        window = sinks = 0
        if op == "attend" and rng.random() < 0.35:
            window, sinks = log(16, 4096), rng.choice([0, 1, 4, 64])
        case = _case("", op, rng.choice(["bfloat16", "bfloat16", "float16"]), rng.choice(["same", "e4m3"]),
                     (q_heads, kv_heads), dim, page, batch, q, kv, window, sinks, rng.randrange(1 << 30))
        del case["name"]
        if q_heads > 64 or _dense(case) > 1_250_000_000:
            continue
        w = work(case)
        if all(w[k] <= most[k] for k in most):
            return case


def _quantise(x):
    """Values and scales of `x` (..., head_dim) in 8 bits, each row under a power of two that keeps it within 448."""
    x = x.float()
    top = x.abs().amax(-1)
    part, power = torch.frexp(top)  # top = part * 2^power, 1/2 <= part < 1, and 448 = 7/8 * 2^9
    power = power - 9 + (part > 0.875).to(power.dtype)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), power), torch.ones_like(top))
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, dt = "cuda", _TYPES[case["dtype"]]
    hq, hk, d, ps = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    lengths = _lengths(case)
    batch = len(lengths)
    q_len = torch.tensor([q for q, _ in lengths], dtype=torch.int32, device=dev)
    kv_lens = torch.tensor([kv for _, kv in lengths], dtype=torch.int32, device=dev)
    pages = [-(-kv // ps) for _, kv in lengths]
    total = sum(pages)
    # pages in any order, as a server hands them out; entries behind a sequence's pages are not valid
    order = torch.randperm(total + 3, generator=g, device=dev)[:total].to(torch.int32)
    width = max(pages)
    starts = torch.tensor([0] + pages, device=dev).cumsum(0)
    at = starts[:-1, None] + torch.arange(width, device=dev)
    table = torch.where(torch.arange(width, device=dev) < torch.tensor(pages, device=dev)[:, None],
                        order[at.clamp(max=total - 1)], -1).to(torch.int32).contiguous()
    new = int(sum(q for q, _ in lengths))
    uniform = case["q_min"] == case["q_max"]
    cu = torch.zeros(batch + 1, dtype=torch.int32, device=dev)
    cu[1:] = q_len.cumsum(0)
    shape = (batch, case["q_max"]) if uniform else (new,)
    # some channels of keys are several times the others, as in trained models
    gain = torch.exp(0.6 * torch.randn(hk, 1, d, generator=g, device=dev))

    def tensor(heads, spread):
        return (torch.randn(*shape, heads, d, generator=g, device=dev) * spread).to(dt)

    s = {"case": case, "uniform": uniform, "cu": cu, "q_len": q_len, "kv_lens": kv_lens, "table": table,
         "longest": max(kv for _, kv in lengths), "k_scale": None, "v_scale": None}
    cache = (total + 3, hk, ps, d)
    if case["op"] == "write":
        held = torch.float8_e4m3fn if case["cache"] == "e4m3" else dt
        s["k"], s["v"] = tensor(hk, gain.reshape(hk, d)), tensor(hk, 1.0)
        s["k_cache"], s["v_cache"] = (torch.zeros(cache, device=dev, dtype=held) for _ in range(2))
        if case["cache"] == "e4m3":
            s["k_scale"], s["v_scale"] = (torch.ones(cache[:3], device=dev) for _ in range(2))
    else:
        for name, spread in (("k", gain), ("v", 1.0)):
            x = torch.empty(cache, device=dev, dtype=dt).normal_(generator=g) * spread
            if case["cache"] == "e4m3":
                s[name + "_cache"], s[name + "_scale"] = _quantise(x)
            else:
                s[name + "_cache"] = x.to(dt)
            del x
        s["q"] = tensor(hq, 1.0) if case["op"] == "attend" else None
    if own:
        import ako_b200

        s["cache"] = ako_b200.PagedKV(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        if uniform:
            s["batch"] = ako_b200.PagedBatch(table, kv_lens)
        else:
            s["batch"] = ako_b200.PagedBatch(table, kv_lens, cu_seqlens=cu, max_q_len=case["q_max"])
    return s


def _own_run(s):
    import ako_b200

    c = s["case"]
    if c["op"] == "write":
        ako_b200.kv_cache_write_cuda_sm100(s["k"], s["v"], s["cache"], s["batch"])
        return _written(s)
    if c["op"] == "read":
        return ako_b200.kv_cache_read_cuda_sm100(s["cache"], s["batch"], 0, s["longest"], dtype=_TYPES[c["dtype"]])
    return ako_b200.paged_attention_cuda_sm100(s["q"], s["cache"], s["batch"], window=c["window"], sinks=c["sinks"])


def _written(s):
    return [x for x in (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]) if x is not None]


def _places(s):
    """Sequence, and position in it, of each new token."""
    n = int(s["case"]["batch"])
    if s["uniform"]:
        m = s["case"]["q_max"]
        b = torch.arange(n * m, device="cuda") // m
        i = torch.arange(n * m, device="cuda") % m
    else:
        t = torch.arange(s["k" if "k" in s else "q"].shape[0], device="cuda")
        b = torch.searchsorted(s["cu"].long(), t, right=True) - 1
        i = t - s["cu"][b]
    return b, (s["kv_lens"] - s["q_len"])[b] + i


def _store(s, x, cache, scale):
    b, p = _places(s)
    c = s["case"]
    page, off = s["table"][b, p // c["page_size"]].long(), p % c["page_size"]
    x = x.reshape(-1, c["kv_heads"], c["head_dim"])
    if scale is None:
        cache[page, :, off] = x
    else:
        x, by = _quantise(x)
        cache.view(torch.uint8)[page, :, off] = x.view(torch.uint8)
        scale[page, :, off] = by


def _gathered(s, cache, scale):
    """(batch, kv_heads, longest, head_dim) of the cached values, in 32 bits; anything behind a sequence's end."""
    c = s["case"]
    j = torch.arange(s["longest"], device="cuda")
    page, off = s["table"].long().clamp(min=0)[:, j // c["page_size"]], j % c["page_size"]
    x = cache.view(torch.uint8)[page, :, off].view(cache.dtype) if scale is not None else cache[page, :, off]
    x = x.float()
    if scale is not None:
        x = x * scale[page, :, off][..., None]
    return x.transpose(1, 2)


def run(s):
    if own:
        return _own_run(s)
    c = s["case"]
    dt = _TYPES[c["dtype"]]
    if c["op"] == "write":
        _store(s, s["k"], s["k_cache"], s["k_scale"])
        _store(s, s["v"], s["v_cache"], s["v_scale"])
        return _written(s)
    inside = torch.arange(s["longest"], device="cuda") < s["kv_lens"][:, None]
    k, v = _gathered(s, s["k_cache"], s["k_scale"]), _gathered(s, s["v_cache"], s["v_scale"])
    if c["op"] == "read":
        inside = inside[:, None, :, None]
        return torch.where(inside, k, 0.0).to(dt), torch.where(inside, v, 0.0).to(dt)
    n, hk, g, m, d = c["batch"], c["kv_heads"], c["q_heads"] // c["kv_heads"], c["q_max"], c["head_dim"]
    q = s["q"]
    b, p = _places(s)
    i = p - (s["kv_lens"] - s["q_len"])[b]
    if not s["uniform"]:
        padded = torch.zeros(n, m, hk * g, d, device="cuda", dtype=dt)
        padded[b, i] = q
        q = padded
    q = q.float().reshape(n, m, hk, g, d).permute(0, 2, 3, 1, 4).reshape(n, hk, g * m, d)
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).view(n, hk, g, m, -1)
    pos = (s["kv_lens"] - s["q_len"])[:, None] + torch.arange(m, device="cuda")  # (n, m)
    j = torch.arange(s["longest"], device="cuda")
    sees = (j <= pos[..., None]) & inside[:, None]
    if c["window"]:
        sees &= (j > pos[..., None] - c["window"]) | (j < c["sinks"])
    scores.masked_fill_(~sees[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(n, hk, g * m, -1), torch.where(inside[:, None, :, None], v, 0.0))
    out = out.view(n, hk, g, m, d) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, m, hk * g, d)
    return (out if s["uniform"] else out[b, i]).to(dt)


def exact(case, seed):
    s = prepare(case, seed)
    c, ps, hk, d = case, case["page_size"], case["kv_heads"], case["head_dim"]
    lengths = _lengths(case)
    table = s["table"].cpu().numpy()
    if c["op"] == "write":
        got = []
        for x in (s["k"], s["v"]):
            x = x.double().cpu().numpy().reshape(-1, hk, d)
            held = np.zeros(tuple(s["k_cache"].shape))
            by = np.ones(held.shape[:3])
            if c["cache"] == "e4m3":
                top = np.abs(x).max(-1)
                scale = np.exp2(np.ceil(np.log2(np.where(top > 0, top, 448.0) / 448.0)))
                y = x / scale[..., None]
                step = np.exp2(np.maximum(np.floor(np.log2(np.where(y == 0, 1.0, np.abs(y)))), -6) - 3)
                x = np.rint(y / step) * step
            t = 0
            for n, (q, kv) in enumerate(lengths):
                p = np.arange(kv - q, kv)
                held[table[n, p // ps], :, p % ps] = x[t:t + q]
                if c["cache"] == "e4m3":
                    by[table[n, p // ps], :, p % ps] = scale[t:t + q]
                t += q
            got.append((torch.from_numpy(held), torch.from_numpy(by)))
        return [x for x, _ in got] + ([y for _, y in got] if c["cache"] == "e4m3" else [])

    def row(n, kv, name):  # (kv, kv_heads, head_dim)
        pages = torch.from_numpy(table[n, :-(-kv // ps)].astype(np.int64)).cuda()
        x = s[name + "_cache"].view(torch.uint8)[pages].view(s[name + "_cache"].dtype).double()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][pages].double().unsqueeze(-1)
        return x.permute(0, 2, 1, 3).reshape(-1, hk, d)[:kv]

    if c["op"] == "read":
        if c["batch"] * s["longest"] * hk * d > 600_000_000:
            return None
        outs = [torch.zeros(c["batch"], hk, s["longest"], d, dtype=torch.float64, device="cuda") for _ in range(2)]
        for n, (_, kv) in enumerate(lengths):
            for out, name in zip(outs, ("k", "v")):
                out[n, :, :kv] = row(n, kv, name).transpose(0, 1)
        return tuple(outs)
    g = c["q_heads"] // hk
    flat = s["q"].reshape(-1, c["q_heads"], d)
    out = torch.zeros(flat.shape, dtype=torch.float64, device="cuda")
    t = 0
    for n, (q, kv) in enumerate(lengths):
        k, v = row(n, kv, "k"), row(n, kv, "v")
        p = torch.arange(kv - q, kv, device="cuda")[:, None]
        j = torch.arange(kv, device="cuda")[None]
        hidden = j > p
        if c["window"]:
            hidden |= (j + c["window"] <= p) & (j >= c["sinks"])
        for h in range(hk):
            for i in range(g):
                w = flat[t:t + q, h * g + i].double() @ k[:, h].T
                w = torch.softmax((w / d ** 0.5).masked_fill_(hidden, -math.inf), -1)
                out[t:t + q, h * g + i] = w @ v[:, h]
        t += q
    return out.reshape(s["q"].shape)
