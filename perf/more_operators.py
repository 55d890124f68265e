"""Operators on the paged 16-bit KV cache, as measurable cases: attention of new tokens
over it, with what every cached token got of that attention added up, and eviction by
those sums.

A layer's cache is ``key_cache`` and ``value_cache``, [block][token][K/V head][D]; token t
of sequence b lies in block ``table[b][t / T]`` at t % T.  ``weights[b][h][t]`` is what
token t of sequence b got of the attention of K/V head h's queries.

Kinds:
  write    new tokens of one layer go to their slots (``write_kv_tokens``)
  attend   attention of the queries over the cache (``paged_attention``): single tokens, a
           few, or the rest of a prompt; ``weigh``: each cached token's share is added up
  step     the new tokens are written, then attended over and weighed
  evict    each sequence keeps, for every K/V head, its most recent tokens and those with
           the largest sums, in blocks of their own (``evict_kv_tokens``)
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _attend(name, kind, batch, longest, new, heads, group, dim=128, tokens=16, dtype="bf16",
            blockwise=False, weigh=False):
    """longest: keys of the longest sequence.  new: queries of the longest
    request (the last `new` tokens of its sequence); 1 for every sequence
    when 1."""
    return dict(name=name, kind=kind, batch=batch, longest=longest, new=new, heads=heads,
                group=group, dim=dim, tokens=tokens, dtype=dtype, blockwise=blockwise,
                weigh=weigh)


def _write(name, count, heads, dim, tokens=16, dtype="bf16"):
    return dict(name=name, kind="write", count=count, heads=heads, dim=dim, tokens=tokens,
                dtype=dtype)


def _evict(name, batch, longest, budget, recent, heads, dim=128, tokens=16, dtype="bf16",
           blockwise=False):
    return dict(name=name, kind="evict", batch=batch, longest=longest, budget=budget,
                recent=recent, heads=heads, dim=dim, tokens=tokens, dtype=dtype,
                blockwise=blockwise)


def listed():
    return [
        # One user's next token, a short conversation: all latency.
        _attend("decode_1seq", "attend", 1, 777, 1, 8, 4),
        # The decode step of a busy server, one layer of Llama-3-8B.
        _attend("decode_32seq", "attend", 32, 8192, 1, 8, 4),
        # Long documents on the tensor-parallel shard: one K/V head, so few
        # rows and a long axis to split.
        _attend("decode_long_shard", "attend", 16, 65536, 1, 1, 8, dtype="fp16"),
        # Prefix hits: the unmatched rest of four prompts attends over cached
        # prefixes of some thousand tokens.
        _attend("extend_4seq", "attend", 4, 6150, 411, 8, 4, tokens=32),
        # A chunk of a long prompt over what is cached before it.
        _attend("prompt_2048_of_8192", "attend", 1, 8192, 2048, 8, 4),
        # The busy server's step where the cache is to be evicted from: every
        # cached token's share is added to its sum.
        _attend("weigh_decode_32seq", "attend", 32, 8192, 1, 8, 4, weigh=True),
        # The last 64 tokens of long prompts decide what to keep of them.
        _attend("weigh_window_4seq", "attend", 4, 16384, 64, 8, 4, weigh=True),
        # Five drafted tokens of each sequence are written and verified;
        # generic heads of 64, the cache block-wise.
        _attend("step_verify_16seq", "step", 16, 2000, 5, 8, 8, dim=64, dtype="fp16",
                blockwise=True, weigh=True),
        # A prompt's tokens, one layer.
        _write("write_8191tok", 8191, 8, 128),
        # The busy server's sequences are cut to 2048 tokens, one layer.
        _evict("evict_32seq_to_2048", 32, 8192, 2048, 512, 8),
        # Two long documents on the tensor-parallel shard.
        _evict("evict_2long_shard", 2, 65536, 8192, 1024, 1, dtype="fp16"),
        # One short conversation: all latency.
        _evict("evict_1seq_777_to_500", 1, 777, 500, 50, 8),
    ]


def _log(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "attend", "step", "write", "evict", "evict"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    tokens = rng.choice((16, 16, 32, 64, 8, 1))
    blockwise = rng.random() < 0.3
    if kind == "write":
        c = _write("", _log(rng, 1, 16384), rng.choice((1, 2, 8)), rng.choice((64, 128, 128, 256)),
                   tokens, dtype)
    elif kind == "evict":
        heads, dim = rng.choice((1, 2, 8, 8)), rng.choice((64, 128, 128, 256))
        batch = _log(rng, 1, 32)
        most = min(65536, (1 << 28) // (batch * heads * dim))
        longest = _log(rng, 16, most)
        # no more tokens stay than of the busy server's sequences
        budget = min(_log(rng, 1, longest), max(1, (1 << 26) // (batch * heads * dim)))
        c = _evict("", batch, longest, budget, rng.randrange(budget + 1) // 2, heads, dim, tokens,
                   dtype, blockwise)
    else:
        heads, group = rng.choice(((8, 4), (8, 4), (1, 8), (8, 8), (2, 5), (8, 1), (1, 16)))
        dim = rng.choice((64, 128, 128, 128, 256))
        form = rng.choice(("one", "one", "few", "many"))
        if form == "one":
            batch, new = _log(rng, 1, 64), 1
        elif form == "few":
            batch, new = _log(rng, 1, 32), rng.randrange(2, 17)
        else:
            batch, new = _log(rng, 1, 8), _log(rng, 17, 2048)
        # no more bytes of keys and values than the busy server's step reads, and
        # no more products than the chunk of the long prompt makes
        pairs = 2048 * 8192 * 32 * 128 // (batch * heads * group * dim)
        new = min(new, math.isqrt(pairs))
        most = min(65536, (1 << 28) // (batch * heads * dim), pairs // new)
        new = min(new, most)
        longest = max(new, _log(rng, 1, most))
        c = _attend("", kind, batch, longest, new, heads, group, dim, tokens, dtype, blockwise,
                    kind == "step" or rng.random() < 0.4)
    del c["name"]
    return c


# -- what the cases share ------------------------------------------------------


def _lengths(case):
    """Keys and queries of each sequence: the longest first, the others
    spread below it; a sequence has at least as many keys as queries."""
    new = case.get("new", 1)
    r = random.Random(case["batch"] * 1000003 + case["longest"] * 31 + new)
    keys, queries = [case["longest"]], [new]
    for _ in range(case["batch"] - 1):
        n = new if new <= 16 else r.randrange(max(1, new // 4), new + 1)
        queries.append(n)
        keys.append(max(n, r.randrange(max(1, case["longest"] // 4), case["longest"] + 1)))
    return keys, queries


def _channels(g, dim):
    """Sizes of the channels of K and V as models have them: most near 1, some far larger."""
    return torch.exp(0.7 * torch.randn(dim, generator=g, device=DEVICE))


def _cache(g, blocks, case):
    """Keys and values [block][token][head][D], filled, as views of one tensor: K before
    all V, or block by block."""
    H, T, D = case["heads"], case["tokens"], case["dim"]
    dt = TYPES[case["dtype"]]
    cache = torch.empty(2, blocks, T, H, D, dtype=dt, device=DEVICE)
    for half in cache:
        size = _channels(g, D)
        step = max(1, (1 << 26) // (T * H * D))
        for b in range(0, blocks, step):
            x = half[b:b + step]
            x.copy_(torch.randn(x.shape, generator=g, device=DEVICE).mul_(size))
    if case.get("blockwise"):
        cache = cache.transpose(0, 1).contiguous().transpose(0, 1)
    return cache


def _tables(counts, perm):
    """A table of blocks for each sequence, taken from `perm`, rows filled up with 0."""
    width, table, at = max(counts), [], 0
    for p in counts:
        table.append(perm[at:at + p] + [0] * (width - p))
        at += p
    return torch.tensor(table, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dt = TYPES[case["dtype"]]
    H, T, D = case["heads"], case["tokens"], case["dim"]
    s = {"case": case}
    if case["kind"] == "write":
        n = case["count"]
        blocks = (n + 2 * T - 2) // T
        pool = blocks + blocks // 4 + 3
        # four queries a K/V head lie before K and V
        qkv = (torch.randn(n, 6 * H, D, generator=g, device=DEVICE) * _channels(g, D)).to(dt)
        s["key"], s["value"] = qkv[:, 4 * H:5 * H], qkv[:, 5 * H:]
        s["cache"] = _cache(g, pool, case)
        table = torch.randperm(pool, generator=g, device=DEVICE)[:blocks]
        at = torch.arange(n, device=DEVICE) + int(seed) % T      # the tokens follow others
        s["slots"] = table[at // T] * T + at % T
        return s
    keys, queries = _lengths(case)
    B = case["batch"]
    pages = [-(-k // T) for k in keys]
    s["lens"] = torch.tensor(keys, dtype=torch.int32, device=DEVICE)
    if case["kind"] == "evict":
        new_pages = [-(-min(k, case["budget"]) // T) for k in keys]
        pool = sum(pages) + sum(new_pages) + 3
        perm = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32).tolist()
        s["table"] = _tables(pages, perm)
        s["new_table"] = _tables(new_pages, perm[sum(pages):])
        s["cache"] = _cache(g, pool, case)
        # few tokens get most of the attention, and some so little that it rounds to nothing
        w = torch.exp(2.5 * torch.randn(B, H, s["table"].shape[1] * T, generator=g, device=DEVICE))
        s["weights"] = torch.where(w < 0.01, 0.0, w)
        s["new_weights"] = torch.zeros(B, H, case["budget"], device=DEVICE)
        return s
    G, width, pool = case["group"], max(pages), sum(pages) + 3
    s["cache"] = _cache(g, pool, case)
    perm = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32).tolist()
    s["table"] = _tables(pages, perm)
    starts = [0]
    for n in queries:
        starts.append(starts[-1] + n)
    total = starts[-1]
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE) if case["new"] > 1 \
        else None
    s["scale"] = 1 / math.sqrt(D)
    qkv = torch.randn(total, H * (G + 2), D, generator=g, device=DEVICE).to(dt)
    s["query"] = qkv[:, :H * G]
    if case["weigh"]:
        s["weights"] = torch.rand(B, H, width * T, generator=g, device=DEVICE)
    # for the plain form: the place of every query in [sequence, newest tokens]
    seq = [b for b, n in enumerate(queries) for _ in range(n)]
    off = [i for n in queries for i in range(n)]
    s["seq"] = torch.tensor(seq, device=DEVICE)
    s["off"] = torch.tensor(off, device=DEVICE)
    s["pos"] = torch.tensor([keys[b] - queries[b] + i for b, i in zip(seq, off)], device=DEVICE)
    if case["kind"] == "step":
        s["key"], s["value"] = qkv[:, H * G:H * (G + 1)], qkv[:, H * (G + 1):]
        s["slots"] = s["table"][s["seq"], s["pos"] // T].to(torch.int64) * T + s["pos"] % T
    return s


# -- the plain form --------------------------------------------------------------


def _plain_write(s):
    T = s["case"]["tokens"]
    block, t = s["slots"] // T, s["slots"] % T
    s["cache"][0][block, t] = s["key"]
    s["cache"][1][block, t] = s["value"]


def _plain_attention(s):
    case = s["case"]
    H, G, D = case["heads"], case["group"], case["dim"]
    B, n = case["batch"], case["new"]
    table = s["table"].to(torch.int64)
    # [sequence, head, key, D]
    k, v = (c[table].flatten(1, 2).transpose(1, 2).to(torch.float32) for c in s["cache"])
    q = torch.zeros(B, n, H * G, D, device=DEVICE)
    q[s["seq"], s["off"]] = s["query"].to(torch.float32)
    q = q.view(B, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    w = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    last = torch.full((B, n), -1, device=DEVICE, dtype=torch.int64)
    last[s["seq"], s["off"]] = s["pos"]
    seen = torch.arange(w.shape[-1], device=DEVICE) <= last[..., None]
    w = w.view(B, H, G, n, -1).masked_fill_(~seen[:, None, None], -math.inf)
    w = w - w.amax(-1, keepdim=True).clamp_(min=-1e30)
    w = w.exp_()
    w = w / w.sum(-1, keepdim=True).clamp_(min=1e-30)
    o = torch.matmul(w.view(B, H, G * n, -1), v.contiguous()).view(B, H, G, n, D)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, H * G, D)[s["seq"], s["off"]].to(s["query"].dtype)
    if not case["weigh"]:
        return o
    return o, s["weights"] + w.sum((2, 3))


def _plain_evict(s):
    case = s["case"]
    T, budget, recent = case["tokens"], case["budget"], case["recent"]
    w, lens = s["weights"], s["lens"].to(torch.int64)
    B, H, width = w.shape
    at = torch.arange(width, device=DEVICE)
    # the most recent first, then by weight, ties by place; what is no token last
    rank = torch.where(at >= (lens - recent)[:, None], math.inf, 0.0)[:, None] + w
    rank = rank.masked_fill((at >= lens[:, None])[:, None], -1.0)
    order = torch.argsort(rank, dim=-1, descending=True, stable=True)[..., :budget]
    order = torch.nn.functional.pad(order, (0, budget - order.shape[-1]), value=width)
    counts = lens.clamp(max=budget)
    there = (torch.arange(budget, device=DEVICE) < counts[:, None])[:, None].expand(B, H, budget)
    kept = order.masked_fill(~there, width).sort(-1).values
    s["new_weights"].copy_(torch.where(there, w.gather(-1, kept.clamp(max=width - 1)), 0.0))
    b, h, i = there.nonzero(as_tuple=True)
    t = kept[b, h, i]
    old, new = s["table"][b, t // T].to(torch.int64), s["new_table"][b, i // T].to(torch.int64)
    for c in s["cache"]:
        c[new, i % T, h] = c[old, t % T, h]
    return kept.masked_fill(~there, -1).to(torch.int32), s["new_weights"], s["cache"]


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "evict":
        return _plain_evict(s)
    if kind in ("write", "step"):
        _plain_write(s)
    if kind == "write":
        return s["cache"]
    out = _plain_attention(s)
    return (*out, s["cache"]) if kind == "step" else out


# -- the framework's calls ---------------------------------------------------------


def _own(s):
    from flexkv_amd import c_ext

    case = s["case"]
    kind = case["kind"]
    key_cache, value_cache = s["cache"][0], s["cache"][1]
    if kind == "evict":
        kept = c_ext.evict_kv_tokens(key_cache, value_cache, s["weights"], s["table"], s["lens"],
                                     s["new_table"], case["budget"], case["recent"],
                                     new_weights=s["new_weights"])
        return kept, s["new_weights"], s["cache"]
    if kind in ("write", "step"):
        c_ext.write_kv_tokens(s["key"], s["value"], key_cache, value_cache, s["slots"])
    if kind == "write":
        return s["cache"]
    # a pass adds to the same sums each time
    weights = s["weights"].clone() if case["weigh"] else None
    out = c_ext.paged_attention(s["query"], key_cache, value_cache, s["table"], s["lens"],
                                s["starts"], scale=s["scale"], weights=weights)
    if not case["weigh"]:
        return out
    return (out, weights, s["cache"]) if kind == "step" else (out, weights)


def run(state):
    return _own(state) if own else _plain(state)


# -- what a pass cannot do without, and what it ought to return ----------------------


def work(case):
    size = TYPES[case["dtype"]].itemsize
    H, D = case["heads"], case["dim"]
    if case["kind"] == "write":
        return {"bytes": 4 * case["count"] * H * D * size + 8 * case["count"], "flops": 0}
    keys, queries = _lengths(case)
    if case["kind"] == "evict":
        stay = sum(min(k, case["budget"]) for k in keys)
        return {"bytes": H * (4 * stay * D * size + 4 * sum(keys) + 8 * stay), "flops": 0}
    rows = H * case["group"] * sum(queries)
    pairs = H * case["group"] * sum(n * (k - n) + n * (n + 1) // 2
                                    for k, n in zip(keys, queries))
    new = 4 * sum(queries) * H * D * size if case["kind"] == "step" else 0
    sums = 8 * sum(keys) * H if case["weigh"] else 0
    return {"bytes": 2 * sum(keys) * H * D * size + 2 * rows * D * size + new + sums,
            "flops": 4 * pairs * D}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    T, H, D = case["tokens"], case["heads"], case["dim"]
    cache = s["cache"].to(torch.float64)
    if kind in ("write", "step"):
        for half, x in zip(cache, (s["key"], s["value"])):
            for h in range(H):
                half[s["slots"] // T, s["slots"] % T, h] = x[:, h].to(torch.float64)
    if kind == "write":
        return cache
    keys, queries = _lengths(case)
    if kind == "evict":
        budget = case["budget"]
        w = s["weights"].cpu().to(torch.float64)
        kept = torch.full((case["batch"], H, budget), -1, dtype=torch.int64)
        sums = torch.zeros(case["batch"], H, budget, dtype=torch.float64)
        for b, n in enumerate(keys):
            stay = min(n, budget)
            first = n - min(case["recent"], stay)          # of the most recent
            for h in range(H):
                # by weight, of equal ones the earlier
                best = torch.sort(-w[b, h, :first], stable=True).indices[:stay - (n - first)]
                kept[b, h, :stay] = torch.cat((best.sort().values, torch.arange(first, n)))
                sums[b, h, :stay] = w[b, h, kept[b, h, :stay]]
            t = kept[b, :, :stay].to(DEVICE)
            i = torch.arange(stay, device=DEVICE)
            for h in range(H):
                old = s["table"][b, t[h] // T].to(torch.int64)
                new = s["new_table"][b, i // T].to(torch.int64)
                cache[:, new, i % T, h] = cache[:, old, t[h] % T, h]
        return kept.to(torch.int32), sums, cache
    G, rows, at = case["group"], [], 0
    sums = s["weights"].to(torch.float64) if case["weigh"] else None
    for b, (k, n) in enumerate(zip(keys, queries)):
        pages = s["table"][b, :-(-k // T)].to(torch.int64)
        kv = cache[:, pages].reshape(2, -1, H, D)[:, :k]
        q = s["query"][at:at + n].to(torch.float64) * s["scale"]
        reach = torch.arange(k, device=DEVICE)[None] - torch.arange(n, device=DEVICE)[:, None]
        per_head = []
        for h in range(H * G):
            w = q[:, h] @ kv[0, :, h // G].T
            w = torch.softmax(w.masked_fill(reach > k - n, -math.inf), -1)
            per_head.append(w @ kv[1, :, h // G])
            if sums is not None:
                sums[b, h // G, :k] += w.sum(0)
        rows.append(torch.stack(per_head, 1))
        at += n
    out = torch.cat(rows)
    if sums is None:
        return out
    return (out, sums, cache) if kind == "step" else (out, sums)
