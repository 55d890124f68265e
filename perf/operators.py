"""Operators of a KV cache held in 4 bits, as measurable cases.

The format is OCP MXFP4: elements of 4 bits (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives), one power-of-two scale byte (e8m0) for 32 neighbouring elements of
a head's row.  A chunk (the tokens of one block, K or V, of one layer) is
``[head][token][D/2]`` code bytes (element 2i in the low half of byte i) followed by
``[head][D/32][token]`` scale bytes.

Kinds:
  demote   blocks of the 16-bit paged cache, every layer, go to the 4-bit cache
           (``quantize_kv_blocks``) and come back (``dequantize_kv_blocks``)
  promote  blocks of the 4-bit cache come back to the 16-bit one
  write    new tokens of one layer go to their slots of the 4-bit cache
           (``quantize_kv_tokens``); the blocks that hold them are read back
  attend   attention of the queries over the paged 4-bit cache of one layer
           (``mx4_attention``): single tokens, a few, or the rest of a prompt
  step     the new tokens are written, then attended over: one layer of a step
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# (layers, K/V heads, head size, one latent half): the Llama-3-8B cache, a
# Llama-3-70B TP-8 shard, the DeepSeek MLA latent and the 4-layer CPU-plumbing
# shape of the benchmark configurations.
LLAMA8B = dict(layers=32, heads=8, dim=128, mla=False)
LLAMA70B_TP8 = dict(layers=80, heads=1, dim=128, mla=False)
MLA = dict(layers=61, heads=1, dim=576, mla=True)
SMALL = dict(layers=4, heads=8, dim=128, mla=False)


def _blocks(name, kind, model, blocks, tokens=16, dtype="bf16", layers=0):
    c = dict(name=name, kind=kind, **model, blocks=blocks, tokens=tokens, dtype=dtype)
    c["layers"] = layers or model["layers"]
    return c


def _write(name, count, heads, dim, tokens=16, dtype="bf16"):
    return dict(name=name, kind="write", count=count, heads=heads, dim=dim, tokens=tokens,
                dtype=dtype)


def _attend(name, kind, batch, longest, new, heads, group, dim=128, tokens=16, dtype="bf16",
            blockwise=False):
    """longest: keys of the longest sequence.  new: queries of the longest
    request (the last `new` tokens of its sequence); 1 for every sequence
    when 1."""
    return dict(name=name, kind=kind, batch=batch, longest=longest, new=new, heads=heads,
                group=group, dim=dim, tokens=tokens, dtype=dtype, blockwise=blockwise)


def listed():
    return [
        # One user's next token, a short conversation: all latency.
        _attend("decode_1seq", "attend", 1, 777, 1, 8, 4),
        # The decode step of a busy server, one layer of Llama-3-8B.
        _attend("decode_32seq", "attend", 32, 8192, 1, 8, 4),
        # Long documents on the tensor-parallel shard: one K/V head, so few
        # rows and a long axis to split.
        _attend("decode_long_shard", "attend", 16, 65536, 1, 1, 8, dtype="fp16"),
        # Five drafted tokens of each sequence are written and verified;
        # generic heads of 64, the cache block-wise.
        _attend("step_verify_16seq", "step", 16, 2000, 5, 8, 8, dim=64, dtype="fp16",
                blockwise=True),
        # Prefix hits: the unmatched rest of four prompts attends over cached
        # prefixes of some thousand tokens.
        _attend("extend_4seq", "attend", 4, 6150, 411, 8, 4, tokens=32),
        # A chunk of a long prompt over what is cached before it.
        _attend("prompt_2048_of_8192", "attend", 1, 8192, 2048, 8, 4),
        # 16384 tokens of Llama-3-8B (2 GiB) leave the 16-bit cache and return.
        _blocks("demote_1024blk", "demote", LLAMA8B, 1024),
        # A short request of the MLA latent, blocks of 64 tokens.
        _blocks("demote_mla_5blk", "demote", MLA, 5, tokens=64),
        # A prefix hit of the tensor-parallel shard.
        _blocks("promote_shard_173blk", "promote", LLAMA70B_TP8, 173),
        # One layer of a 256-token prefix: the layer-wise schedule's call.
        _blocks("promote_1layer_16blk", "promote", SMALL, 16, dtype="fp16", layers=1),
        # The tokens of one decode step.
        _write("write_64tok", 64, 8, 128),
        # A prompt's tokens, one layer.
        _write("write_8191tok", 8191, 8, 128),
    ]


def _log(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "step", "demote", "promote", "write"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    tokens = rng.choice((16, 16, 32, 64))
    if kind in ("demote", "promote"):
        model = rng.choice((LLAMA8B, LLAMA8B, LLAMA70B_TP8, MLA, SMALL))
        layers = rng.choice((model["layers"], model["layers"], 1, 2))
        block = layers * (1 if model["mla"] else 2) * tokens * model["heads"] * model["dim"] * 2
        blocks = _log(rng, 1, min(8192, (1 << 30) // block))
        c = _blocks("", kind, model, blocks, tokens, rng.choice((dtype, dtype, "fp32")), layers)
    elif kind == "write":
        c = _write("", _log(rng, 1, 16384), rng.choice((1, 2, 8)), rng.choice((64, 128, 128, 256)),
                   tokens, rng.choice((dtype, dtype, "fp32")))
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
        c = _attend("", kind, batch, longest, new, heads, group, dim, tokens, dtype,
                    rng.random() < 0.3)
    del c["name"]
    return c


# -- what the cases share ------------------------------------------------------


def _lengths(case):
    """Keys and queries of each sequence: the longest first, the others
    spread below it; a sequence has at least as many keys as queries."""
    r = random.Random(case["batch"] * 1000003 + case["longest"] * 31 + case["new"])
    keys, queries = [case["longest"]], [case["new"]]
    for _ in range(case["batch"] - 1):
        n = case["new"] if case["new"] <= 16 else r.randrange(max(1, case["new"] // 4),
                                                              case["new"] + 1)
        queries.append(n)
        keys.append(max(n, r.randrange(max(1, case["longest"] // 4), case["longest"] + 1)))
    return keys, queries


def _chunk(case):
    return case["tokens"] * case["heads"] * case["dim"] * 17 // 32


def _values(g, *shape):
    """K/V rows as models have them: most channels of unit size, some far larger."""
    x = torch.randn(*shape, generator=g, device=DEVICE)
    return x * torch.exp(0.7 * torch.randn(shape[-1], generator=g, device=DEVICE))


def _random_pages(g, halves, blocks, case):
    """Pages of the 4-bit cache, [halves, blocks, chunk] bytes, holding unit-sized
    values: e2m1 codes as normal values have them, scales around 2^-1."""
    H, T, D = case["heads"], case["tokens"], case["dim"]
    pages = torch.empty(halves, blocks, _chunk(case), dtype=torch.uint8, device=DEVICE)
    codes = T * H * D // 2
    step = max(1, (1 << 28) // codes)
    for k in range(halves):
        for b in range(0, blocks, step):
            n = min(step, blocks - b)
            x = torch.randn(2, n, codes, generator=g, device=DEVICE).mul_(2.0)
            c = (x.abs() * 2).round_().clamp_(max=7).to(torch.uint8) + (x < 0).to(torch.uint8) * 8
            pages[k, b:b + n, :codes] = c[0] | (c[1] << 4)
            pages[k, b:b + n, codes:] = torch.randint(
                125, 128, (n, codes // 16), generator=g, device=DEVICE, dtype=torch.uint8)
    return pages


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dt = TYPES[case["dtype"]]
    H, T, D = case["heads"], case["tokens"], case["dim"]
    chunk = _chunk(case)
    s = {"case": case}
    if case["kind"] in ("demote", "promote"):
        L, halves, n = case["layers"], 1 if case["mla"] else 2, case["blocks"]
        pool = n + n // 4 + 3

        def ids():
            d = torch.randperm(pool, generator=g, device=DEVICE)[:n]
            return d, d.cpu().pin_memory()
        s["gpu_ids"], s["gpu_ids_host"] = ids()
        s["mx_ids"], s["mx_ids_host"] = ids()
        s["cache"] = torch.zeros(L, halves, pool, T, H, D, dtype=dt, device=DEVICE)
        if case["kind"] == "demote":
            for l in range(L):
                s["cache"][l] = _values(g, halves, pool, T, H, D).to(dt)
            s["mx"] = torch.zeros(pool, L, halves, chunk, dtype=torch.uint8, device=DEVICE)
            s["back"] = torch.zeros_like(s["cache"])
        else:
            s["mx"] = _random_pages(g, 1, pool * L * halves, case).view(pool, L, halves, chunk)
            s["back"] = s.pop("cache")
        for name in ("cache", "back"):
            if name in s:
                s[name + "_ptrs"] = torch.tensor([x.data_ptr() for x in s[name]],
                                                 dtype=torch.int64).pin_memory()
        return s
    if case["kind"] == "write":
        n = case["count"]
        blocks = (n + 2 * T - 2) // T
        pool = blocks + blocks // 4 + 3
        qkv = _values(g, n, 6 * H, D).to(dt)     # four queries a K/V head lie before K and V
        s["key"], s["value"] = qkv[:, 4 * H:5 * H], qkv[:, 5 * H:]
        s["mx"] = _random_pages(g, 2, pool, case)
        table = torch.randperm(pool, generator=g, device=DEVICE)[:blocks]
        at = torch.arange(n, device=DEVICE) + int(seed) % T      # the tokens follow others
        s["slots"] = table[at // T] * T + at % T
        s["ids"], s["ids_host"] = table, table.cpu().pin_memory()
        s["back"] = torch.zeros(2, blocks, T, H, D, dtype=dt, device=DEVICE)
        s["back_ids_host"] = torch.arange(blocks).pin_memory()
        s["back_ptrs"] = torch.tensor([s["back"].data_ptr()], dtype=torch.int64).pin_memory()
        return s
    keys, queries = _lengths(case)
    B, G = case["batch"], case["group"]
    pages = [-(-k // T) for k in keys]
    width, pool = max(pages), sum(pages) + 3
    mx = _random_pages(g, 2, pool, case)
    if case["blockwise"]:     # [block][K|V][chunk], seen as [K|V][block][chunk]
        mx = mx.transpose(0, 1).contiguous().transpose(0, 1)
    s["mx"] = mx
    perm = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32).tolist()
    table, at = [], 0
    for p in pages:
        table.append(perm[at:at + p] + [0] * (width - p))
        at += p
    s["table"] = torch.tensor(table, dtype=torch.int32, device=DEVICE)
    s["lens"] = torch.tensor(keys, dtype=torch.int32, device=DEVICE)
    starts = [0]
    for n in queries:
        starts.append(starts[-1] + n)
    total = starts[-1]
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE) if case["new"] > 1 \
        else None
    s["scale"] = 1 / math.sqrt(D)
    qkv = torch.randn(total, H * (G + 2), D, generator=g, device=DEVICE).to(dt)
    s["query"] = qkv[:, :H * G]
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

_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _encode(x):
    """Rows [..., D] as codes [..., D/2] and scale bytes [..., D/32]."""
    x = x.to(torch.float32).unflatten(-1, (-1, 32))
    big = x.abs().amax(-1)
    # the exponent of the largest, one more where its mantissa is over 1.75
    e = (((big.view(torch.int32) + 0x1FFFFF) >> 23).clamp(max=254) - 2).clamp(min=0)
    a = torch.ldexp(x, (127 - e)[..., None])
    m = a.abs()
    c = (m > 0.25).to(torch.uint8)
    c += m >= 0.75
    c += m > 1.25
    c += m >= 1.75
    c += m > 2.5
    c += m >= 3.5
    c += m > 5
    c = (c | (torch.signbit(a).to(torch.uint8) << 3)).flatten(-2)
    lost = ~torch.isfinite(big)
    c = torch.where(lost.repeat_interleave(32, -1), 0, c)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.where(lost, 255, e).to(torch.uint8)


def _decode(codes, scales):
    """The values of codes [..., D/2] and scale bytes [..., D/32], in 32 bits."""
    grid = torch.tensor(_GRID, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    s = torch.where(scales == 255, math.nan,
                    torch.ldexp(torch.ones_like(scales, dtype=torch.float32),
                                scales.to(torch.int32) - 127))
    return (grid[c.to(torch.int64)].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _pack(codes, scales):
    """Codes [..., T, H, D/2] and scales [..., T, H, D/32] as chunks."""
    return torch.cat((codes.transpose(-2, -3).flatten(-3),
                      scales.movedim(-3, -1).flatten(-3)), -1)


def _unpack(chunks, case):
    """Chunks [..., bytes] as codes [..., H, T, D/2] and scales [..., H, T, D/32]."""
    H, T, D = case["heads"], case["tokens"], case["dim"]
    split = T * H * D // 2
    return (chunks[..., :split].unflatten(-1, (H, T, D // 2)),
            chunks[..., split:].unflatten(-1, (H, D // 32, T)).transpose(-1, -2))


def _rounded(x, dt):
    top = torch.finfo(dt).max
    return x.clamp(-top, top).to(dt)


def _plain_write(s):
    case = s["case"]
    H, T, D = case["heads"], case["tokens"], case["dim"]
    codes, scales = _encode(torch.stack((s["key"], s["value"])))
    block, t = s["slots"] // T, s["slots"] % T
    c, sc = _unpack(s["mx"], case)               # views of the cache
    c[:, block, :, t] = codes.transpose(0, 1)
    sc[:, block, :, t] = scales.transpose(0, 1)


def _plain_attention(s):
    case = s["case"]
    H, G, T, D = case["heads"], case["group"], case["tokens"], case["dim"]
    B, n = case["batch"], case["new"]
    codes, scales = _unpack(s["mx"][:, s["table"].to(torch.int64)], case)
    kv = _decode(codes.transpose(2, 3).flatten(3, 4), scales.transpose(2, 3).flatten(3, 4))
    q = torch.zeros(B, n, H * G, D, device=DEVICE)
    q[s["seq"], s["off"]] = s["query"].to(torch.float32)
    q = q.view(B, n, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, D)
    w = torch.matmul(q, kv[0].transpose(-1, -2).contiguous()) * s["scale"]
    last = torch.full((B, n), -1, device=DEVICE, dtype=torch.int64)
    last[s["seq"], s["off"]] = s["pos"]
    seen = torch.arange(w.shape[-1], device=DEVICE) <= last[..., None]
    w = w.view(B, H, G, n, -1).masked_fill_(~seen[:, None, None], -math.inf)
    w = w - w.amax(-1, keepdim=True).clamp_(min=-1e30)
    w = w.exp_()
    w = w / w.sum(-1, keepdim=True).clamp_(min=1e-30)
    v = kv[1].masked_fill(~(torch.arange(kv.shape[-2], device=DEVICE)
                            < s["lens"][:, None])[:, None, :, None], 0)
    o = torch.matmul(w.view(B, H, G * n, -1), v).view(B, H, G, n, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, H * G, D)[s["seq"], s["off"]].to(
        s["query"].dtype)


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "demote":
        x = s["cache"][:, :, s["gpu_ids"]]
        s["mx"][s["mx_ids"]] = _pack(*_encode(x)).permute(2, 0, 1, 3)
    if kind in ("demote", "promote"):
        codes, scales = _unpack(s["mx"][s["mx_ids"]], case)
        x = _decode(codes, scales).permute(1, 2, 0, 4, 3, 5)
        s["back"][:, :, s["gpu_ids"]] = _rounded(x, s["back"].dtype)
        return s["back"]
    if kind in ("write", "step"):
        _plain_write(s)
    if kind == "write":
        x = _decode(*_unpack(s["mx"][:, s["ids"]], case))
        s["back"][:] = _rounded(x.transpose(2, 3), s["back"].dtype)
        return s["back"]
    return _plain_attention(s)


# -- the framework's calls ---------------------------------------------------------


def _own(s):
    from flexkv_amd import c_ext

    case = s["case"]
    kind = case["kind"]
    chunk = _chunk(case)
    shape = (case["tokens"], case["heads"], case["dim"])
    if kind in ("demote", "promote"):
        mx = s["mx"]
        halves = mx.shape[2]
        strides = (chunk, halves * chunk, mx.stride(0))     # K|V, layer, block
        size = shape[0] * shape[1] * shape[2] * s["back"].element_size()
        rest = (s["mx_ids_host"], mx, *strides, *shape, s["back"].dtype, 0, halves == 1)
        if kind == "demote":
            c_ext.quantize_kv_blocks(s["gpu_ids_host"], s["cache_ptrs"],
                                     s["cache"].shape[2] * size, size, *rest)
        c_ext.dequantize_kv_blocks(s["gpu_ids_host"], s["back_ptrs"], s["back"].shape[2] * size,
                                   size, *rest)
        return s["back"]
    if kind in ("write", "step"):
        c_ext.quantize_kv_tokens(s["key"], s["value"], s["mx"], s["slots"])
    if kind == "write":
        mx, back = s["mx"], s["back"]
        size = shape[0] * shape[1] * shape[2] * back.element_size()
        c_ext.dequantize_kv_blocks(s["back_ids_host"], s["back_ptrs"], back.shape[1] * size, size,
                                   s["ids_host"], mx, mx.stride(0), 0, chunk, *shape, back.dtype)
        return back
    return c_ext.mx4_attention(s["query"], s["mx"], case["heads"], s["table"], s["lens"],
                               s["starts"], scale=s["scale"])


def run(state):
    return _own(state) if own else _plain(state)


# -- what a pass cannot do without, and what it ought to return ----------------------


def work(case):
    size = TYPES[case["dtype"]].itemsize
    H, D = case["heads"], case["dim"]
    if case["kind"] in ("demote", "promote"):
        n = case["layers"] * (1 if case["mla"] else 2) * case["blocks"] * case["tokens"] * H * D
        once = n * (size + 17 / 32)
        return {"bytes": once * (2 if case["kind"] == "demote" else 1), "flops": 0}
    if case["kind"] == "write":
        n = 2 * case["count"] * H * D
        T = case["tokens"]
        whole = 2 * ((case["count"] + 2 * T - 2) // T) * T * H * D
        return {"bytes": (n + whole) * (size + 17 / 32), "flops": 0}
    keys, queries = _lengths(case)
    rows = H * case["group"] * sum(queries)
    pairs = H * case["group"] * sum(n * (k - n) + n * (n + 1) // 2
                                    for k, n in zip(keys, queries))
    new = 2 * sum(queries) * H * D * (size + 17 / 32) if case["kind"] == "step" else 0
    return {"bytes": 2 * sum(keys) * H * D * 17 / 32 + 2 * rows * D * size + new,
            "flops": 4 * pairs * D}


def _read64(chunks, case):
    """[..., bytes] -> [..., T, H, D] in 64 bits, from the format's definition."""
    H, T, D = case["heads"], case["tokens"], case["dim"]
    cut = T * H * D // 2
    b = chunks[..., :cut].reshape(*chunks.shape[:-1], H, T, D // 2, 1).to(torch.int64)
    c = torch.cat((b % 16, b // 16), -1).reshape(*chunks.shape[:-1], H, T, D)
    m, e = c % 2, c // 2 % 4
    mag = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * 2.0 ** (e - 1).to(torch.float64))
    sc = chunks[..., cut:].reshape(*chunks.shape[:-1], H, D // 32, T).to(torch.float64)
    sc = torch.where(sc == 255, math.nan, 2.0 ** (sc - 127)).transpose(-1, -2)
    x = torch.where(c >= 8, -mag, mag) * sc.repeat_interleave(32, -1)
    return x.transpose(-2, -3)


def _quantised64(x):
    """The values that rows [..., D] have once held in 4 bits, in 64 bits."""
    shape = x.shape
    x = x.to(torch.float64).reshape(-1, 32)
    big = x.abs().amax(1, keepdim=True)
    m, e = torch.frexp(big)                       # big = m 2^e, m in [0.5, 1)
    e = torch.where(big > 0, e + (m > 0.875).to(e.dtype) - 1, -127).clamp(max=127)
    s = 2.0 ** (e - 2).clamp(min=-127).to(torch.float64)
    a = (x / s).abs()
    # steps of 0.5 below 2, of 1 below 4, of 2 below 6; torch rounds ties to even
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(torch.float64)
    a = ((a / step).round() * step).clamp(max=6)
    return torch.where(torch.isfinite(big), torch.copysign(a, x) * s, math.nan).reshape(shape)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    T = case["tokens"]
    if kind in ("demote", "promote"):
        if s["back"].numel() > 1 << 31:
            return None
        out = torch.zeros(s["back"].shape, dtype=torch.float64, device=DEVICE)
        for l in range(case["layers"]):
            out[l][:, s["gpu_ids"]] = _quantised64(s["cache"][l][:, s["gpu_ids"]]) \
                if kind == "demote" else _read64(s["mx"][s["mx_ids"], l], case).transpose(0, 1)
        return out
    if kind == "write":
        out = _read64(s["mx"][:, s["ids"]], case).contiguous()
        where = torch.empty(s["mx"].shape[1], dtype=torch.int64, device=DEVICE)
        where[s["ids"]] = torch.arange(s["ids"].numel(), device=DEVICE)
        new = _quantised64(torch.stack((s["key"], s["value"])))
        out[:, where[s["slots"] // T], s["slots"] % T] = new
        return out
    keys, queries = _lengths(case)
    H, G, D = case["heads"], case["group"], case["dim"]
    rows, at = [], 0
    for b, (k, n) in enumerate(zip(keys, queries)):
        pages = s["table"][b, :-(-k // T)].to(torch.int64)
        kv = _read64(s["mx"][:, pages], case).reshape(2, -1, H, D)[:, :k].clone()
        if kind == "step":
            kv[:, k - n:] = _quantised64(torch.stack((s["key"][at:at + n],
                                                      s["value"][at:at + n])))
        q = s["query"][at:at + n].to(torch.float64) * s["scale"]
        per_head = []
        for h in range(H * G):
            w = q[:, h] @ kv[0, :, h // G].T
            reach = torch.arange(k, device=DEVICE)[None] - torch.arange(n, device=DEVICE)[:, None]
            w = torch.softmax(w.masked_fill(reach > k - n, -math.inf), -1)
            per_head.append(w @ kv[1, :, h // G])
        rows.append(torch.stack(per_head, 1))
        at += n
    return torch.cat(rows)
