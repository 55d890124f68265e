"""The 4-bit KV cache on the device: quantised bytes and values read back against the
oracle bit for bit, attention over the cache against 64 bits."""
import math

import numpy as np
import pytest
import torch

from flexkv_amd import _lib, c_ext
from flexkv_amd.common.storage import KVCacheLayout, KVCacheLayoutType
from flexkv_amd.storage.allocator import pinned_empty

import mx4_oracle as mo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _hard_rows(shape, dtype, g):
    """Values over many magnitudes, with ties, zeros, extremes, infinities and NaN."""
    x = torch.randn(shape, generator=g) * torch.exp2(
        torch.randint(-20, 14, (*shape[:-1], 1), generator=g).float())
    flat = x.view(-1, 32)
    n = flat.shape[0]
    ties = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5., 6., 7., .5, 1., 1.5, 2., 3., 4., 0.])
    flat[1 % n, :16] = ties
    flat[1 % n, 16:] = -ties
    flat[2 % n] = 0
    flat[3 % n] = -0.0
    flat[4 % n] = torch.finfo(dtype).max
    flat[5 % n, 7] = float("inf")
    flat[6 % n, 8] = float("nan")
    flat[7 % n] = torch.finfo(dtype).tiny * torch.rand(32, generator=g)
    flat[8 % n, 3] = -float("inf")
    flat[9 % n] = torch.finfo(dtype).max * torch.rand(32, generator=g)
    flat[10 % n] = 1.75 * 2.0 ** torch.randint(-3, 2, (32,), generator=g)
    return x.to(dtype)


def _bytes(t):
    return t.cpu().contiguous().view(torch.uint8)


def _same(a, b):
    """Equal as bytes, NaN for NaN."""
    a, b = a.cpu(), b.cpu()
    both = torch.isnan(a) & torch.isnan(b)
    same = _bytes(a).view(*a.shape, -1) == _bytes(b).view(*b.shape, -1)
    return bool((same.all(-1) | both).all())


# -- blocks ------------------------------------------------------------------------

class Blocks:
    """A wide GPU cache, a 4-bit one, and the calls between them."""

    def __init__(self, L, T, H, D, dtype, mla=False, n_gpu=6, n_mx=7, kind="BLOCKWISE", start=0,
                 mx_layers=None, host=False, seed=0):
        self.shape, self.dtype, self.mla, self.start = (T, H, D), dtype, mla, start
        self.L, self.kv = L, 1 if mla else 2
        g = _gen(seed)
        self.wide_host = [_hard_rows((self.kv, n_gpu, T, H, D), dtype, g) for _ in range(L)]
        self.wide = [t.to(DEV) for t in self.wide_host]
        self.ptrs = torch.tensor([t.data_ptr() for t in self.wide], dtype=torch.int64)
        wide = KVCacheLayout(KVCacheLayoutType.LAYERWISE, 1, n_gpu, T, H, D, is_mla=mla)
        self.chunk, self.gkv, _, self.gblk = wide.byte_strides(dtype)
        self.lay = KVCacheLayout(KVCacheLayoutType(kind), mx_layers or L + start, n_mx, T, H, D,
                                 is_mla=mla).mx4()
        self.mchunk, self.mkv, self.mlay, self.mblk = self.lay.byte_strides(torch.uint8)
        n = self.lay.get_total_elements()
        fill = torch.randint(0, 256, (n,), generator=g, dtype=torch.uint8)
        self.before = fill.clone()
        if host:
            self.mx = pinned_empty(n, torch.uint8)
            self.mx.copy_(fill)
        else:
            self.mx = fill.to(DEV)

    def call(self, fn, gids, mids):
        gids, mids = (torch.tensor(i, dtype=torch.int64) for i in (gids, mids))
        fn(gids, self.ptrs, self.gkv, self.gblk, mids, self.mx, self.mkv, self.mlay,
           self.mblk, *self.shape, self.dtype, self.start, self.mla)

    def at(self, l, k, mid):
        return (l + self.start) * self.mlay + k * self.mkv + mid * self.mblk

    def want_mx(self, gids, mids):
        out = self.before.numpy().copy()
        for l in range(self.L):
            for k in range(self.kv):
                for gid, mid in zip(gids, mids):
                    x = self.wide_host[l][k, gid].double().numpy()
                    o = self.at(l, k, mid)
                    out[o:o + self.mchunk] = mo.pack_chunk(*mo.encode(x))
        return torch.from_numpy(out)

    def want_wide(self, gids, mids, mx):
        out = [t.clone() for t in self.wide_host]
        for l in range(self.L):
            for k in range(self.kv):
                for gid, mid in zip(gids, mids):
                    o = self.at(l, k, mid)
                    v = mo.chunk_values(mx[o:o + self.mchunk].numpy(), *self.shape)
                    out[l][k, gid] = mo.as_type(v, self.dtype)
        return out


BLOCK_SHAPES = [
    dict(L=3, T=16, H=2, D=64, dtype=BF16),
    dict(L=2, T=32, H=1, D=128, dtype=FP16, kind="LAYERWISE"),
    dict(L=1, T=16, H=3, D=32, dtype=FP32),
    dict(L=2, T=16, H=1, D=576, dtype=BF16, mla=True),
    dict(L=2, T=48, H=5, D=96, dtype=FP16, start=2, mx_layers=5),
    dict(L=2, T=16, H=2, D=128, dtype=BF16, host=True),
    dict(L=130, T=16, H=1, D=32, dtype=BF16),
    dict(L=2, T=64, H=1, D=576, dtype=BF16, mla=True, host=True),
    dict(L=1, T=32, H=2, D=1024, dtype=FP32),
]


@pytest.mark.parametrize("kw", BLOCK_SHAPES, ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_blocks_quantise_and_come_back_bit_for_bit(kw):
    c = Blocks(**kw)
    gids, mids = [4, 0, 3], [6, 2, 5]
    c.call(c_ext.quantize_kv_blocks, gids, mids)
    want = c.want_mx(gids, mids)
    assert torch.equal(c.mx.cpu(), want)
    # read into other blocks, from bytes of every kind where nothing was written
    gids, mids = [1, 5, 2, 0], [2, 0, 6, 3]
    c.call(c_ext.dequantize_kv_blocks, gids, mids)
    for got, w in zip(c.wide, c.want_wide(gids, mids, want)):
        assert _same(got, w)
    assert torch.equal(c.mx.cpu(), want)


def test_many_blocks_take_the_table_on_the_device():
    n = 300                                  # more than the kernel arguments carry
    c = Blocks(L=2, T=16, H=1, D=32, dtype=BF16, n_gpu=n + 9, n_mx=n + 4)
    g = _gen(5)
    gids, mids = torch.randperm(n + 9, generator=g)[:n].tolist(), torch.randperm(
        n + 4, generator=g)[:n].tolist()
    c.call(c_ext.quantize_kv_blocks, gids, mids)
    want = c.want_mx(gids, mids)
    assert torch.equal(c.mx.cpu(), want)
    c.call(c_ext.dequantize_kv_blocks, gids[::-1], mids)
    for got, w in zip(c.wide, c.want_wide(gids[::-1], mids, want)):
        assert _same(got, w)


def test_ids_past_32_bits_are_addressed():
    c = Blocks(L=1, T=16, H=1, D=64, dtype=BF16)
    c.gblk = 0                               # every id is the first block
    c.call(c_ext.quantize_kv_blocks, [(1 << 40) + 3], [2])
    assert torch.equal(c.mx.cpu(), c.want_mx([0], [2]))


def test_every_bf16_and_fp16_pattern_is_rounded_as_the_oracle_does():
    for dtype in (BF16, FP16):
        bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
        # a power of two of the same group size keeps the scale fixed for 31 of 32
        x = bits.view(dtype).view(1, 1, 32, 16, 128).clone()
        x = x.nan_to_num(0.5, 1.5, -3.0)
        c = Blocks(L=1, T=32, H=16, D=128, dtype=dtype, mla=True, n_gpu=1, n_mx=1)
        c.wide_host = [x.view(1, 1, 32, 16, 128)]
        c.wide[0].copy_(c.wide_host[0])
        c.call(c_ext.quantize_kv_blocks, [0], [0])
        assert torch.equal(c.mx.cpu(), c.want_mx([0], [0]))


def test_every_code_and_scale_reads_back():
    T, H, D = 16, 16, 32                    # 256 groups: one for each scale byte
    for dtype in (BF16, FP16, FP32):
        c = Blocks(L=1, T=T, H=H, D=D, dtype=dtype, mla=True, n_gpu=1, n_mx=1)
        codes = np.tile(np.arange(32, dtype=np.uint8) % 16, (T, H, 1))
        scales = np.arange(256, dtype=np.uint8).reshape(T, H, 1)
        c.mx.copy_(torch.from_numpy(mo.pack_chunk(codes, scales)))
        c.call(c_ext.dequantize_kv_blocks, [0], [0])
        assert _same(c.wide[0][0, 0], mo.as_type(mo.decode(codes, scales), dtype))


def test_blocks_are_refused_where_they_leave_their_allocations():
    c = Blocks(L=2, T=16, H=1, D=64, dtype=BF16)
    # torch serves small tensors from larger allocations: ids far past both
    for gids, mids, word in (([1 << 30], [0], "gpu block ids"), ([0], [1 << 30], "4-bit block ids")):
        with pytest.raises(RuntimeError, match=word):
            c.call(c_ext.quantize_kv_blocks, gids, mids)
    c.call(c_ext.quantize_kv_blocks, [], [])
    assert torch.equal(c.mx.cpu(), c.before)
    kept, c.mx = c.mx, torch.zeros(4, 4).to_sparse()         # torch's own errors come through
    with pytest.raises((RuntimeError, NotImplementedError)):
        c.call(c_ext.quantize_kv_blocks, [0], [0])
    assert torch.equal(kept.cpu(), c.before)


def test_blocks_are_refused_under_capture():
    c = Blocks(L=1, T=16, H=1, D=64, dtype=BF16)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="capture"):
            c.call(c_ext.quantize_kv_blocks, [0], [0])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.mx.cpu(), c.before)


def test_four_bit_blocks_move_to_the_host_and_back_as_blocks():
    """The 4-bit cache is a cache to the transfer: quantise, D2H, H2D into other
    blocks, read back."""
    L, T, H, D, N = 2, 16, 2, 128, 6
    c = Blocks(L=L, T=T, H=H, D=D, dtype=BF16, kind="LAYERWISE", n_mx=N)
    gids, mids = [0, 3, 5], [1, 4, 2]
    c.call(c_ext.quantize_kv_blocks, gids, mids)
    host_lay = KVCacheLayout(KVCacheLayoutType.BLOCKWISE, L, 4, T, H, D).mx4()
    chunk, hkv, hlay, hblk = host_lay.byte_strides(torch.uint8)
    host = pinned_empty(host_lay.get_total_elements(), torch.uint8)
    ptrs = torch.tensor([c.mx.data_ptr() + l * c.mlay for l in range(L)])
    cids = torch.tensor([3, 0, 1])
    c_ext.transfer_kv_blocks(torch.tensor(mids), ptrs, c.mkv, c.mblk, cids, host, hkv, hlay, hblk,
                             chunk, 0, -1, False)
    back = torch.tensor([0, 3, 5])
    c_ext.transfer_kv_blocks(back, ptrs, c.mkv, c.mblk, cids, host, hkv, hlay, hblk, chunk, 0, -1,
                             True)
    for t in c.wide:
        t.zero_()
    c.call(c_ext.dequantize_kv_blocks, gids, back.tolist())
    for l in range(L):
        for gid in gids:
            x = c.wide_host[l][:, gid].double().numpy()
            assert _same(c.wide[l][:, gid].cpu(), mo.as_type(mo.decode(*mo.encode(x)), BF16))


# -- tokens --------------------------------------------------------------------------

@pytest.mark.parametrize("T,H,D,dtype,halves,n,slot_type,blockwise", [
    (16, 8, 128, BF16, 2, 1, torch.int64, False),
    (16, 2, 64, FP16, 2, 37, torch.int32, True),
    (32, 1, 576, BF16, 1, 50, torch.int64, False),
    (48, 3, 256, FP32, 2, 5, torch.int64, True),
    (16, 1, 32, FP16, 2, 0, torch.int64, False),
])
def test_tokens_reach_their_slots_and_nothing_else(T, H, D, dtype, halves, n, slot_type,
                                                   blockwise):
    g = _gen(n)
    blocks = 5
    chunk = c_ext.mx4_chunk_bytes(T, H, D)
    mx = torch.randint(0, 256, (blocks, halves, chunk), generator=g, dtype=torch.uint8)
    if not blockwise:
        mx = mx.transpose(0, 1).contiguous().transpose(0, 1)
    want = mx.clone().numpy()
    wide = _hard_rows((n, 3 * H, D), dtype, g) if n else torch.zeros(0, 3 * H, D, dtype=dtype)
    dev = wide.to(DEV)
    key, value = dev[:, H:2 * H], dev[:, 2 * H:] if halves == 2 else None
    slots = torch.randperm(blocks * T, generator=g)[:n].to(slot_type)
    if n > 4:                                # padding
        slots[1], slots[3] = -1, blocks * T
    dmx = mx.to(DEV)
    if not blockwise:
        dmx = dmx.transpose(0, 1).contiguous().transpose(0, 1)
    c_ext.quantize_kv_tokens(key, value, dmx.transpose(0, 1), slots.to(DEV))
    for i in range(n):
        s = int(slots[i])
        if not 0 <= s < blocks * T:
            continue
        for k in range(halves):
            codes, scales = mo.unpack_chunk(want[s // T, k], T, H, D)
            codes, scales = codes.copy(), scales.copy()
            codes[s % T], scales[s % T] = mo.encode(
                wide[i, (k + 1) * H:(k + 2) * H].double().numpy())
            want[s // T, k] = mo.pack_chunk(codes, scales)
    assert torch.equal(dmx.cpu(), torch.from_numpy(want))


def test_token_calls_refuse_what_they_cannot_take():
    x = torch.zeros(3, 2, 64, device=DEV, dtype=BF16)
    mx = torch.zeros(2, 4, c_ext.mx4_chunk_bytes(16, 2, 64), device=DEV, dtype=torch.uint8)
    slots = torch.arange(3, device=DEV)
    call = c_ext.quantize_kv_tokens
    call(x, x, mx, slots)
    for args in ((x.transpose(1, 2), x, mx, slots), (x, x[:2], mx, slots), (x, x.half(), mx, slots),
                 (x, None, mx, slots), (x, x, mx[0], slots), (x, x, mx.view(torch.int8), slots),
                 (x, x, mx[..., :-16], slots), (x, x, mx, slots.float()), (x, x, mx, slots[:2]),
                 (x, x, mx, torch.arange(6, device=DEV)[::2]), (x[:, :, :48], x[:, :, :48], mx,
                                                                slots)):
        with pytest.raises(ValueError):
            call(*args)
    with pytest.raises(TypeError):
        call(x.to(torch.int16), x.to(torch.int16), mx, slots)
    with pytest.raises(ValueError):
        call(x.to_sparse(), x, mx, slots)
    with pytest.raises(RuntimeError, match="device tensor"):
        call(x, x, mx, slots.cpu())
    odd = torch.zeros(3 * 2 * 64 + 1, device=DEV, dtype=BF16)[1:].view(3, 2, 64)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        call(odd, x, mx, slots)
    chunk = mx.shape[2]
    assert _lib.load().fkv_quantize_kv_tokens(
        3, x.data_ptr(), 256, 128, x.data_ptr(), 256, 128, slots.data_ptr(), 1, mx.data_ptr(),
        4 * chunk, chunk, 1 << 30, 16, 2, 64, _lib.FKV_DTYPE_BF16, None) == 1
    assert "allocation" in _lib.last_error()


# -- attention -----------------------------------------------------------------------

class Case:
    """Sequences of `keys` keys whose last `queries` tokens ask."""

    def __init__(self, keys, queries, H=2, G=4, D=128, T=16, dtype=BF16, index=torch.int32,
                 blockwise=False, spread=1.0, seed=0, spare_rows=0, width=0):
        self.keys, self.queries, self.spare = keys, queries, spare_rows
        self.H, self.G, self.D, self.T, self.dtype = H, G, D, T, dtype
        g = _gen(seed)
        pages = [-(-k // T) for k in keys]
        self.N = sum(pages) + 2
        chunk = c_ext.mx4_chunk_bytes(T, H, D)
        codes = torch.randint(0, 256, (2, self.N, chunk), generator=g, dtype=torch.uint8)
        cut = T * H * D // 2
        codes[..., cut:] = torch.randint(124, 128, codes[..., cut:].shape, generator=g,
                                         dtype=torch.uint8)
        self.mx = codes
        perm = torch.randperm(self.N, generator=g).tolist()
        self.table = torch.zeros(len(keys), max([width, 1, *pages]), dtype=index)
        for b, p in enumerate(pages):
            self.table[b, :p] = torch.tensor([perm.pop() for _ in range(p)], dtype=index)
        self.lens = torch.tensor(keys, dtype=index)
        self.rows = sum(queries) + spare_rows
        self.starts = torch.tensor([0, *np.cumsum(queries)], dtype=index)
        self.qkv = (torch.randn(self.rows, H * (G + 2), D, generator=g) * spread).to(dtype)
        self.blockwise = blockwise

    def poison_unseen(self):
        """NaN and infinite bytes wherever no sequence has a token."""
        T, cut = self.T, self.T * self.H * self.D // 2
        seen = torch.zeros(self.N, T, dtype=torch.bool)
        for b, k in enumerate(self.keys):
            for t in range(k):
                seen[self.table[b, t // T], t % T] = True
        sc = self.mx[..., cut:].view(2, self.N, -1, T)
        sc[:] = torch.where(seen[None, :, None], sc, torch.tensor(255, dtype=torch.uint8))

    def to_device(self):
        self.dmx = self.mx.to(DEV)
        if self.blockwise:
            self.dmx = self.dmx.transpose(0, 1).contiguous().transpose(0, 1)
        self.dq = self.qkv.to(DEV)[:, :self.H * self.G]
        self.dtable, self.dlens = self.table.to(DEV), self.lens.to(DEV)
        self.dstarts = self.starts.to(DEV)

    def run(self, causal=True, scale=None, single=False, lse=True, **kw):
        self.to_device()
        lse = torch.full((self.rows, self.H * self.G), 77.0, device=DEV) if lse else None
        out = c_ext.mx4_attention(self.dq, self.dmx, self.H, self.dtable, self.dlens,
                                  None if single else self.dstarts, scale, causal, lse=lse, **kw)
        return out.cpu(), lse.cpu() if lse is not None else None

    def check(self, out, lse, causal=True, scale=None):
        scale = self.D ** -0.5 if scale is None else scale
        at = 0
        for b, (k, n) in enumerate(zip(self.keys, self.queries)):
            pages = self.table[b, :-(-k // self.T)].long()
            kv = np.stack([[mo.chunk_values(self.mx[h, p].numpy(), self.T, self.H, self.D)
                            for p in pages] for h in (0, 1)]) if k else \
                np.zeros((2, 0, self.T, self.H, self.D))
            kv = torch.from_numpy(kv.reshape(2, -1, self.H, self.D)[:, :k])
            vis = [max(0, k - n + i + 1) if causal else k for i in range(n) for _ in range(self.G)]
            for h in range(self.H):
                rows = slice(h * self.G, (h + 1) * self.G)
                q = self.qkv[at:at + n, rows].reshape(-1, self.D)
                o, l, big, mags = mo.attention(q, kv[0, :, h], kv[1, :, h], scale, vis)
                vmax = float(kv[1].nan_to_num().abs().max()) if k else 0.0
                tol = mo.tolerance(o, big, mags, k, self.dtype, vmax)
                got = out[at:at + n, rows].reshape(-1, self.D).double()
                assert torch.equal(torch.isnan(got), torch.isnan(o)), (b, h)
                err = (got - o).abs()
                ok = (err <= tol) | torch.isnan(o)
                assert ok.all(), (b, h, float((err / tol).nan_to_num().max()))
                if lse is not None:
                    gl = lse[at:at + n, rows].reshape(-1).double()
                    none = torch.isinf(l)
                    assert torch.equal(gl[none], l[none])
                    slack = mags * 2.0 ** -14 + k * 2.0 ** -23 + 2.0 ** -18 * (1 + l.abs())
                    assert ((gl - l).abs() <= slack)[~none & ~torch.isnan(l)].all()
            at += n


DECODE = [
    dict(keys=[1], H=1, G=1),
    dict(keys=[0, 1, 15, 16, 17, 31, 32, 33, 48, 63], H=2, G=4),
    dict(keys=[257, 5, 640], H=1, G=8, D=64, T=32),
    dict(keys=[130, 77], H=2, G=3, D=256, dtype=FP16, T=48),
    dict(keys=[300, 1000, 20], H=1, G=16, D=64, dtype=FP16, index=torch.int64),
    dict(keys=[200, 513], H=1, G=20, D=128, blockwise=True),
    dict(keys=[90, 33], H=8, G=1, D=128, dtype=FP16, T=64),
    dict(keys=[3000, 2050, 1], H=2, G=5, D=128, width=400),
    dict(keys=[5000, 7777, 1, 0], H=2, G=5, D=128, width=600),
    dict(keys=[9000, 40], H=1, G=33, D=256, T=32, dtype=FP16),
    # groups of more rows than a row tile, over several row tiles
    dict(keys=[33, 0, 70], H=64, G=40, D=64),
    dict(keys=[20, 37], H=96, G=90, D=128),
]


@pytest.mark.parametrize("kw", DECODE, ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_one_query_a_sequence(kw):
    c = Case(queries=[1] * len(kw["keys"]), seed=len(kw["keys"]), **kw)
    c.poison_unseen()
    c.check(*c.run(single=True))
    c.check(*c.run(single=False))


PACKED = [
    dict(keys=[5, 40, 0, 100, 16], queries=[5, 3, 0, 1, 16]),
    dict(keys=[64, 700], queries=[64, 33], H=1, G=8, D=64, T=32),
    dict(keys=[129, 33, 1], queries=[129, 2, 1], H=2, G=1, D=128, dtype=FP16),
    dict(keys=[70, 200], queries=[40, 17], H=1, G=5, D=256, index=torch.int64),
    dict(keys=[10, 3], queries=[13, 5], H=2, G=2, D=64),             # queries before any key
    dict(keys=[900, 333, 80], queries=[150, 90, 80], H=2, G=4, D=128, T=16, blockwise=True),
    dict(keys=[500, 12, 260, 31], queries=[1, 12, 100, 1], H=1, G=16, D=128, dtype=FP16, T=48),
]


@pytest.mark.parametrize("kw", DECODE, ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_nothing_beside_the_rows_of_single_queries_is_written(kw):
    """Whatever the number of sequences and heads, rows before and behind stay."""
    c = Case(queries=[1] * len(kw["keys"]), seed=len(kw["keys"]), **kw)
    c.to_device()
    want, lse = c.run(single=True)
    big = torch.full((c.rows + 80, c.H * c.G, c.D), 5.0, dtype=c.dtype, device=DEV)
    bl = torch.full((c.rows + 80, c.H * c.G), 77.0, device=DEV)
    at = slice(40, 40 + c.rows)
    c_ext.mx4_attention(c.dq, c.dmx, c.H, c.dtable, c.dlens, None, out=big[at], lse=bl[at])
    assert torch.equal(big[at].cpu(), want) and torch.equal(bl[at].cpu(), lse)
    big[at], bl[at] = 5, 77
    assert (big == 5).all() and (bl == 77).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kw", PACKED, ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_packed_queries(kw, causal):
    c = Case(seed=7, spare_rows=3, **kw)
    c.poison_unseen()
    out = torch.full((c.rows, c.H * c.G, c.D), 5.0, dtype=c.dtype, device=DEV)
    got, lse = c.run(causal=causal, out=out)
    c.check(got, lse, causal=causal)
    # rows of no sequence are left as they were
    assert (got[-3:] == 5).all() and (lse[-3:] == 77).all()


# many heads and rows: several row tiles share a workgroup
MANY_ROWS = [
    dict(keys=[40, 0, 100, 133, 20], queries=[23, 0, 1, 90, 20], H=32, G=4, D=128),
    dict(keys=[300, 45], queries=[61, 45], H=64, G=3, D=64, T=32, dtype=FP16),
    dict(keys=[97, 12, 65], queries=[97, 17, 40], H=32, G=4, D=128, dtype=FP16, blockwise=True),
    dict(keys=[150, 31], queries=[50, 31], H=48, G=2, D=256, T=48),
    dict(keys=[71, 64], queries=[71, 50], H=32, G=3, D=256, dtype=FP16, index=torch.int64),
    # two row tiles where three would leave compute units empty
    dict(keys=[60, 0, 133], queries=[40, 0, 20], H=32, G=4, D=128),
    dict(keys=[90, 45], queries=[50, 14], H=48, G=3, D=64, dtype=FP16, T=48),
    dict(keys=[300, 31, 9], queries=[31, 31, 12], H=32, G=4, D=128, dtype=FP16, blockwise=True),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kw", MANY_ROWS, ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_packed_queries_of_many_heads(kw, causal):
    c = Case(seed=17, spare_rows=2, **kw)
    c.poison_unseen()
    out = torch.full((c.rows, c.H * c.G, c.D), 5.0, dtype=c.dtype, device=DEV)
    got, lse = c.run(causal=causal, out=out)
    c.check(got, lse, causal=causal)
    assert (got[-2:] == 5).all() and (lse[-2:] == 77).all()


@pytest.mark.parametrize("D,dtype", [(64, FP16), (128, BF16), (256, BF16)])
def test_many_heads_nan_growing_scores_and_bad_pages(D, dtype):
    c = Case(keys=[120, 90, 80], queries=[80, 90, 60], H=32, G=4, D=D, dtype=dtype, seed=23)
    cut = c.T * c.H * D // 2
    for half, b, t, head, group in ((0, 0, 60, 0, 1), (1, 0, 75, 31, 0), (1, 1, 0, 7, 1),
                                    (1, 1, 89, 8, 0), (0, 1, 88, 9, 0)):
        sc = c.mx[half, c.table[b, t // c.T], cut:].view(c.H, D // 32, c.T)
        sc[head, group, t % c.T] = 255
    # keys that grow by 2^12 along a sequence: the running reference follows
    for t in range(80):
        sc = c.mx[0, c.table[2, t // c.T], cut:].view(c.H, D // 32, c.T)
        sc[:, :, t % c.T] = 120 + t * 12 // 80
    out, lse = c.run()
    c.check(out, lse)
    c.table[2, 2] = c.N
    bad, lse = c.run()
    # tokens 32 and on: query i of the sequence's 60 sees 21 + i
    assert torch.isnan(bad[182:]).all() and torch.isnan(lse[182:]).all()
    assert _same(bad[:182], out[:182])


@pytest.mark.parametrize("batch,H,D,dtype", [
    (3, 1, 64, BF16), (64, 1, 64, FP16), (65, 1, 128, BF16), (130, 2, 64, BF16),
    (40, 8, 64, FP16), (34, 8, 256, BF16), (70, 8, 64, BF16), (131, 8, 64, BF16)])
def test_cuts_of_ragged_lengths_and_of_many_sequences(batch, H, D, dtype):
    """Long sequences beside short ones, above and below the numbers of sequences and of
    tiles that plan the cuts differently."""
    g = _gen(batch)
    keys = torch.randint(0, 40, (batch,), generator=g).tolist()
    keys[1], keys[2], keys[-1] = 4900, 1500, 6100
    c = Case(keys=keys, queries=[1] * batch, H=H, G=3, D=D, T=32, dtype=dtype, seed=batch)
    c.poison_unseen()
    c.check(*c.run(single=True))
    c.check(*c.run(single=False))


@pytest.mark.parametrize("byte,lost", [(252, False), (253, True), (254, True), (255, True)])
def test_value_scales_that_quantising_never_writes_count_as_nan(byte, lost):
    for keys, queries, H in (([70], [3], 2), ([70, 33], [70, 33], 64)):
        c = Case(keys=keys, queries=queries, H=H, G=4, D=128, seed=byte)
        cut = c.T * H * c.D // 2
        c.mx[1, c.table[0, 1], cut:].view(H, c.D // 32, c.T)[1, 2, 5] = byte
        out, _ = c.run()
        rows = queries[0]
        hit = torch.zeros(c.rows, H, c.G, c.D, dtype=torch.bool)
        first = max(0, 21 - (keys[0] - rows))           # the first query that sees token 21
        hit[first:rows, 1, :, 64:96] = lost
        assert torch.equal(torch.isnan(out.view_as(hit)), hit)


@pytest.mark.parametrize("keys,queries,H,width", [([1, 40], [1, 1], 2, 0),
                                                   ([50, 33], [50, 20], 32, 0),
                                                   ([7000, 9], [1, 1], 1, 500)])
def test_values_past_fp16_come_out_as_its_largest(keys, queries, H, width):
    """Values of 65504 are held as 65536: finite when read back, and here."""
    c = Case(keys=keys, queries=queries, H=H, G=4, D=64, dtype=FP16, seed=47, width=width)
    c.to_device()
    n = c.N * c.T
    x = torch.full((n, H, c.D), 65504.0, dtype=FP16)
    x[:, :, 1::2] = -65504.0
    x[:, :, 32:] = 3.0
    c_ext.quantize_kv_tokens(c.qkv.to(DEV)[:1, :H].expand(n, H, c.D).contiguous(), x.to(DEV), c.dmx,
                             torch.arange(n, device=DEV))
    c.mx = c.dmx.cpu()
    out, _ = c.run()
    # weights that sum to one within their rounding, so 65504 but for it or from beyond
    assert torch.isfinite(out).all()
    assert ((out[..., 0:32:2] - 65504).abs() <= 64).all()
    assert ((out[..., 1:32:2] + 65504).abs() <= 64).all()
    assert ((out[..., 32:].float() - 3).abs() <= 2.0 ** -8).all()


@pytest.mark.parametrize("flat", [False, True])
@pytest.mark.parametrize("kw", [
    dict(keys=[70, 33], queries=[3, 1], H=2, G=4, D=128),
    dict(keys=[1400], queries=[1], H=1, G=8, D=64),
    dict(keys=[200, 150], queries=[90, 150], H=32, G=4, D=128),
    dict(keys=[120], queries=[120], H=48, G=2, D=256),
    dict(keys=[9000, 30], queries=[1, 1], H=1, G=4, D=128, width=600)],
    ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_large_values_do_not_overflow_the_sums(kw, flat):
    """Values up to 2^119 over the keys, beside ordinary ones."""
    c = Case(seed=53, **kw)
    cut = c.T * c.H * c.D // 2
    sc = c.mx[1, :, cut:].view(c.N, c.H, c.D // 32, c.T)
    byte = 127 + 119 - 3 - math.ceil(math.log2(max(c.keys)))       # 6 is below 2^3
    sc[:, -1, 1] = byte
    sc[:, 0, 0, 3::5] = byte
    # keys that grow, so that scores pass the first ones by a little again and again
    if not flat:
        for b, k in enumerate(c.keys):
            for t in range(k):
                ks = c.mx[0, c.table[b, t // c.T], cut:].view(c.H, c.D // 32, c.T)
                ks[:, :, t % c.T] = 122 + t * 5 // k
    scale = 0.0 if flat else None
    out, lse = c.run(scale=scale)
    assert torch.isfinite(out).all()
    c.check(out, lse, scale=scale)


def test_a_large_value_of_small_weight_counts():
    """A weight of 2^-104 and a value of 2^103 and more beside one of weight 1, in one step, in
    another and in another workgroup's: the row's result is made of it."""
    for keys, far, width in ((30, 7, 0), (1000, 900, 0), (9000, 8000, 600)):
        c = Case(keys=[keys], queries=[1], H=1, G=2, D=128, seed=57, width=width)
        cut = c.T * c.D // 2
        c.mx[0, :, :cut] = 0
        c.mx[1, :, :cut] = 0x22                      # 1
        c.mx[:, :, cut:] = 127
        c.qkv[:] = 0
        c.qkv[:, :2, 0] = 104.0
        for t, code in ((3, 2), (far, 10)):          # scores of 104 and -104, the others 0
            c.mx[0, c.table[0, t // c.T], (t % c.T) * c.D // 2] = code
        page = c.mx[1, c.table[0, far // c.T]]
        page[cut:].view(c.D // 32, c.T)[2, far % c.T] = 127 + 103
        scale = math.log(2) / 2                      # weights 1, 2^-52 and 2^-104
        out, lse = c.run(single=True, scale=scale)
        c.check(out, lse, scale=scale)
        # 2^103 2^-104, and of the others 1
        assert ((out[0, :, 64:96] - 1.5).abs() <= 2.0 ** -6).all()
        assert ((out[0, :, :64] - 1).abs() <= 2.0 ** -6).all()


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, FP16), (256, BF16)])
def test_the_largest_value_of_a_single_key(dim, dtype):
    """Scale byte 252, the last that is no NaN: the value itself, or fp16's largest."""
    c = Case(keys=[1], queries=[1], H=2, G=2, D=dim, dtype=dtype, seed=59)
    cut = c.T * c.H * dim // 2
    c.mx[1, :, cut:] = 252
    out, lse = c.run()
    v = mo.chunk_values(c.mx[1, c.table[0, 0]].numpy(), c.T, c.H, dim)[0]
    want = mo.as_type(v, dtype).repeat_interleave(c.G, 0)
    assert torch.equal(out[0], want)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (-0.3, 1.0), (1.0, 4.0), (1e-3, 300.0)])
def test_scales_flat_sharp_and_negative(dtype, scale, spread):
    c = Case(keys=[333, 60], queries=[2, 60], G=4, dtype=dtype, spread=spread, seed=3)
    c.check(*c.run(scale=scale), scale=scale)


FORMS = [dict(keys=[1400], queries=[1], H=1, G=8, D=128),            # a wide workgroup
         dict(keys=[600, 500], queries=[300, 400], H=16, G=4, D=64),   # several row tiles
         dict(keys=[400], queries=[200], H=48, G=2, D=256),
         dict(keys=[9000, 30], queries=[1, 1], H=1, G=4, D=128, width=600),   # cut keys
         dict(keys=[7000], queries=[40], H=2, G=4, D=64, dtype=FP16, T=32, width=256)]


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("log2", [20, 27, 30, 32, 34, 60, 100])
@pytest.mark.parametrize("kw", FORMS, ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_scores_of_any_size_pick_the_largest(kw, log2, sign):
    """Scores near 2^log2: of two equal keys the largest by half, the others without weight.
    Equal scores have equal weights, so the result is the two values' mean, within the
    rounding of the weights and its own."""
    c = Case(seed=43, **kw)
    g = _gen(44)
    T, H, D = c.T, c.H, c.D
    direction = torch.randn(D, generator=g).clamp(-4, 4)
    direction[direction.abs() < 2.0 ** -6] = 2.0 ** -6
    factor = 1 + torch.rand(c.rows, H * c.G, 1, generator=g)
    q = (direction * factor).to(c.dtype)
    c.qkv[:, :H * c.G] = q
    side = (sign * direction < 0).to(torch.uint8) * 8       # codes that agree in sign
    cut = T * H * D // 2
    top = {}
    for b, k in enumerate(c.keys):
        # the smallest scores are -3 or less where they are negative, the largest -0.5
        first = max(1, k - c.queries[b])                     # all rows see tokens before it
        top[b] = sorted({0, first // 2, first - 1})[-2:]
        for t in range(k):
            mag = torch.randint(0, 6, (H, D), generator=g, dtype=torch.uint8)
            if sign < 0:
                mag = mag % 3 + 5
            if t in top[b]:
                mag[:] = 7 if sign > 0 else 1
            codes = mag | side
            page = c.mx[0, c.table[b, t // T]]
            page[:cut].view(H, T, D // 2)[:, t % T] = codes[:, 0::2] | codes[:, 1::2] << 4
            page[cut:].view(H, D // 32, T)[:, :, t % T] = 127
    scale = 0.7 * 2.0 ** log2 / float(direction.abs().sum())
    out, lse = c.run(scale=scale)
    at = 0
    for b, (k, n) in enumerate(zip(c.keys, c.queries)):
        pages = c.table[b, :-(-k // T)].long()
        v = np.stack([mo.chunk_values(c.mx[1, p].numpy(), T, H, D) for p in pages])
        v = torch.from_numpy(v.reshape(-1, H, D))[top[b]]
        want = v.mean(0).repeat_interleave(c.G, 0)
        half = torch.finfo(c.dtype).eps / 2
        p = 2.0 ** -8 if c.dtype == BF16 else 2.0 ** -16
        tol = (p + 2.0 ** -18) * v.abs().mean(0).repeat_interleave(c.G, 0) * (1 + half) + \
            half * want.abs() + torch.finfo(c.dtype).smallest_normal
        assert ((out[at:at + n].double() - want).abs() <= tol).all(), b
        s = (q[at:at + n].double() * direction.sign() * (6 if sign > 0 else -0.5)).sum(-1) * scale
        assert ((lse[at:at + n].double() - s).abs() <= s.abs() * 2.0 ** -14 + 1).all()
        at += n


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("kw", FORMS, ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_scores_past_32_bits_make_their_rows_nan(kw, sign):
    """q . k of 2^131 and more, all of one sign, for one query and head."""
    c = Case(seed=45, **{**kw, "dtype": BF16})
    want, lse = c.run()
    cut = c.T * c.H * c.D // 2
    c.mx[0, :, :cut] = 0x66                      # 4, with scales from 2^-3 on
    c.qkv[0, 1] = sign * 2.0 ** 124              # 64 products and more of 2^125
    out, got = c.run()
    assert torch.isnan(out[0, 1]).all() and torch.isnan(got[0, 1])
    assert torch.isnan(out).sum() == c.D and torch.isnan(got).sum() == 1


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale", [0.0, 1e-33, -1e-33, 1e-40])
def test_scales_of_zero_and_near_it_beside_large_products(scale, dtype):
    c = Case(keys=[333, 60], queries=[2, 60], G=4, dtype=dtype, seed=3)
    cut = c.T * c.H * c.D // 2
    up = 50 if dtype == BF16 else 0
    c.mx[0, :, cut:] += 106 - up                 # keys of 2^(103 - up) .. 2^(106 - up)
    c.qkv = (c.qkv.float() * 2.0 ** up).to(dtype)
    c.check(*c.run(scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("apart", [0, 6, 10, 13])
def test_scores_of_rows_of_uneven_elements(D, dtype, apart):
    """The score of a single key, its lse, within what the header says: of the products of
    eight neighbours, the bits under 2^-13 of the largest are cut, for each part of the
    query, a part being 2^-4 of the one before."""
    B = 300
    c = Case(keys=[1] * B, queries=[1] * B, H=2, G=4, D=D, dtype=dtype, seed=60 + apart)
    g = _gen(61)
    c.qkv = (c.qkv.float() * torch.exp2(-torch.randint(0, apart + 1, c.qkv.shape,
                                                       generator=g).float())).to(dtype)
    scale = D ** -0.5
    _, lse = c.run(single=True, scale=scale)
    page = c.table[:, 0].long()
    k = torch.from_numpy(np.stack([mo.chunk_values(c.mx[0, p].numpy(), c.T, c.H, D)[0]
                                   for p in page])).repeat_interleave(c.G, 1)
    q = c.qkv[:, :c.H * c.G].double()
    s, mags = (q * k).sum(-1) * scale, (q * k).abs().sum(-1) * scale
    cut = (q * k).abs().unflatten(-1, (-1, 8)).amax(-1).sum(-1) * scale * 7 * 2.0 ** -13
    parts = q.abs().amax(-1) * k.abs().sum(-1) * scale * 2.0 ** -21
    # sums and the step from log2 to log in 32 bits, exp and log of one weight
    rest = mags * 2.0 ** -20 + 2.0 ** -20
    assert ((lse.double() - s).abs() <= cut * (1 + 2.0 ** -4 + 2.0 ** -8) + parts + rest).all()


def test_extreme_scales_and_queries_stay_in_range():
    """Keys and values near the ends of what the format holds, queries whose
    elements span 2^-30 .. 2^7."""
    c = Case(keys=[100], queries=[3], H=1, G=2, D=128, seed=9)
    cut = c.T * c.H * c.D // 2
    c.mx[0, :, cut:] = torch.randint(60, 100, c.mx[0, :, cut:].shape, dtype=torch.uint8)
    c.mx[1, :, cut:] = torch.randint(0, 12, c.mx[1, :, cut:].shape, dtype=torch.uint8)
    c.qkv = (c.qkv.float() * torch.exp2(torch.randint(-30, 7, c.qkv.shape).float())).to(BF16)
    c.check(*c.run(scale=2.0 ** 20), scale=2.0 ** 20)


def test_nan_reaches_the_rows_that_see_it_and_no_other():
    """A NaN key or value token within the causal corner: rows before it are as
    without it, rows from it on are NaN where a 64-bit softmax has NaN."""
    for half, T in ((0, 16), (1, 16), (1, 32)):
        c = Case(keys=[200, 90], queries=[60, 90], H=2, G=3, D=128, T=T, seed=21)
        cut = c.T * c.H * c.D // 2
        for b, t, head, group in ((0, 155, 0, 1), (0, 170, 1, 3), (1, 0, 1, 0), (1, 33, 0, 2)):
            sc = c.mx[half, c.table[b, t // T], cut:].view(c.H, c.D // 32, T)
            sc[head, group, t % T] = 255
        out, lse = c.run()
        c.check(out, lse)
        assert torch.isnan(out).any() and not torch.isnan(out[:15, :3]).any()


def test_nan_and_infinite_queries_stay_in_their_row():
    c = Case(keys=[50, 20], queries=[4, 20], seed=2)
    for r, h, v in ((1, 3, float("nan")), (10, 0, float("inf")), (11, 7, -float("inf"))):
        c.qkv[r, h, 5] = v
    out, _ = c.run()
    rows = torch.isnan(out).all(-1)
    assert torch.equal(torch.isnan(out).any(-1), rows)
    assert sorted(map(tuple, rows.nonzero().tolist())) == [(1, 3), (10, 0), (11, 7)]
    c.qkv.nan_to_num_(0.25, 0.25, 0.25)
    keep = ~rows
    clean, _ = c.run()
    assert torch.equal(out[keep], clean[keep])


def test_bad_pages_and_lengths_make_their_rows_nan():
    for index in (torch.int32, torch.int64):
        c = Case(keys=[100, 60, 200, 40], queries=[2, 3, 1, 40], seed=4, index=index)
        good, _ = c.run()
        c.table[0, 3] = c.N                # one past the cache
        c.table[2, 0] = -1
        bad, lse = c.run()
        hit = torch.tensor([True] * 2 + [False] * 3 + [True] + [False] * 40)
        assert torch.isnan(bad[hit]).all() and torch.isnan(lse[hit]).all()
        assert torch.equal(bad[~hit], good[~hit])
        c.table[0, 3], c.table[2, 0] = 0, 0
        c.lens[1] = c.table.shape[1] * c.T + 1
        long, _ = c.run()
        assert torch.isnan(long[2:5]).all() and not torch.isnan(long[5:]).any()
        c.lens[1] = -5                     # as no keys
        none, lse = c.run()
        assert (none[2:5] == 0).all() and torch.isinf(lse[2:5]).all()


# one row tile, several, and cut keys: rows that see no key share a tile with rows that do
KEYLESS = [dict(keys=[10], queries=[13]),
           dict(keys=[40, 3], queries=[60, 40], H=32, G=4, D=64, dtype=FP16),
           dict(keys=[7], queries=[30], H=64, G=4),
           dict(keys=[20, 7000], queries=[25, 9], H=1, G=2, T=32, width=256)]


@pytest.mark.parametrize("bad", [-1, "past"])
@pytest.mark.parametrize("kw", KEYLESS, ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_rows_without_keys_stay_zero_beside_a_bad_first_page(kw, bad):
    c = Case(seed=41, **kw)
    good, gl = c.run()
    c.check(good, gl)
    c.table[0, 0] = c.N if bad == "past" else bad
    out, lse = c.run()
    n, k = c.queries[0], c.keys[0]
    assert (out[:n - k] == 0).all() and (lse[:n - k] == -math.inf).all()
    assert torch.isnan(out[n - k:n]).all() and torch.isnan(lse[n - k:n]).all()
    assert torch.equal(out[n:], good[n:]) and torch.equal(lse[n:], gl[n:])


@pytest.mark.parametrize("keys,queries,H,width", [
    ([100, 0, 31, 333], [1, 1, 1, 1], 2, 40), ([100, 0, 31, 6000], [1, 0, 9, 3], 2, 512),
    ([100, 0, 31, 333], [60, 0, 31, 90], 32, 40)])
def test_table_entries_without_keys_are_not_looked_at(keys, queries, H, width):
    c = Case(keys=keys, queries=queries, H=H, seed=14, width=width)
    single = queries == [1] * len(queries)
    want, _ = c.run(single=single)
    for fill in (-1, c.N, 2 ** 31 - 1):
        for b, k in enumerate(keys):
            c.table[b, -(-k // c.T):] = fill
        got, _ = c.run(single=single)
        assert torch.equal(got, want)


def test_strides_of_out_and_lse():
    c = Case(keys=[77, 30], queries=[7, 9], G=2, seed=5)
    want, lse = c.run()
    c.to_device()
    wide = torch.full((c.rows, 3, c.H * c.G, c.D), 9.0, dtype=c.dtype, device=DEV)
    lt = torch.zeros(c.H * c.G, c.rows, device=DEV)
    got = c_ext.mx4_attention(c.dq, c.dmx, c.H, c.dtable, c.dlens, c.dstarts, out=wide[:, 1],
                              lse=lt.t())
    assert got.data_ptr() == wide[:, 1].data_ptr()
    assert torch.equal(wide[:, 1].cpu(), want) and torch.equal(lt.t().cpu(), lse)
    assert (wide[:, 0] == 9).all() and (wide[:, 2] == 9).all()


@pytest.mark.parametrize("D,dtype,T", [(64, FP16, 32), (128, BF16, 16), (256, BF16, 64)])
def test_many_rows_over_long_tables_are_cut(D, dtype, T):
    """Tiles of several row tiles, too few for the device, whose keys are cut: among
    rows of one tile some see keys of few cuts."""
    c = Case(keys=[7000, 90, 5100], queries=[40, 30, 17], H=2, G=4, D=D, T=T, dtype=dtype, seed=33,
             width=8192 // T)
    c.poison_unseen()
    cut = c.T * c.H * D // 2
    sc = c.mx[1, c.table[0, 6980 // T], cut:].view(c.H, D // 32, T)
    sc[1, 1, 6980 % T] = 255                 # seen by the later queries alone
    for causal in (True, False):
        out, lse = c.run(causal=causal)
        c.check(out, lse, causal=causal)
        again, _ = c.run(causal=causal)
        assert _same(out, again)
    assert torch.isnan(out[0, 4:]).any() and not torch.isnan(c.run()[0][19, 4:]).any()


def test_many_rows_of_many_sequences_over_long_tables():
    """More sequences than the plan ranks, their tiles of many rows cut."""
    g = _gen(70)
    keys = torch.randint(5, 60, (70,), generator=g).tolist()
    keys[3], keys[69] = 6000, 4500
    c = Case(keys=keys, queries=[9] * 70, H=1, G=4, D=64, T=32, seed=70, width=256)
    c.poison_unseen()
    c.check(*c.run())


def test_results_do_not_change_from_call_to_call():
    c = Case(keys=[6000, 4777, 64], queries=[1, 5, 64], H=2, G=4, seed=8)
    first = c.run()
    for _ in range(3):
        again = c.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("compiled", [True, False])
def test_inputs_that_require_gradients_are_refused_but_under_no_grad(compiled, monkeypatch):
    if not compiled:
        monkeypatch.setattr(c_ext, "_fast", _lib._CtypesCalls(_lib.load()))
    c = Case(keys=[40, 20], queries=[1, 1])
    want, _ = c.run()
    kv = c.qkv.to(DEV)
    key = kv[:, -2 * c.H:-c.H]
    slots = torch.full((2,), -1, device=DEV)
    with_grad = [t.clone().requires_grad_() for t in (c.dq, key)]
    out = torch.empty_like(c.dq).requires_grad_()
    for call in (lambda: c_ext.mx4_attention(with_grad[0], c.dmx, c.H, c.dtable, c.dlens),
                 lambda: c_ext.mx4_attention(c.dq, c.dmx, c.H, c.dtable, c.dlens, out=out),
                 lambda: c_ext.quantize_kv_tokens(with_grad[1], key, c.dmx, slots),
                 lambda: c_ext.quantize_kv_tokens(key, with_grad[1], c.dmx, slots)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    with torch.inference_mode():
        got = c_ext.mx4_attention(with_grad[0], c.dmx, c.H, c.dtable, c.dlens)
    assert torch.equal(got.cpu(), want) and not got.requires_grad


def test_out_that_overlaps_query_is_refused():
    c = Case(keys=[40, 20, 9], queries=[3, 2, 1])
    want, _ = c.run()
    n, HG, D = c.rows, c.H * c.G, c.D
    def call(q, out):
        return c_ext.mx4_attention(q, c.dmx, c.H, c.dtable, c.dlens, c.dstarts, out=out)
    both = torch.zeros(n + 2, 2 * HG, D, dtype=c.dtype, device=DEV)
    q = both[:n, :HG]
    q.copy_(c.dq)
    kept = both.clone()
    for out in (q, both[1:n + 1, :HG], both[:n, 1:HG + 1], both[2:, :HG],
                both.view(-1)[D // 2:D // 2 + 2 * n * HG * D].view(n, 2 * HG, D)[:, :HG]):
        with pytest.raises(ValueError, match="overlap"):
            call(q, out)
    assert torch.equal(both, kept)
    # beside it, in the same rows, or before or behind it
    assert torch.equal(call(q, both[:n, HG:]).cpu(), want)
    assert torch.equal(both[:n, HG:].cpu(), want) and torch.equal(both[:, :HG], kept[:, :HG])
    pairs = torch.zeros(n, HG, 2, D, dtype=c.dtype, device=DEV)
    pairs[:, :, 1] = c.dq
    assert torch.equal(call(pairs[:, :, 1], pairs[:, :, 0]).cpu(), want)


def test_attention_refuses_what_it_cannot_take():
    c = Case(keys=[40, 20], queries=[1, 1])
    c.to_device()
    q, mx, H, tab, lens, st = c.dq, c.dmx, c.H, c.dtable, c.dlens, c.dstarts
    call = c_ext.mx4_attention
    call(q, mx, H, tab, lens, st)
    for args in ((q.float(), mx, H, tab, lens, st), (q[0], mx, H, tab, lens, st),
                 (q.transpose(1, 2), mx, H, tab, lens, st), (q, mx, 3, tab, lens, st),
                 (q, mx, 0, tab, lens, st), (q, mx[:1], H, tab, lens, st),
                 (q, mx[..., :-16], H, tab, lens, st), (q, mx, H, tab.long(), lens, st),
                 (q, mx, H, tab, lens, st.long()), (q, mx, H, tab, lens.float(), st),
                 (q, mx, H, tab[:1], lens, st), (q, mx, H, tab, lens, st[:2]),
                 (q[:1], mx, H, tab, lens, None)):
        with pytest.raises(ValueError):
            call(*args)
    for kw in (dict(out=torch.empty_like(q).half()), dict(out=torch.empty_like(q[:1])),
               dict(lse=torch.empty(2, c.H * c.G, device=DEV, dtype=FP16)),
               dict(lse=torch.empty(2, 1, device=DEV))):
        with pytest.raises(ValueError):
            call(q, mx, H, tab, lens, st, **kw)
    with pytest.raises(RuntimeError, match="device tensor"):
        call(q, mx, H, tab.cpu(), lens, st)
    with pytest.raises(RuntimeError, match="scale"):
        call(q, mx, H, tab, lens, st, scale=math.inf)
    with pytest.raises(RuntimeError, match="head_size"):
        w = torch.zeros(2, 2, 96, device=DEV, dtype=BF16)
        call(w, torch.zeros(2, 4, c_ext.mx4_chunk_bytes(16, 2, 96), device=DEV,
                            dtype=torch.uint8), 2, tab, lens, st)
    assert call(q[:0], mx, H, tab[:0], lens[:0], None).shape == (0, c.H * c.G, c.D)


def test_long_cache_offsets_pass_32_bits():
    """Blocks beyond 4 GiB of the 4-bit cache, K and V apart by more."""
    T, H, D = 64, 8, 256
    chunk = c_ext.mx4_chunk_bytes(T, H, D)
    N = (5 << 30) // chunk
    mx = torch.empty(2, N, chunk, dtype=torch.uint8, device=DEV)
    c = Case(keys=[130], queries=[2], H=H, G=2, D=D, T=T)
    pages = [N - 1, 3, N - 7]
    mx[:, pages] = c.mx[:, c.table[0, :3].long()].to(DEV)
    c.to_device()
    want = c_ext.mx4_attention(c.dq, c.dmx, H, c.dtable, c.dlens, c.dstarts)
    table = torch.tensor([pages], dtype=torch.int32, device=DEV)
    got = c_ext.mx4_attention(c.dq, mx, H, table, c.dlens, c.dstarts)
    assert torch.equal(got, want)
    x = torch.randn(2, H, D, generator=_gen(1)).to(BF16)
    c_ext.quantize_kv_tokens(x.to(DEV), x.to(DEV), mx, torch.tensor([N * T - 1, 3 * T + 1],
                                                                    device=DEV))
    for i, (b, t) in enumerate(((N - 1, T - 1), (3, 1))):
        for k in (0, 1):
            v = mo.chunk_values(mx[k, b].cpu().numpy(), T, H, D)[t]
            assert np.array_equal(v, mo.decode(*mo.encode(x[i].double().numpy())))


# -- used together ---------------------------------------------------------------------

def _step(c, key, value, slots):
    c_ext.quantize_kv_tokens(key, value, c.dmx, slots)
    return c_ext.mx4_attention(c.dq, c.dmx, c.H, c.dtable, c.dlens, c.dstarts)


def test_prompt_then_steps_then_blocks_leave_and_return():
    """A prompt is written and attended over, then single tokens; its blocks go
    back to a 16-bit cache, are quantised again into another 4-bit cache, and
    attention over that is the same."""
    c = Case(keys=[75], queries=[75], H=2, G=4, D=128, seed=31, width=6)
    c.to_device()
    kv = c.qkv.to(DEV)
    T, H, G = c.T, c.H, c.G
    table = torch.tensor([[4, 1, 3, 0, 5, 2]], dtype=torch.int32, device=DEV)
    mx = torch.full((2, 6, c.mx.shape[2]), 255, dtype=torch.uint8, device=DEV)
    n, at = 0, []
    for new in (40, 1, 1, 33):
        rows = slice(n, n + new)
        pos = torch.arange(n, n + new, device=DEV)
        slots = table[0, pos // T].long() * T + pos % T
        c_ext.quantize_kv_tokens(kv[rows, H * G:H * G + H], kv[rows, H * G + H:], mx, slots)
        n += new
        starts = torch.tensor([0, new], dtype=torch.int32, device=DEV)
        lens = torch.tensor([n], dtype=torch.int32, device=DEV)
        at.append(c_ext.mx4_attention(kv[rows, :H * G], mx, H, table, lens, starts))
    c.mx, c.table = mx.cpu(), table.cpu()
    out = torch.cat(at).cpu()
    c.check(out, None)
    # the values are the quantised inputs
    used = [4, 1, 3, 0, 5]
    got = np.concatenate([mo.chunk_values(c.mx[1, p].numpy(), T, H, c.D) for p in used])[:75]
    want = mo.decode(*mo.encode(c.qkv[:, H * G + H:].double().numpy()))
    assert np.array_equal(got, want)
    wide = torch.zeros(2, 8, T, H, c.D, dtype=BF16, device=DEV)
    ptrs = torch.tensor([wide.data_ptr()])
    blk = T * H * c.D * 2
    chunk = mx.shape[2]
    gids = torch.tensor([7, 0, 2, 5, 3])
    c_ext.dequantize_kv_blocks(gids, ptrs, 8 * blk, blk, torch.tensor(used), mx, 6 * chunk, 0,
                               chunk, T, H, c.D, BF16)
    other = torch.zeros(2, 9, chunk, dtype=torch.uint8, device=DEV)
    c_ext.quantize_kv_blocks(gids, ptrs, 8 * blk, blk, torch.tensor([8, 6, 1, 0, 3]), other,
                             9 * chunk, 0, chunk, T, H, c.D, BF16)
    t2 = torch.tensor([[8, 6, 1, 0, 3, 0]], dtype=torch.int32, device=DEV)
    again = c_ext.mx4_attention(kv[42:75, :H * G], other, H, t2, lens, starts)
    assert torch.equal(again.cpu(), out[42:75])


def test_a_captured_step_replays_with_other_lengths_and_tokens():
    c = Case(keys=[6000, 33, 250], queries=[1, 2, 1], H=2, G=4, seed=12, width=512)
    c.to_device()
    kv = c.qkv.to(DEV)
    H, G, T = c.H, c.G, c.T
    key, value = kv[:, H * G:H * G + H].clone(), kv[:, H * G + H:].clone()
    slots = torch.full((4,), -1, dtype=torch.int64, device=DEV)
    fresh = c.dmx.clone()
    _step(c, key, value, slots)               # warm
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(c, key, value, slots)
    other = torch.cuda.CUDAGraph()            # a second graph over the same tensors
    with torch.cuda.graph(other):
        out2 = _step(c, key, value, slots)
    for i, keys in enumerate(([6000, 33, 250], [1, 2, 300], [8192, 512, 31], [0, 5024, 1])):
        c.dlens.copy_(torch.tensor(keys, dtype=torch.int32))
        c.dq.normal_()
        key.normal_()
        slots.copy_(torch.tensor([5 + i, -1, c.N * T - 1 - i, 64]))
        c.dmx.copy_(fresh)
        graph.replay()
        got, cache = out.clone(), c.dmx.clone()
        c.dmx.copy_(fresh)
        other.replay()
        got2 = out2.clone()
        c.dmx.copy_(fresh)
        torch.cuda.synchronize()
        want = _step(c, key, value, slots)
        assert torch.equal(got, want) and torch.equal(got2, want)
        assert torch.equal(cache, c.dmx)


def test_calls_over_ctypes_give_the_same(monkeypatch):
    def run():
        b = Blocks(L=2, T=16, H=2, D=64, dtype=BF16)
        b.call(c_ext.quantize_kv_blocks, [4, 0], [6, 2])
        b.call(c_ext.dequantize_kv_blocks, [1, 5], [2, 0])
        with pytest.raises(RuntimeError, match="gpu block ids"):
            b.call(c_ext.quantize_kv_blocks, [1 << 30], [0])
        with pytest.raises(OverflowError):
            c_ext.quantize_kv_blocks(torch.tensor([0]), b.ptrs, b.gkv, b.gblk, torch.tensor([0]),
                                     b.mx, b.mkv, b.mlay, b.mblk, 16 + (1 << 32), 2, 64, BF16)
        c = Case(keys=[75, 40], queries=[5, 1], seed=6)
        c.to_device()
        kv = c.qkv.to(DEV)
        H, G = c.H, c.G
        out = _step(c, kv[:, H * G:H * G + H], kv[:, H * G + H:], torch.arange(6, device=DEV))
        single = c_ext.mx4_attention(c.dq, c.dmx, H, c.dtable, c.dlens, None, 1, True)[:2]
        with pytest.raises(RuntimeError, match="scale"):
            c_ext.mx4_attention(c.dq, c.dmx, H, c.dtable, c.dlens, scale=math.nan)
        return [b.mx, *b.wide, c.dmx, out, single]
    compiled = run()
    assert type(_lib.fast()).__name__ == "module"
    monkeypatch.setenv("FLEXKV_PY_FASTCALL", "0")
    _lib.reset_fast()
    try:
        plain = run()
        assert type(_lib.fast()).__name__ == "_CtypesCalls"
    finally:
        monkeypatch.undo()
        _lib.reset_fast()
    assert all(_same(x, y) for x, y in zip(compiled, plain))


def test_two_streams_at_once():
    cases = [Case(keys=[6500, 40 + i], queries=[1, 3], H=2, G=4, seed=40 + i) for i in range(2)]
    for c in cases:
        c.to_device()
    want = [c_ext.mx4_attention(c.dq, c.dmx, c.H, c.dtable, c.dlens, c.dstarts) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(c_ext.mx4_attention(c.dq, c.dmx, c.H, c.dtable, c.dlens, c.dstarts))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)
