"""The operators on a paged cache on the device: tokens into their slots and eviction bit for
bit, attention and the tokens' weights against 64 bits."""
import math

import pytest
import torch

from flexkv_amd import _lib, c_ext
from flexkv_amd.storage.allocator import pinned_empty

import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _same(a, b):
    """Equal as bytes, NaN for NaN."""
    a, b = a.cpu(), b.cpu()
    if not a.is_floating_point():
        return torch.equal(a, b)
    both = torch.isnan(a) & torch.isnan(b)
    ints = torch.int16 if a.element_size() == 2 else torch.int32
    same = a.contiguous().view(ints) == b.contiguous().view(ints)
    return bool((same | both).all())


def _on_device(cache, layout):
    """A cache [K|V, block, token, head, D] on the device, its halves as views of that layout."""
    if layout == "layer":                    # [2, N, T, H, D]
        c = cache.to(DEV)
        return c[0], c[1]
    if layout == "block":                    # [N, 2, T, H, D]
        c = cache.transpose(0, 1).contiguous().to(DEV)
        return c[:, 0], c[:, 1]
    if layout == "heads":                    # [2, N, H, T, D]
        c = cache.transpose(2, 3).contiguous().to(DEV).transpose(2, 3)
        return c[0], c[1]
    if layout == "apart":                    # two tensors, V's heads before its tokens
        return cache[0].to(DEV), cache[1].transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    assert layout == "wide"                  # rows with others behind them
    c = torch.full((*cache.shape[:-1], cache.shape[-1] + 24), math.nan, dtype=cache.dtype)
    c[..., :cache.shape[-1]] = cache
    c = c.to(DEV)[..., :cache.shape[-1]]
    return c[0], c[1]


LAYOUTS = ("layer", "block", "heads", "apart", "wide")


# -- tokens --------------------------------------------------------------------------

@pytest.mark.parametrize("T,H,D,dtype,halves,n,slot_type,layout", [
    (16, 8, 128, BF16, 2, 1, torch.int64, "layer"),
    (16, 2, 64, FP16, 2, 37, torch.int32, "block"),
    (1, 3, 8, BF16, 2, 50, torch.int64, "layer"),
    (32, 1, 576, BF16, 1, 70, torch.int64, "layer"),
    (5, 3, 20, FP32, 2, 13, torch.int32, "heads"),
    (64, 2, 256, FP16, 2, 200, torch.int64, "apart"),
    (16, 2, 40, BF16, 2, 9, torch.int64, "wide"),
    (16, 1, 128, BF16, 2, 0, torch.int64, "layer"),
])
def test_tokens_reach_their_slots_and_nothing_else(per_call_path, T, H, D, dtype, halves, n,
                                                   slot_type, layout):
    g = _gen(n)
    blocks = n // T + 7
    cache = torch.randn(2, blocks, T, H, D, generator=g).to(dtype)
    kc, vc = _on_device(cache, layout)
    wide = torch.randn(n, 3 * H, D, generator=g).to(dtype)
    wide.view(-1)[:3] = torch.tensor([math.nan, -math.inf, -0.0])[:wide.numel()]
    dev = wide.to(DEV)
    slots = torch.randperm(blocks * T, generator=g)[:n].to(slot_type)
    if n > 4:                                # padding
        slots[1], slots[3] = -1, blocks * T
    if halves == 1:
        c_ext.write_kv_tokens(dev[:, H:2 * H], None, kc, None, slots.to(DEV))
    else:
        c_ext.write_kv_tokens(dev[:, H:2 * H], dev[:, 2 * H:], kc, vc, slots.to(DEV))
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * T:
            cache[0, s // T, s % T] = wide[i, H:2 * H]
            if halves == 2:
                cache[1, s // T, s % T] = wide[i, 2 * H:]
    assert _same(kc, cache[0]) and _same(vc, cache[1])


def test_token_calls_refuse_what_they_cannot_take(per_call_path):
    x = torch.zeros(3, 2, 64, device=DEV, dtype=BF16)
    cache = torch.zeros(4, 16, 2, 64, device=DEV, dtype=BF16)
    slots = torch.arange(3, device=DEV)
    call = c_ext.write_kv_tokens
    call(x, x, cache, cache.clone(), slots)
    for args in ((x.transpose(1, 2), x, cache, cache, slots), (x, x[:2], cache, cache, slots),
                 (x, x.half(), cache, cache, slots), (x, None, cache, cache, slots),
                 (x, x, cache, None, slots), (x, x, cache[0], cache[0], slots),
                 (x, x, cache, cache[:2], slots), (x, x, cache, cache.half(), slots),
                 (x, x, cache.half(), cache.half(), slots), (x, x, cache, cache, slots.float()),
                 (x, x, cache, cache, slots[:2]), (x[:, :1], x[:, :1], cache, cache, slots),
                 (x, x, cache, cache, torch.arange(6, device=DEV)[::2]),
                 (x, x, cache.transpose(2, 3), cache.transpose(2, 3), slots)):
        with pytest.raises(ValueError):
            call(*args)
    with pytest.raises(TypeError):
        call(x, x, cache.to(torch.int16), cache.to(torch.int16), slots)
    with pytest.raises(RuntimeError, match="device tensor"):
        call(x, x, cache, cache, slots.cpu())
    odd = torch.zeros(3 * 2 * 64 + 1, device=DEV, dtype=BF16)[1:].view(3, 2, 64)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        call(odd, x, cache, cache, slots)
    odd = torch.zeros(4, 16, 2, 68, device=DEV, dtype=BF16)[..., :64]
    with pytest.raises(RuntimeError, match="multiples of 16"):
        call(x, x, odd, odd, slots)
    small = torch.zeros(4, 16, 2, 4, device=DEV, dtype=BF16)
    with pytest.raises(RuntimeError, match="head_size"):
        call(x[..., :4], x[..., :4], small, small, slots)


# -- attention -----------------------------------------------------------------------

class Case:
    """Sequences of `keys` keys whose last `queries` tokens ask."""

    def __init__(self, keys, queries, H=2, G=4, D=128, T=16, dtype=BF16, index=torch.int32,
                 layout="layer", spread=1.0, seed=0, spare_rows=0, width=0):
        self.keys, self.queries, self.spare = keys, queries, spare_rows
        self.H, self.G, self.D, self.T, self.dtype = H, G, D, T, dtype
        g = _gen(seed)
        pages = [-(-max(k, 0) // T) for k in keys]
        self.N = sum(pages) + 2
        # what belongs to no token is NaN
        self.cache = torch.full((2, self.N, T, H, D), math.nan, dtype=dtype)
        perm = torch.randperm(self.N, generator=g).tolist()
        self.table = torch.zeros(len(keys), max([width, 1, *pages]), dtype=index)
        for b, (p, k) in enumerate(zip(pages, keys)):
            ids = [perm.pop() for _ in range(p)]
            self.table[b, :p] = torch.tensor(ids, dtype=index)
            if k > 0:
                t = torch.arange(k)
                self.cache[:, torch.tensor(ids)[t // T], t % T] = torch.randn(
                    2, k, H, D, generator=g).to(dtype)
        self.layout = layout
        self.lens = torch.tensor(keys, dtype=index)
        starts = [0]
        for n in queries:
            starts.append(starts[-1] + n)
        self.total = starts[-1]
        self.starts = torch.tensor(starts, dtype=index)
        rows = self.total + spare_rows
        self.q = (spread * torch.randn(rows, H * G, D, generator=g)).to(dtype)
        self.w = torch.rand(len(keys), H, self.table.shape[1] * T + 3, generator=g)

    def device(self):
        """The calls' arguments on the device."""
        kc, vc = _on_device(self.cache, self.layout)
        return dict(query=self.q.to(DEV), key_cache=kc, value_cache=vc,
                    block_table=self.table.to(DEV), seq_lens=self.lens.to(DEV),
                    query_starts=self.starts.to(DEV))

    def run(self, weights=True, **kw):
        args = {**self.device(), **kw}
        if kw.get("query_starts", 1) is None:
            args["query_starts"] = None
        lse = torch.full(self.q.shape[:2], 77.0, device=DEV)
        w = self.w.to(DEV) if weights else None
        out = c_ext.paged_attention(**args, lse=lse, weights=w)
        torch.cuda.synchronize()
        return out.cpu(), lse.cpu(), w.cpu() if weights else None

    def check(self, got, scale=None, causal=True, lost=()):
        """`lost`: (sequence, token): the rows that see it are NaN, and give NaN weights."""
        out, lse, w = got
        scale = self.D ** -0.5 if scale is None else scale
        at = 0
        want_w = self.w.to(torch.float64)
        for b, (k, n) in enumerate(zip(self.keys, self.queries)):
            keys = max(k, 0)
            kv = [torch.stack([c[int(self.table[b, t // self.T]), t % self.T]
                               for t in range(keys)]) if keys else c[:0, 0] for c in self.cache]
            pos = torch.arange(n).repeat_interleave(self.G)
            visible = (keys - n + pos + 1).clamp(min=0) if causal else torch.full_like(pos, keys)
            for h in range(self.H):
                heads = slice(h * self.G, (h + 1) * self.G)
                q = self.q[at:at + n, heads].reshape(n * self.G, self.D)
                kh, vh = kv[0][:, h], kv[1][:, h]
                wo, wl, p, mags = po.attention(q, kh, vh, scale, visible)
                tol = po.tolerance(wo, p, vh.float().nan_to_num(0, 0, 0), mags, self.dtype)
                gone = torch.zeros(n * self.G, dtype=torch.bool)
                for s, t in lost:
                    if s == b:
                        gone |= visible > t
                go = out[at:at + n, heads].reshape(n * self.G, self.D).double()
                gl = lse[at:at + n, heads].reshape(n * self.G).double()
                assert go[gone].isnan().all() and gl[gone].isnan().all()
                ok = ~gone
                bad = ~((go - wo).abs() <= tol)[ok] & ~(go.isnan() & wo.isnan())[ok]
                assert not bad.any(), (b, h, (go - wo).abs().max(), tol.min(),
                                       bad.nonzero()[:5].tolist())
                none = (visible == 0) & ok
                assert (go[none] == 0).all() and (gl[none] == -math.inf).all()
                seen = (visible > 0) & ok
                ltol = po.score_error(mags, self.D) + keys * 2.0 ** -23 + 2.0 ** -22 * wl.abs() \
                    + 2.0 ** -20
                assert ((gl - wl).abs() <= ltol)[seen].all(), (gl - wl)[seen].abs().max()
                if w is not None:
                    before = want_w[b, h, :keys]
                    total = before + p.sum(0)
                    wtol = po.weights_tolerance(p, mags, self.D, before, total)
                    gw = w[b, h, :keys].double()
                    tok = torch.arange(keys)
                    nan = torch.zeros(keys, dtype=torch.bool)
                    if gone.any():
                        nan = tok < visible[gone].max()
                    assert gw[nan].isnan().all()
                    off = ((gw - total).abs() - wtol)[~nan]
                    assert not (off > 0).any() and not off.isnan().any(), (b, h, off.max())
            if w is not None:
                assert torch.equal(w[b, :, keys:], self.w[b, :, keys:])
            at += n


SHAPES = [
    # one token each, lengths around the steps' and blocks' ends
    dict(keys=[1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100], queries=[1] * 12),
    dict(keys=[777], queries=[1], H=8),
    dict(keys=[300, 5], queries=[1, 1], D=64, G=1, dtype=FP16, layout="block"),
    dict(keys=[129, 1000], queries=[1, 1], D=256, G=8, H=1, layout="heads", index=torch.int64),
    dict(keys=[200, 77], queries=[1, 1], D=128, G=16, H=1, dtype=FP16, T=1, layout="apart"),
    dict(keys=[90, 41], queries=[1, 1], G=5, H=3, T=7, layout="wide"),
    dict(keys=[260, 33], queries=[1, 1], G=23, H=2, T=20),
    # a few and many queries
    dict(keys=[40, 9, 130], queries=[3, 9, 5], D=64, dtype=FP16, layout="block"),
    dict(keys=[500, 301], queries=[5, 4], G=8, D=64, H=3, T=8),
    dict(keys=[70, 300, 64], queries=[70, 41, 1], H=1, T=32),
    dict(keys=[333], queries=[333], G=3, dtype=FP16),
    dict(keys=[150, 20], queries=[37, 20], D=256, G=2, T=16),
    dict(keys=[400], queries=[130], D=256, G=8, H=1, dtype=FP16, T=64),
    dict(keys=[513, 100, 700], queries=[200, 100, 150], G=4, H=2, T=48, layout="block"),
    dict(keys=[600, 90], queries=[129, 64], G=1, H=2, D=64, T=3),
    # rows that see nothing, sequences without keys or queries
    dict(keys=[0, 3, 0, 20, 5], queries=[1, 5, 0, 0, 9]),
    dict(keys=[0], queries=[1], D=64, dtype=FP16),
    dict(keys=[2, 40], queries=[90, 60], G=4, H=1),
    # a long one, cut along the keys, alone and among short ones
    dict(keys=[9000], queries=[1], H=1, G=8, dtype=FP16),
    dict(keys=[8200, 40, 7000], queries=[1, 1, 1], H=2, G=4),
    dict(keys=[12000, 100], queries=[5, 3], H=1, G=8, T=64),
    dict(keys=[7000], queries=[60], H=1, G=4),
    # dealt out among more than 64 sequences, and more than are dealt out; cut among more than 64
    dict(keys=[3000, *range(1, 70)], queries=[1] * 70, H=1, G=3, D=64),
    dict(keys=[40 - n % 40 for n in range(260)], queries=[1] * 260, H=1, G=2, T=8, width=300),
    dict(keys=[3000, *range(10, 79)], queries=[10] * 70, H=1, D=64, dtype=FP16),
    # two tiles of 16 rows for a wavefront, dealt out; two for each sequence
    dict(keys=[4200, 90], queries=[6, 7], H=1),
    dict(keys=[2300], queries=[4], H=2, G=7, D=64, dtype=FP16),
    dict(keys=[2600, 31], queries=[1, 1], H=1, G=23, D=256),
    dict(keys=[70, 5], queries=[3, 2], H=1, G=9, D=256, dtype=FP16),
    # a table so wide that the scores are not kept
    dict(keys=[3000], queries=[2], H=1, G=8, T=1024, width=16500),
    # one row for each share of the rows that weigh, and rows that nothing is seen by
    dict(keys=[30, 257], queries=[100, 200], H=1, G=1, D=64),
    dict(keys=[1100], queries=[700], H=1, G=1, D=256, dtype=FP16, T=128),
]


@pytest.mark.parametrize("kw", SHAPES, ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_attention_and_weights(kw):
    c = Case(**kw)
    c.check(c.run())


@pytest.mark.parametrize("kw,run", [
    (dict(keys=[40, 9], queries=[3, 9]), dict(causal=False)),
    (dict(keys=[300], queries=[70]), dict(causal=False)),
    (dict(keys=[120, 7], queries=[4, 7], dtype=FP16), dict(scale=-0.21)),
    (dict(keys=[130], queries=[80], G=2), dict(scale=-0.3)),
    (dict(keys=[150], queries=[2]), dict(scale=0.0)),
    (dict(keys=[500], queries=[40], spread=20.0), dict()),
    (dict(keys=[500], queries=[1], spread=30.0, dtype=FP16), dict()),
])
def test_attention_with_other_masks_and_scales(kw, run):
    c = Case(**kw)
    c.check(c.run(**run), scale=run.get("scale"), causal=run.get("causal", True))


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, FP16), (256, BF16)])
def test_one_query_a_sequence_without_starts(D, dtype):
    c = Case([50, 600, 1], [1, 1, 1], D=D, dtype=dtype, spare_rows=2)
    out = torch.full((5, c.H * c.G, D), 3.0, device=DEV, dtype=dtype)
    got = c.run(query_starts=None, out=out)
    c.check(got)
    assert (got[0][3:] == 3.0).all() and (got[1][3:] == 77.0).all()


def test_rows_of_no_sequence_are_left_as_they_were():
    c = Case([50, 600], [4, 70], spare_rows=9)
    out = torch.full((83, 8, 128), 3.0, device=DEV, dtype=BF16)
    got = c.run(out=out)
    c.check(got)
    assert (got[0][74:] == 3.0).all() and (got[1][74:] == 77.0).all()


@pytest.mark.parametrize("queries", [[1, 1], [5, 3], [90, 64]])
def test_without_weights_or_lse_the_output_is_the_same(per_call_path, queries):
    c = Case([300, 70], queries)
    out, _, _ = c.run()
    plain = c_ext.paged_attention(**c.device())
    assert _same(out, plain)
    assert _same(out, c_ext.paged_attention(**c.device()))      # and from run to run


@pytest.mark.parametrize("queries", [[1, 1], [40, 64]])
def test_queries_and_outputs_of_any_stride(queries):
    c = Case([90, 200], queries, G=2)
    rows, heads, D = c.q.shape
    for layout in ("rows", "heads"):
        if layout == "rows":
            q = torch.full((rows, heads + 3, D + 8), math.nan, dtype=BF16)[:, 1:heads + 1, :D]
            out = torch.zeros(rows, heads + 1, D + 16, device=DEV, dtype=BF16)[:, :heads, 8:D + 8]
        else:
            q = torch.empty(heads, rows, D, dtype=BF16).transpose(0, 1)
            out = torch.zeros(heads, rows, D, device=DEV, dtype=BF16).transpose(0, 1)
        q.copy_(c.q)
        dq = torch.empty_strided(q.shape, q.stride(), dtype=BF16, device=DEV).copy_(q)
        c.check(c.run(query=dq, out=out))


@pytest.mark.parametrize("queries,T,D", [(1, 16, 128), (3, 16, 128), (100, 16, 128), (100, 5, 128),
                                         (6, 16, 128), (8, 8, 64), (50, 16, 64), (4, 16, 256),
                                         (60, 32, 256)])
def test_what_is_not_a_number_reaches_only_those_that_see_it(queries, T, D):
    """In keys and values, at the first, some and the last token."""
    n = 150
    for half in (0, 1):
        for t in (0, n - queries // 2 - 1, n - 1):
            for x in (math.nan, math.inf):
                c = Case([n, 40], [queries, 1], H=1, G=4, D=D, T=T, seed=t)
                c.cache[half, int(c.table[0, t // T]), t % T, 0, 5] = x
                out, lse, w = c.run()
                visible = n - queries + 1 + torch.arange(queries)
                sees = visible > t
                hit = ~out[:queries].isfinite()
                if half:
                    # only this element of the rows that see it
                    want = torch.zeros_like(hit)
                    want[sees, :, 5] = True
                    assert torch.equal(hit, want)
                else:
                    # a score that is NaN, or infinite: then a weight of 0 or NaN
                    assert not hit[~sees].any()
                    if math.isnan(x):
                        assert hit[sees].all()
                assert out[queries:].isfinite().all()
                # the rest is as without it
                c.cache[half, int(c.table[0, t // T]), t % T, 0, 5] = 0.5
                plain = c.run()[0]
                rest = ~hit if half else ~sees[:, None, None].expand_as(hit)
                tol = 0.04                   # other roundings where products are made one by one
                assert ((out[:queries] - plain[:queries]).abs()[rest] <= tol).all()


@pytest.mark.parametrize("queries", [1, 4, 100])
def test_blocks_outside_the_cache_make_their_rows_nan(queries):
    for token, block in ((0, -1), (120, 1 << 20), (191, -5)):
        c = Case([192, 60], [queries, 1], index=torch.int64, seed=token)
        args = c.device()
        table = c.table.clone()
        table[0, token // 16] = block
        got = c.run(block_table=table.to(DEV))
        c.check(got, lost=[(0, token // 16 * 16)])
        del args


@pytest.mark.parametrize("queries", [1, 40])
def test_lengths_that_cannot_be(queries):
    c = Case([100, 100], [queries, queries], index=torch.int64)
    lens = torch.tensor([113, -4])           # a row of the table holds 112
    out, lse, w = c.run(seq_lens=lens.to(DEV))
    assert out[:queries].isnan().all() and lse[:queries].isnan().all()
    assert (out[queries:] == 0).all() and (lse[queries:] == -math.inf).all()
    assert torch.equal(w, c.w)


def test_starts_past_the_rows_are_cut_off():
    c = Case([100, 100], [3, 3], index=torch.int64)
    out = torch.full((6, 8, 128), 3.0, device=DEV, dtype=BF16)
    c.run(query_starts=torch.tensor([0, 3, 1 << 40], device=DEV), out=out)
    c.run(query_starts=torch.tensor([-7, 3, 6], device=DEV), out=out)


@pytest.mark.parametrize("queries,D", [(1, 64), (10, 64), (30, 64), (1, 256), (30, 256)])
def test_scores_far_from_zero(queries, D):
    """Products of 2^27 and more: weights as their rounded products have them."""
    c = Case([200], [queries], H=1, G=2, D=D, seed=3)
    c.q = torch.full_like(c.q, 2.0 ** 14)
    for t in range(200):
        c.cache[0, int(c.table[0, t // 16]), t % 16] = 2.0 ** 13 if t == 30 else 2.0 ** 12
    out, lse, w = c.run(scale=1.0)
    v = c.cache[1, int(c.table[0, 1]), 14, 0]
    assert (out == v).all()
    want = c.w[0, 0].clone()
    want[30] += 2 * queries
    assert torch.allclose(w[0, 0], want, rtol=2.0 ** -20, atol=0)
    out, _, _ = c.run(scale=-1.0)
    assert out.isfinite().all()


@pytest.mark.parametrize("keys,queries,D", [(70, 1, 64), (4300, 1, 128), (90, 6, 128), (300, 100, 128),
                                            (3000, 40, 256)])
def test_the_largest_values_of_fp16_stay_finite(keys, queries, D):
    """All values are one of the two largest: so are results, to a rounding of the weights (2^-11, one
    of 11 bits, and 2^-12 of the sums) and one of their own."""
    c = Case([keys], [queries], H=1, D=D, dtype=FP16, seed=keys)
    c.cache[1] = torch.where(c.cache[1] > 0, 65504.0, -65504.0)
    c.cache[1, ..., 0] = 65504.0
    c.cache[1, ..., 1] = -65472.0
    out, _, _ = c.run()
    assert out.isfinite().all()
    assert ((out[..., 0].double() - 65504).abs() <= 65504 * 2.0 ** -10).all()
    assert ((out[..., 1].double() + 65472).abs() <= 65504 * 2.0 ** -10).all()


def test_a_cache_past_4_gib():
    T, H, D = 16, 1, 128
    N = (1 << 32) // (T * H * D * 2) + 64
    cache = torch.empty(2, N, T, H, D, dtype=BF16, device=DEV)
    g = _gen(5)
    c = Case([500, 77], [9, 1], H=H, D=D, T=T, seed=4)
    far = (N - 1 - torch.randperm(60, generator=g)[:c.N]).to(torch.int32)
    cache[:, far.to(DEV).long()] = c.cache.to(DEV)
    table = far[c.table.long()].to(torch.int32).to(DEV)
    c.check(c.run(key_cache=cache[0], value_cache=cache[1], block_table=table))
    # and tokens written there
    slots = (far[:3].long() * T + 5).to(DEV)
    x = torch.randn(3, H, D, generator=g).to(BF16).to(DEV)
    c_ext.write_kv_tokens(x, -x, cache[0], cache[1], slots)
    assert _same(cache[0][far[:3].to(DEV).long(), 5], x)
    assert _same(cache[1][far[:3].to(DEV).long(), 5], -x)


def test_attention_refuses_what_it_cannot_take(per_call_path):
    c = Case([50, 20], [3, 1])
    d = c.device()

    def call(**kw):
        return c_ext.paged_attention(**{**d, **kw})
    call()
    q, kc, vc = d["query"], d["key_cache"], d["value_cache"]
    w = torch.zeros(2, 2, 64, device=DEV)
    for kw in (dict(query=q.float()), dict(query=q[0]), dict(query=q.transpose(1, 2)),
               dict(query=q[:, :7]), dict(query=q.half()), dict(key_cache=kc[0]),
               dict(key_cache=kc.half(), value_cache=vc.half()), dict(value_cache=vc[:, :8]),
               dict(key_cache=kc[..., :64], value_cache=vc[..., :64]),
               dict(seq_lens=d["seq_lens"].long()), dict(seq_lens=d["seq_lens"].float()),
               dict(seq_lens=d["seq_lens"][:1]), dict(block_table=d["block_table"].t()),
               dict(query_starts=d["query_starts"][:2]), dict(query_starts=None, query=q[:1]),
               dict(query_starts=d["query_starts"].long()),
               dict(out=torch.empty(4, 8, 128, device=DEV)), dict(out=q), dict(out=q[:2]),
               dict(lse=torch.empty(4, 7, device=DEV)),
               dict(lse=torch.empty(4, 8, device=DEV, dtype=BF16)),
               dict(weights=w[:1]), dict(weights=w[:, :1]), dict(weights=w[..., :63]),
               dict(weights=w.double()),
               dict(weights=torch.zeros(2, 2, 128, device=DEV)[..., ::2]),
               dict(weights=w[:, :1].expand_as(w)), dict(weights=w[:1].expand_as(w)),
               dict(lse=torch.empty(4, 1, device=DEV).expand(4, 8)),
               dict(out=torch.empty(1, 8, 128, device=DEV, dtype=BF16).expand(4, 8, 128))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(TypeError):
        call(value_cache=None)
    with pytest.raises(RuntimeError, match="device tensor"):
        call(seq_lens=c.lens)
    with pytest.raises(RuntimeError, match="scale"):
        call(scale=math.inf)
    with pytest.raises(RuntimeError, match="head_size"):
        call(query=q[..., :96], key_cache=kc[..., :96], value_cache=vc[..., :96])
    with pytest.raises(RuntimeError, match="gradient"):
        call(query=q.clone().requires_grad_())
    with torch.no_grad():
        call(query=q.clone().requires_grad_())


def test_on_another_stream_and_in_captured_graphs():
    """Two graphs that share their memory, replayed in turn with eager calls and with other
    lengths, on a stream of their own."""
    cases = [Case([300, 41], [1, 1], H=1, seed=1), Case([700, 70], [40, 5], seed=2),
             Case([9000], [1], H=1, G=8, seed=3), Case([320, 30], [150, 9], H=1, seed=4)]
    stream = torch.cuda.Stream()
    graphs, outs, pool = [], [], None
    for c in cases:
        d = c.device()
        w = c.w.to(DEV)
        before = w.clone()
        out = torch.zeros_like(d["query"])
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.default_stream())
            c_ext.paged_attention(**d, out=out, weights=w)
        stream.synchronize()
        c.check((out.cpu(), torch.full(c.q.shape[:2], 0.0), w.cpu())[:1] + c.run()[1:])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, pool=pool):
            w.copy_(before)
            c_ext.paged_attention(**d, out=out, weights=w)
        pool = graph.pool()
        graphs.append((graph, d, out, w, before))
    for i in range(3):
        for c, (graph, d, out, w, _) in zip(cases, graphs):
            lens = c.lens - 7 * i
            d["seq_lens"].copy_(lens)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            eager, lse, ew = c.run(seq_lens=lens.to(DEV))
            assert _same(out, eager) and _same(w, ew)


# -- eviction ------------------------------------------------------------------------

class Evict:
    def __init__(self, keys, budget, H=2, D=64, T=16, dtype=BF16, index=torch.int32,
                 layout="layer", halves=2, ties=False, seed=0, spare=2, width=0):
        self.keys, self.budget, self.T, self.H, self.halves = keys, budget, T, H, halves
        g = _gen(seed)
        pages = [-(-max(k, 0) // T) for k in keys]
        new_pages = [-(-min(max(k, 0), budget) // T) for k in keys]
        self.N = sum(pages) + sum(new_pages) + spare
        self.cache = torch.randn(2, self.N, T, H, D, generator=g).to(dtype)
        perm = torch.randperm(self.N, generator=g).tolist()

        def tables(counts, least):
            t = torch.full((len(keys), max([least, 1, *counts])), 0, dtype=index)
            for b, p in enumerate(counts):
                t[b, :p] = torch.tensor([perm.pop() for _ in range(p)], dtype=index)
            return t
        self.table = tables(pages, width)
        most = self.table.shape[1] * T
        self.new_table = tables(new_pages, -(-min(budget, most) // T))
        self.layout, self.lens = layout, torch.tensor(keys, dtype=index)
        self.w = torch.rand(len(keys), H, most + 1, generator=g)
        if ties:
            self.w = (self.w * 4).round() / 4
        self.given = torch.rand(len(keys), H, min(budget, most) + 2, generator=g)

    def run(self, recent, in_place=False, **kw):
        self.kc, self.vc = _on_device(self.cache, self.layout)
        w = self.w.to(DEV)
        nw = w if in_place else self.given.to(DEV)
        args = dict(key_cache=self.kc, value_cache=self.vc if self.halves == 2 else None,
                    weights=w, block_table=self.table.to(DEV), seq_lens=self.lens.to(DEV),
                    new_table=self.new_table.to(DEV), budget=self.budget, recent=recent,
                    new_weights=nw)
        args.update(kw)
        kept = c_ext.evict_kv_tokens(**args)
        torch.cuda.synchronize()
        if not in_place:
            assert _same(w, self.w)
        return kept.cpu(), nw.cpu()

    def check(self, got, recent, in_place=False, no_copy=()):
        kept, nw = got
        want = self.cache.clone()
        for b, n in enumerate(self.keys):
            n = max(n, 0)
            for h in range(self.H):
                stay = po.choose(self.w[b, h], n, self.budget, recent)
                pad = [-1] * (self.budget - len(stay))
                assert kept[b, h].tolist() == stay + pad, (b, h)
                wide = torch.zeros(nw.shape[2])
                wide[:len(stay)] = self.w[b, h, stay]
                assert _same(nw[b, h], wide)
                for i, t in enumerate(stay):
                    if (b, t // self.T) in no_copy:
                        continue
                    old = int(self.table[b, t // self.T]), t % self.T, h
                    new = int(self.new_table[b, i // self.T]), i % self.T, h
                    for k in range(self.halves):
                        want[k][new] = self.cache[k][old]
        assert _same(self.kc, want[0]) and _same(self.vc, want[1])


EVICT = [
    (dict(keys=[100, 20, 64], budget=30), 7),
    (dict(keys=[100, 20, 0], budget=30, H=1, D=128, dtype=FP16, layout="block"), 30),
    (dict(keys=[1, 2, 3], budget=1, D=8, T=1), 0),
    (dict(keys=[1, 2, 3], budget=2, D=8, T=1, index=torch.int64), 1),
    (dict(keys=[300, 301], budget=300, ties=True, layout="heads"), 0),
    (dict(keys=[500, 77], budget=64, ties=True, H=3, T=5, D=20, dtype=FP32, layout="apart"), 13),
    (dict(keys=[200], budget=90, H=1, D=576, halves=1, T=64), 16),
    (dict(keys=[90], budget=1000, width=9), 100),
    (dict(keys=[9000, 8192, 1024], budget=5000, H=1, D=8, ties=True), 1000),
    (dict(keys=[40000], budget=17000, H=1, D=8, T=64), 0),
    (dict(keys=[2500, 700], budget=129, H=8, D=128, layout="wide"), 64),
]


@pytest.mark.parametrize("kw,recent", EVICT, ids=str)
def test_eviction_bit_for_bit(per_call_path, kw, recent):
    c = Evict(**kw)
    c.check(c.run(recent), recent)


@pytest.mark.parametrize("kw,recent", [EVICT[0], EVICT[5], EVICT[8]], ids=str)
def test_eviction_of_the_weights_in_place(kw, recent):
    c = Evict(**kw)
    c.check(c.run(recent, in_place=True), recent)


# several workgroups choose for one sequence: few sequences, and table rows of 2^15 tokens or more
LONG = [
    (dict(keys=[40000, 0, 1, 20001], budget=17000, H=1, D=8, T=64), 1000),
    (dict(keys=[16385, 1023, 16384], budget=1025, H=3, D=8, T=1, ties=True, width=33000), 1024),
    (dict(keys=[30000, 700], budget=20000, H=2, D=8, T=32, index=torch.int64, width=2000), 20000),
    (dict(keys=[17000, 9000], budget=9000, H=1, D=8, T=16, ties=True, width=2100), 0),
    (dict(keys=[100], budget=40, H=1, D=64, T=16, width=2500), 3),
    (dict(keys=[150001], budget=100, H=1, D=8, T=32, ties=True), 7),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kw,recent", LONG, ids=str)
def test_eviction_of_long_sequences(kw, recent, in_place):
    c = Evict(**kw)
    c.check(c.run(recent, in_place), recent, in_place)


def test_eviction_of_long_sequences_orders_every_kind_of_weight(per_call_path):
    c = Evict([20000, 16400], 5000, D=8, T=16, width=2048)
    hard = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 1e38, -3.0,
                         -math.nan, 2.0 ** -126, 0.5])
    c.w[0, 0, :18000] = hard.repeat(1500)
    c.w[0, 1, :20000] = 0.0
    c.w[1, 0, :16400] = math.nan
    c.w[1, 1, :16400] = torch.linspace(1, 0, 16400)
    for recent in (0, 3000, 5000):
        c.check(c.run(recent), recent)
    kept = torch.full((2, 2, 5000), 9, dtype=torch.int32, device=DEV)
    got, _ = c.run(7, new_weights=None, kept=kept)
    assert torch.equal(kept.cpu(), got)
    c.check(c.run(7), 7)
    assert torch.equal(c.run(7)[0], got)
    kept, nw = c.run(5, seq_lens=torch.tensor([32769, -2], dtype=torch.int32, device=DEV))
    assert (kept == -1).all()
    assert _same(nw[0], c.given[0]) and (nw[1] == 0).all()


def test_eviction_of_long_sequences_in_captured_graphs():
    """Two graphs, replayed in turn; of one the lengths change."""
    c = [Evict([20000, 16400], 5000, H=1, D=8, T=16, seed=1, width=2048), Evict([40000], 300, D=8, seed=2)]
    state = []
    for e in c:
        kc, vc = _on_device(e.cache, "layer")
        dev = [x.to(DEV) for x in (e.w, e.table, e.lens, e.new_table)]
        args = (kc, vc, *dev, e.budget, 20, e.given.to(DEV))
        c_ext.evict_kv_tokens(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = c_ext.evict_kv_tokens(*args)
        state.append((e, graph, args, kept))
    for i in range(3):
        for e, graph, args, kept in state:
            e.w = torch.rand(e.w.shape, generator=_gen(i))
            args[2].copy_(e.w)
            if len(e.keys) == 2:
                e.keys = [20000 - 7 * i, 16400 >> 4 * i]
                args[4].copy_(torch.tensor(e.keys))
            args[0].copy_(e.cache[0]), args[1].copy_(e.cache[1])
            graph.replay()
        torch.cuda.synchronize()
        for e, graph, args, kept in state:
            e.kc, e.vc = args[:2]
            e.check((kept.cpu(), args[8].cpu()), 20)


def test_eviction_orders_every_kind_of_weight():
    c = Evict([64, 64], 20, T=8)
    hard = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 1e38, -3.0,
                         -math.nan, 2.0 ** -126, 0.5])
    c.w[0, :, :60] = hard.repeat(5)
    c.w[1, 0, :64] = 0.0
    c.w[1, 1, :64] = -0.0
    c.w[1, 1, 1:64:2] = 0.0
    for recent in (0, 3):
        c.check(c.run(recent), recent)
    c.w[0, :, :64] = math.nan
    c.check(c.run(2), 2)


def test_eviction_without_new_weights_and_with_a_given_list(per_call_path):
    c = Evict([100, 20], 30)
    kept = torch.full((2, 2, 30), 9, dtype=torch.int32, device=DEV)
    got, _ = c.run(7, new_weights=None, kept=kept)
    again, nw = c.run(7)
    assert torch.equal(got, again) and torch.equal(kept.cpu(), got)
    c.check((again, nw), 7)


def test_eviction_leaves_out_what_lies_outside_the_cache():
    c = Evict([100, 50], 60, index=torch.int64)
    table, new_table = c.table.clone(), c.new_table.clone()
    table[0, 2], new_table[1, 1] = 1 << 40, -3
    got = c.run(5, block_table=table.to(DEV), new_table=new_table.to(DEV))
    c.new_table[1, 1] = c.N + 5              # the oracle writes that page into rows cut off below
    pad = torch.zeros(2, 6, *c.cache.shape[2:], dtype=c.cache.dtype)
    c.cache = torch.cat((c.cache, pad), 1)
    c.kc = torch.cat((c.kc, c.kc.new_zeros(6, *c.kc.shape[1:])))
    c.vc = torch.cat((c.vc, c.vc.new_zeros(6, *c.vc.shape[1:])))
    for h in range(2):                       # what the oracle puts into that block
        for i, t in enumerate(po.choose(c.w[1, h], 50, 60, 5)):
            if i // 16 == 1:
                for k, half in enumerate((c.kc, c.vc)):
                    half[c.N + 5, i % 16, h] = c.cache[k][int(c.table[1, t // 16]), t % 16, h].to(
                        DEV)
    c.check(got, 5, no_copy={(0, 2)})


def test_eviction_of_lengths_that_cannot_be():
    c = Evict([100, 50], 40, index=torch.int64)
    kept, nw = c.run(5, seq_lens=torch.tensor([113, -2], device=DEV))
    assert (kept == -1).all()
    assert _same(nw[0], c.given[0]) and (nw[1] == 0).all()
    assert _same(c.kc, c.cache[0]) and _same(c.vc, c.cache[1])


def test_eviction_refuses_what_it_cannot_take(per_call_path):
    c = Evict([100, 20], 30)
    ok = dict(key_cache=c.cache[0].to(DEV), value_cache=c.cache[1].to(DEV), weights=c.w.to(DEV),
              block_table=c.table.to(DEV), seq_lens=c.lens.to(DEV), new_table=c.new_table.to(DEV),
              budget=30, recent=3)

    def call(**kw):
        return c_ext.evict_kv_tokens(**{**ok, **kw})
    call()
    w = ok["weights"]
    for kw in (dict(budget=0), dict(budget=-2), dict(recent=-1), dict(recent=31),
               dict(weights=w[..., :111]), dict(weights=w[:1]), dict(weights=w.half()),
               dict(new_weights=w[..., :29]), dict(new_weights=w[..., 1:]),
               dict(new_weights=w.clone()[:, :1].expand_as(w)),
               dict(new_table=c.new_table.long().to(DEV)), dict(new_table=c.new_table[:1].to(DEV)),
               dict(block_table=c.table.t().to(DEV)), dict(seq_lens=c.lens.float().to(DEV)),
               dict(kept=torch.empty(2, 2, 29, dtype=torch.int32, device=DEV)),
               dict(kept=torch.empty(2, 2, 30, dtype=torch.int64, device=DEV)),
               dict(value_cache=ok["value_cache"][:3]), dict(key_cache=ok["key_cache"][0])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(RuntimeError, match="do not hold"):
        call(new_table=ok["new_table"][:, :1])
    with pytest.raises(RuntimeError, match="device tensor"):
        call(seq_lens=c.lens)
    with pytest.raises((TypeError, OverflowError)):
        call(budget=1 << 40)


def test_eviction_in_a_captured_graph():
    c = Evict([700, 90], 200)
    kc, vc = _on_device(c.cache, "layer")
    w, nw = c.w.to(DEV), c.given.to(DEV)
    table, lens, new = c.table.to(DEV), c.lens.to(DEV), c.new_table.to(DEV)
    graph = torch.cuda.CUDAGraph()
    c_ext.evict_kv_tokens(kc, vc, w, table, lens, new, 200, 20, nw)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kept = c_ext.evict_kv_tokens(kc, vc, w, table, lens, new, 200, 20, nw)
    for i in range(3):
        c.w = torch.rand(c.w.shape, generator=_gen(i))
        w.copy_(c.w)
        kc.copy_(c.cache[0]), vc.copy_(c.cache[1])
        graph.replay()
        torch.cuda.synchronize()
        c.kc, c.vc = kc, vc
        c.check((kept.cpu(), nw.cpu()), 20)


# -- together --------------------------------------------------------------------------

def test_a_prefix_comes_back_is_extended_weighed_and_evicted_from():
    """Blocks of a prefix come from the host cache, the rest of the prompt is written and attends
    over them, the tokens with the least of it go, and the next token goes on from there."""
    T, H, G, D, prefix, rest, budget, recent = 16, 2, 4, 128, 96, 30, 64, 16
    g = _gen(11)
    n = prefix + rest
    x = torch.randn(2, n + 1, H, D, generator=g).to(BF16)
    q = torch.randn(n + 1, H * G, D, generator=g).to(BF16)
    N = 20
    cache = torch.zeros(2, N, T, H, D, dtype=BF16, device=DEV)
    perm = torch.randperm(N, generator=g)
    old, new = perm[:8], perm[8:13]
    # the host cache: block-wise, one layer
    chunk = T * H * D * 2
    host = pinned_empty(6 * 2 * T * H * D, BF16)
    host.view(6, 2, T, H, D).copy_(x[:, :prefix].reshape(2, 6, T, H, D).transpose(0, 1))
    ptrs = torch.tensor([cache.data_ptr()])
    c_ext.transfer_kv_blocks(old[:6].contiguous(), ptrs, N * chunk, chunk, torch.arange(6), host,
                             chunk, 2 * chunk, 2 * chunk, chunk, 0, -1, True)
    table = old.to(torch.int32)[None].to(DEV)
    pos = torch.arange(prefix, n)
    slots = (old[pos // T] * T + pos % T).to(DEV)
    new_kv = x[:, prefix:n].to(DEV)
    c_ext.write_kv_tokens(new_kv[0], new_kv[1], cache[0], cache[1], slots)
    weights = torch.zeros(1, H, 8 * T, device=DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, rest], dtype=torch.int32, device=DEV)
    out = c_ext.paged_attention(q[prefix:n].to(DEV), cache[0], cache[1], table, lens, starts,
                                weights=weights)
    visible = (prefix + 1 + torch.arange(rest)).repeat_interleave(G)
    kept_w = torch.zeros(1, H, 5 * T, device=DEV)
    kept = c_ext.evict_kv_tokens(cache[0], cache[1], weights, table, lens,
                                 new.to(torch.int32)[None].to(DEV), budget, recent, kept_w)
    # the next token
    lens.clamp_(max=budget)
    slot = new[budget // T] * T + budget % T
    c_ext.write_kv_tokens(x[0, n:].to(DEV), x[1, n:].to(DEV), cache[0], cache[1],
                          slot[None].to(DEV))
    last = c_ext.paged_attention(q[n:].to(DEV), cache[0], cache[1],
                                 new.to(torch.int32)[None].to(DEV), lens + 1, weights=kept_w)
    for h in range(H):
        rows = q[prefix:n, h * G:(h + 1) * G].reshape(-1, D)
        wo, _, p, mags = po.attention(rows, x[0, :n, h], x[1, :n, h], D ** -0.5, visible)
        tol = po.tolerance(wo, p, x[1, :n, h].float(), mags, BF16)
        got = out[:, h * G:(h + 1) * G].reshape(-1, D).cpu().double()
        assert ((got - wo).abs() <= tol).all()
        stay = po.choose(weights[0, h].cpu(), n, budget, recent)
        assert kept[0, h].tolist() == stay
        k, v = (torch.cat((x[i, stay, h], x[i, n:, h])) for i in (0, 1))
        wo, _, p, mags = po.attention(q[n, h * G:(h + 1) * G], k, v, D ** -0.5,
                                      torch.full((G,), budget + 1))
        tol = po.tolerance(wo, p, v.float(), mags, BF16)
        assert ((last[0, h * G:(h + 1) * G].cpu().double() - wo).abs() <= tol).all()
        before = torch.zeros(budget + 1)
        before[:budget] = weights[0, h, stay].cpu()
        total = before.double() + p.sum(0)
        wtol = po.weights_tolerance(p, mags, D, before.double(), total)
        assert ((kept_w[0, h, :budget + 1].cpu().double() - total).abs() <= wtol).all()
        assert (kept_w[0, h, budget + 1:] == 0).all()
