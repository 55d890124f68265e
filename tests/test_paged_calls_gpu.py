"""Calls on a paged cache that are refused, or that are allowed and easily got wrong."""
import pytest
import torch

from flexkv_amd import c_ext

from test_paged_gpu import BF16, DEV, Case, Evict, _gen, _same

pytestmark = pytest.mark.gpu


# -- caches whose rows overlap -----------------------------------------------------------

def _overlapping():
    c = torch.zeros(4, 16, 2, 64, device=DEV, dtype=BF16)
    other = torch.zeros_like(c)
    flat = torch.zeros(8 * 16 * 2 * 64, device=DEV, dtype=BF16)
    shape, step = (4, 16, 2, 64), 16 * 2 * 64
    yield "key cache", c[:1].expand(shape), other
    yield "key cache", c[:, :1].expand(shape), other
    yield "value cache", other, c[:, :, :1].expand(shape)
    yield "value cache", other, flat.as_strided(shape, (step - 8, 128, 64, 1))
    yield "key and value", c, c
    yield "key and value", flat.as_strided(shape, (step, 128, 64, 1)), \
        flat.as_strided(shape, (step, 128, 64, 1), 3 * step + 128)


def test_caches_whose_rows_overlap_are_not_written_to(per_call_path):
    x = torch.ones(3, 2, 64, device=DEV, dtype=BF16)
    slots = torch.arange(3, device=DEV)
    e = Evict([40, 20], 16, T=16)
    args = [t.to(DEV) for t in (e.w, e.table[:, :2], e.lens, e.new_table)]
    for word, kc, vc in _overlapping():
        with pytest.raises(RuntimeError, match=f"{word}.*overlap"):
            c_ext.write_kv_tokens(x, x, kc, vc, slots)
        with pytest.raises(RuntimeError, match=f"{word}.*overlap"):
            c_ext.evict_kv_tokens(kc, vc, *args, 16, 3)
        if word == "key cache":
            with pytest.raises(RuntimeError, match="key cache overlap"):
                c_ext.write_kv_tokens(x, None, kc, None, slots)
        assert not kc.any() and not vc.any()
        # attention only reads them
        c_ext.paged_attention(x, kc, vc, args[1][:1], args[2][1:], None)


def test_caches_side_by_side_are_written_to(per_call_path):
    """K and V next to each other in each row, or in each token."""
    g = _gen(1)
    x = torch.randn(2, 5, 2, 64, generator=g).to(BF16)
    slots = torch.randperm(64, generator=g)[:5]
    for kc, vc in (torch.zeros(4, 16, 2, 2, 64, device=DEV, dtype=BF16).unbind(3),
                   torch.zeros(4, 16, 2, 2, 64, device=DEV, dtype=BF16).unbind(2)):
        c_ext.write_kv_tokens(x[0].to(DEV), x[1].to(DEV), kc, vc, slots.to(DEV))
        for half, want in ((kc, x[0]), (vc, x[1])):
            cache = torch.zeros(64, 2, 64, dtype=BF16)
            cache[slots] = want
            assert _same(half, cache.view(4, 16, 2, 64))


# -- tokens that come from the cache itself -------------------------------------------------

@pytest.mark.parametrize("halves", [1, 2])
def test_tokens_move_within_their_cache(per_call_path, halves):
    """Each token to the next one's slot, all at once, from views of the cache."""
    g = _gen(3)
    blocks, T, H, D = 300, 16, 2, 64
    cache = torch.randn(2, blocks, T, H, D, generator=g).to(BF16)
    dev = cache.to(DEV)
    flat = dev.view(2, blocks * T, H, D)
    slots = torch.arange(blocks * T).roll(-1)
    if halves == 2:
        # and what was K becomes V
        c_ext.write_kv_tokens(flat[1], flat[0], dev[0], dev[1], slots.to(DEV))
        want = cache.flip(0)
    else:
        c_ext.write_kv_tokens(flat[0], None, dev[0], None, slots.to(DEV))
        want = cache
    want = want.reshape(2, blocks * T, H, D).roll(1, 1).view_as(cache)
    assert _same(dev[0], want[0])
    assert _same(dev[1], want[1] if halves == 2 else cache[1])


# -- starts, and other streams ------------------------------------------------------------

@pytest.mark.parametrize("first,last", [(0, 1 << 40), (-7, 0), (-(1 << 50), 1)])
@pytest.mark.parametrize("queries", [3, 40])
def test_starts_outside_the_rows_are_those_at_their_ends(first, last, queries):
    """`last`: how far behind the rows."""
    c = Case([100, 100], [queries, queries], index=torch.int64)
    starts = torch.tensor([first, queries, 2 * queries + last], device=DEV)
    out = torch.full((2 * queries, 8, 128), 3.0, device=DEV, dtype=BF16)
    c.check(c.run(query_starts=starts, out=out))


@pytest.mark.parametrize("queries", [1, 6, 50])
def test_calls_on_two_streams_at_once(queries):
    """Each with the weights and lse that it makes itself; so are those of replayed graphs."""
    cases = [Case([900, 70], [queries, 1], H=1, seed=1), Case([9000], [queries], H=1, G=8, seed=2)]
    streams = [torch.cuda.Stream() for _ in cases]
    state = []
    for c in cases:
        d = c.device()
        state.append((d, torch.zeros_like(d["query"]), torch.zeros(c.q.shape[:2], device=DEV),
                      c.w.to(DEV)))
    torch.cuda.synchronize()

    def got():
        torch.cuda.synchronize()
        return [tuple(t.cpu() for t in s[1:]) for s in state]
    for c, s, (d, out, lse, w) in zip(cases, streams, state):
        with torch.cuda.stream(s):
            c_ext.paged_attention(**d, out=out, lse=lse, weights=w)
    eager = got()
    for c, g in zip(cases, eager):
        c.check(g)
    graphs = []
    for c, s, (d, out, lse, w) in zip(cases, streams, state):
        before = c.w.to(DEV)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            w.copy_(before)
            c_ext.paged_attention(**d, out=out, lse=lse, weights=w)
        graphs.append((graph, before))
    for _ in range(3):
        for d, out, lse, w in state:
            out.zero_(), lse.zero_(), w.zero_()
        torch.cuda.synchronize()
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        for a, b in zip(got(), eager):
            assert all(_same(x, y) for x, y in zip(a, b))


# -- tables of no blocks -------------------------------------------------------------------

@pytest.mark.parametrize("wide", [0, 5])
def test_sequences_whose_tables_have_no_blocks(per_call_path, wide):
    """Nothing is seen, weighed or kept."""
    cache = torch.ones(4, 16, 2, 64, device=DEV, dtype=BF16)
    table = torch.zeros(3, 0, device=DEV, dtype=torch.int64)
    lens = torch.tensor([0, -1, 1], device=DEV)          # the last: more than its row holds
    w = torch.ones(3, 2, wide, device=DEV)
    out = c_ext.paged_attention(torch.ones(3, 4, 64, device=DEV, dtype=BF16), cache, cache, table,
                                lens, weights=w)
    assert (out[:2] == 0).all() and out[2].isnan().all() and (w == 1).all()
    new_weights = torch.full((3, 2, 7), 5.0, device=DEV)
    kept = c_ext.evict_kv_tokens(cache, None, w, table, lens, table, 9, 2, new_weights)
    assert kept.shape == (3, 2, 9) and (kept == -1).all()
    assert (new_weights[:2] == 0).all() and (new_weights[2] == 5).all()
    assert (cache == 1).all()
