"""The operators on a paged cache without a device: the oracle's pins, and what the entry
points refuse before any device work."""
import ctypes
import math

import numpy as np
import pytest
import torch

from flexkv_amd import _lib, c_ext

import paged_oracle as po


# -- the oracle ------------------------------------------------------------------

def test_oracle_attention_is_the_formula():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, 8, generator=g).double() for n in (3, 5, 5))
    out, lse, p, mags = po.attention(q, k, v, 0.4, torch.tensor([5, 2, 0]))
    for r, n in enumerate((5, 2)):
        e = [math.exp(0.4 * float(q[r] @ k[t])) for t in range(n)]
        assert abs(float(lse[r]) - math.log(sum(e))) < 1e-12
        for t in range(n):
            assert abs(float(p[r, t]) - e[t] / sum(e)) < 1e-12
        want = sum(e[t] / sum(e) * v[t] for t in range(n))
        assert (out[r] - want).abs().max() < 1e-12
        assert abs(float(mags[r]) - max(0.4 * float(q[r].abs() @ k[t].abs())
                                        for t in range(n))) < 1e-12
    assert (out[2] == 0).all() and lse[2] == -math.inf and (p[2] == 0).all()


def test_oracle_leaves_out_what_a_row_does_not_see():
    q, k = torch.ones(2, 4), torch.ones(3, 4)
    v = torch.ones(3, 4)
    v[2], k[2] = math.nan, math.inf
    out, lse, p, _ = po.attention(q, k, v, 1.0, torch.tensor([2, 1]))
    assert ((out - 1).abs() < 1e-12).all() and lse.isfinite().all() and p.isfinite().all()


@pytest.mark.parametrize("w,n,budget,recent,want", [
    ([5, 1, 4, 2, 3], 5, 3, 0, [0, 2, 4]),
    ([5, 1, 4, 2, 3], 5, 3, 2, [0, 3, 4]),
    ([5, 1, 4, 2, 3], 5, 3, 3, [2, 3, 4]),
    ([5, 1, 4, 2, 3], 5, 9, 3, [0, 1, 2, 3, 4]),
    ([1, 1, 1, 1], 4, 2, 0, [0, 1]),
    ([1, 1, 1, 1], 4, 2, 1, [0, 3]),
    ([0.0, -0.0, 0.0], 3, 2, 0, [0, 1]),
    ([2, math.nan, math.inf, -math.inf], 4, 2, 0, [1, 2]),
    ([2, 3], 0, 2, 0, []),
])
def test_oracle_choice(w, n, budget, recent, want):
    assert po.choose(w, n, budget, recent) == want


def test_oracle_rows():
    cache = np.arange(3 * 2 * 1 * 1).reshape(3, 2, 1, 1)
    assert po.rows_of(cache, [2, 0], 3)[:, 0, 0].tolist() == [4, 5, 0]


# -- refusals of the C entries -------------------------------------------------------

LAYER = dict(key=4096, value=8192, key_block_stride_bytes=4096, key_token_stride_bytes=256,
             key_head_stride_bytes=256, value_block_stride_bytes=4096,
             value_token_stride_bytes=256, value_head_stride_bytes=256, num_blocks=3,
             tokens_per_block=16, num_heads=1, head_size=128, dtype=0)
BAD_LAYERS = [
    (dict(tokens_per_block=0), "tokens_per_block"),
    (dict(tokens_per_block=1 << 21), "tokens_per_block"), (dict(num_heads=0), "num_heads"),
    (dict(num_heads=5000), "num_heads"), (dict(head_size=0), "head_size"),
    (dict(head_size=2048), "head_size"), (dict(head_size=100), "head_size"),
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(num_blocks=0), "num_blocks"),
    (dict(num_blocks=1 << 31), "num_blocks"), (dict(key=None), "null"),
    (dict(key=4100), "multiple of 16"), (dict(key_block_stride_bytes=-16), "multiples of 16"),
    (dict(key_token_stride_bytes=8), "multiples of 16"), ({}, "not device memory")]


def _layer(kw):
    return _lib.PagedLayer(**{**LAYER, **kw})


def _write(layer={}, **kw):
    args = dict(n=4, key=4096, kts=256, khs=256, value=8192, vts=256, vhs=256, slots=4096, is64=1,
                stream=None)
    args.update(kw)
    return _lib.load().fkv_write_kv_tokens(_layer(layer), *args.values()), _lib.last_error()


def test_token_calls_refuse():
    assert _lib.load().fkv_write_kv_tokens(None, 1, None, 0, 0, None, 0, 0, None, 0, None) == 1
    for layer, word in BAD_LAYERS:
        rc, msg = _write(layer)
        assert rc == 1 and word in msg, (layer, rc, msg)
    rc, msg = _write(n=-1)
    assert rc == 1 and "negative count" in msg


def _attend(layer={}, **kw):
    args = dict(layer=_layer(layer), query=4096, out=8192, lse=None, query_row_stride_bytes=256,
                query_head_stride_bytes=256, out_row_stride_bytes=256, out_head_stride_bytes=256,
                block_table=4096, seq_lens=4096, query_starts=None, table_row_stride=2,
                table_width=2, batch=2, num_queries=2, group_size=1, causal=1, scale=1.0)
    args.update(kw)
    a = _lib.PagedAttentionArgs(**args)
    return _lib.load().fkv_paged_attention(a, None), _lib.last_error()


def test_attention_refuses():
    assert _lib.load().fkv_paged_attention(None, None) == 1
    assert _lib.load().fkv_paged_attention_workspace(None, None) == 1
    for layer, word in BAD_LAYERS + [(dict(head_size=96), "head_size"),
                                     (dict(head_size=512), "head_size"), (dict(dtype=2), "dtype"),
                                     (dict(value=None), "null"),
                                     (dict(value_head_stride_bytes=40), "multiples of 16")]:
        rc, msg = _attend(layer)
        # a host pointer is only found out behind it
        assert rc == 1 and (word in msg or "not device memory" in msg), (layer, rc, msg)
    for kw, word in ((dict(batch=-1), "negative count"), (dict(num_queries=-1), "negative count"),
                     (dict(group_size=0), "group_size"), (dict(group_size=5000), "group_size"),
                     (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
                     (dict(table_width=-1), "table_width"),
                     (dict(table_width=1 << 27), "table_width"),
                     (dict(num_queries=1 << 30), "too many"),
                     (dict(num_queries=1), "one query each"),
                     (dict(query=None), "null"), (dict(out=None), "null"),
                     (dict(seq_lens=None), "null"), (dict(block_table=None), "null"),
                     (dict(query=4104), "multiples of 16"), (dict(out=8200), "multiples of 16"),
                     (dict(query_row_stride_bytes=250), "multiples of 16"),
                     (dict(out_head_stride_bytes=8), "multiples of 16"),
                     (dict(weights=4096, weights_width=31), "do not hold"),
                     (dict(weights=4096, weights_width=32, batch=1 << 17, num_queries=1 << 17),
                      "too many")):
        rc, msg = _attend(**kw)
        assert rc == 1 and word in msg, (kw, rc, msg)
    assert _attend(batch=0, num_queries=0)[0] == 0
    assert _attend(num_queries=0, query_starts=4096)[0] == 0


def test_calls_of_more_threads_than_a_launch_has_are_refused():
    lib, need = _lib.load(), ctypes.c_size_t()

    def attend(queries, heads, group, **kw):
        a = _lib.PagedAttentionArgs(layer=_layer(dict(num_heads=heads)), query_starts=4096,
                                    batch=1, num_queries=queries, table_width=64,
                                    group_size=group, scale=1.0, **kw)
        return lib.fkv_paged_attention_workspace(a, need), _lib.last_error()
    assert attend(1000, 8, 4)[0] == 0
    rc, msg = attend(1 << 24, 1024, 48)
    assert rc == 1 and "too many" in msg
    rc, msg = _write(dict(num_heads=1024, head_size=1024), n=(1 << 31) - 1)
    assert rc == 1


def _evict(layer={}, **kw):
    args = dict(layer=_layer(layer), weights=4096, new_weights=None, weights_seq_stride=32,
                weights_head_stride=32, block_table=4096, new_table=4096, seq_lens=4096,
                table_row_stride=2, new_table_row_stride=2, kept=4096, table_width=2,
                new_table_width=1, batch=2, budget=9, recent=2, weights_width=32)
    args.update(kw)
    return _lib.load().fkv_evict_kv_tokens(_lib.EvictArgs(**args), None), _lib.last_error()


def test_eviction_refuses():
    assert _lib.load().fkv_evict_kv_tokens(None, None) == 1
    for layer, word in BAD_LAYERS:
        rc, msg = _evict(layer)
        assert rc == 1 and (word in msg or "not device memory" in msg or "do not hold" in msg), (
            layer, rc, msg)
    for kw, word in ((dict(batch=-1), "negative count"), (dict(budget=0), "budget"),
                     (dict(budget=(1 << 28) + 1), "budget"), (dict(recent=10), "recent"),
                     (dict(recent=-1), "recent"), (dict(table_width=-1), "table_width"),
                     (dict(table_width=1 << 27), "table_width"),
                     (dict(new_table_width=0), "do not hold"),
                     (dict(budget=17), "do not hold"), (dict(weights_width=31), "do not hold"),
                     (dict(new_weights=4096, new_weights_width=8), "do not hold"),
                     (dict(batch=(1 << 21) + 1), "too many"), (dict(weights=None), "null"),
                     (dict(kept=None), "null"), (dict(seq_lens=None), "null"),
                     (dict(block_table=None), "null"), (dict(new_table=None), "null")):
        rc, msg = _evict(**kw)
        assert rc == 1 and word in msg, (kw, rc, msg)
    assert _evict(batch=0)[0] == 0


def test_workspace_of_an_eviction():
    lib, need = _lib.load(), ctypes.c_size_t(1)

    def of(**kw):
        args = dict(layer=_layer({}), table_width=2, new_table_width=4096, batch=2, budget=9,
                    recent=2, weights_width=1 << 20, new_weights_width=1 << 20)
        args.update(kw)
        rc = lib.fkv_evict_kv_tokens_workspace(_lib.EvictArgs(**args), need)
        return rc, need.value
    assert lib.fkv_evict_kv_tokens_workspace(None, need) == 1
    assert of() == (0, 0) and of(batch=0, table_width=4096) == (0, 0)
    assert of(budget=0, table_width=4096) == (1, 0)
    long = of(table_width=4096)
    assert long[0] == 0 and long[1] > 0
    kept = of(table_width=4096, new_weights=4096)
    heads = 2 * _layer({}).num_heads
    assert kept == (0, long[1] + heads * 9 * 4)
    # no more than many sequences' own workgroups need
    assert of(table_width=4096, batch=512) == (0, 0)


# -- refusals of the Python entries --------------------------------------------------

def test_python_entries_refuse_host_tensors_and_gradients(per_call_path):
    x = torch.zeros(2, 1, 128, dtype=torch.bfloat16)
    cache = torch.zeros(3, 16, 1, 128, dtype=torch.bfloat16)
    ids = torch.zeros(2, dtype=torch.int64)
    table = torch.zeros(2, 1, dtype=torch.int64)
    w = torch.zeros(2, 1, 16)
    with pytest.raises(RuntimeError, match="device tensor"):
        c_ext.write_kv_tokens(x, x, cache, cache, ids)
    with pytest.raises(RuntimeError, match="device tensor"):
        c_ext.paged_attention(x, cache, cache, table, ids)
    with pytest.raises(RuntimeError, match="device tensor"):
        c_ext.evict_kv_tokens(cache, cache, w, table, ids, table, 4)
    for call in (lambda: c_ext.write_kv_tokens(None, x, cache, cache, ids),
                 lambda: c_ext.paged_attention(None, cache, cache, table, ids),
                 lambda: c_ext.evict_kv_tokens(None, cache, w, table, ids, table, 4)):
        with pytest.raises(TypeError):
            call()
    leaf = x.clone().requires_grad_()
    for call in (lambda: c_ext.write_kv_tokens(leaf, x, cache, cache, ids),
                 lambda: c_ext.paged_attention(leaf, cache, cache, table, ids)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="device tensor"):
            call()
