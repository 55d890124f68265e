"""The 4-bit KV cache without a device: the oracle's pins, sizes and layouts, and
what the entry points refuse before any device work."""
import ctypes
import itertools

import numpy as np
import pytest
import torch

from flexkv_amd import _lib, c_ext
from flexkv_amd.common.storage import KVCacheLayout, KVCacheLayoutType

import mx4_oracle as mo


# -- the oracle ------------------------------------------------------------------

def test_oracle_reads_every_code_and_scale():
    codes = np.tile(np.arange(16, dtype=np.uint8), 2)
    for b in (0, 1, 126, 127, 128, 254):
        got = mo.decode(codes, np.array([b], np.uint8))
        want = [(-1.0 if c >= 8 else 1.0) * (0, .5, 1, 1.5, 2, 3, 4, 6)[c % 8] * 2.0 ** (b - 127)
                for c in codes]
        assert got.tolist() == want
    assert np.isnan(mo.decode(codes, np.array([255], np.uint8))).all()


@pytest.mark.parametrize("top,byte", [(1.0, 125), (1.75, 125), (np.nextafter(1.75, 2), 126),
                                      (1.99, 126), (2.0, 126), (6.0, 127), (7.0, 127),
                                      (7.01, 128), (0.0, 0), (2.0 ** -126, 0),
                                      (1.9 * 2.0 ** 127, 252)])
def test_oracle_scale_of_the_largest(top, byte):
    row = np.zeros(32)
    row[5] = -top
    assert mo.encode(row)[1].tolist() == [byte]


def test_oracle_rounds_ties_to_the_even_code():
    row = np.zeros(32)
    row[:9] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -2.5]
    codes, scales = mo.encode(row)
    assert scales.tolist() == [127]
    assert codes[:9].tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 12]


def test_oracle_error_is_within_one_scale_and_values_come_back():
    g = np.random.default_rng(3)
    x = g.standard_normal((50, 64)) * np.exp(3 * g.standard_normal((50, 1)))
    codes, scales = mo.encode(x)
    y = mo.decode(codes, scales)
    s = np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, -1)
    assert (np.abs(y - x) <= s).all()
    again = mo.encode(y)
    assert np.array_equal(mo.decode(*again), y)


def test_oracle_chunk_is_a_bijection():
    T, H, D = 16, 3, 64
    g = np.random.default_rng(4)
    chunk = g.integers(0, 256, c_ext.mx4_chunk_bytes(T, H, D), dtype=np.uint8)
    assert np.array_equal(mo.pack_chunk(*mo.unpack_chunk(chunk, T, H, D)), chunk)
    codes, scales = mo.unpack_chunk(chunk, T, H, D)
    h, t, d = 2, 5, 37
    assert codes[t, h, d] == chunk[(h * T + t) * D // 2 + d // 2] >> 4
    assert scales[t, h, d // 32] == chunk[T * H * D // 2 + (h * D // 32 + d // 32) * T + t]


# -- sizes and layouts --------------------------------------------------------------

def test_chunk_bytes():
    assert c_ext.mx4_chunk_bytes(16, 8, 128) == 16 * 8 * (64 + 4)
    for bad in ((8, 8, 128), (17, 8, 128), (0, 8, 128), (16, 0, 128), (16, 8, 100), (16, 8, 0)):
        with pytest.raises(ValueError):
            c_ext.mx4_chunk_bytes(*bad)


@pytest.mark.parametrize("kind,mla", itertools.product(KVCacheLayoutType, (False, True)))
def test_layout_in_four_bits(kind, mla):
    wide = KVCacheLayout(kind, 5, 7, 32, 2, 96, is_mla=mla)
    lay = wide.mx4()
    chunk, kv, layer, block = lay.byte_strides(torch.uint8)
    assert chunk == c_ext.mx4_chunk_bytes(32, 2, 96) and chunk % 16 == 0
    assert lay.get_total_elements() == chunk * 5 * 7 * (1 if mla else 2)
    assert (kv * 64, layer * 64, block * 64) == tuple(
        s * 17 for s in wide.byte_strides(torch.bfloat16)[1:])
    assert wide.head_size == 96


def test_layout_in_four_bits_refuses_what_does_not_divide():
    for tokens, dim in ((16, 80), (8, 128)):
        with pytest.raises(ValueError):
            KVCacheLayout(KVCacheLayoutType.BLOCKWISE, 2, 2, tokens, 2, dim).mx4()


# -- refusals of the C entries -------------------------------------------------------

def _blocks(fn="fkv_quantize_kv_blocks", **kw):
    ids = np.array([0, 1], dtype=np.int64)
    buf = np.zeros(1 << 16, dtype=np.uint8)
    base = (buf.ctypes.data + 255) & ~255
    ptrs = (ctypes.c_void_p * 1)(base)
    args = dict(num_blocks=2, start=0, layers=1, gids=ids.ctypes.data, ptrs=ptrs, gkv=4096,
                gblk=4096, mids=ids.ctypes.data, mx=base, mkv=1088, mlay=0, mblk=1088, tokens=16,
                heads=1, dim=128, dtype=0, stream=None, mla=1)
    args.update(kw)
    rc = getattr(_lib.load(), fn)(*args.values())
    del buf
    return rc, _lib.last_error()


@pytest.mark.parametrize("fn", ["fkv_quantize_kv_blocks", "fkv_dequantize_kv_blocks"])
def test_block_calls_refuse(fn):
    neg = np.array([0, -2], dtype=np.int64)
    for kw, word in ((dict(num_blocks=-1), "negative count"), (dict(start=-1), "negative count"),
                     (dict(layers=-3), "negative count"), (dict(gids=None), "null"),
                     (dict(mids=None), "null"), (dict(ptrs=None), "null"), (dict(mx=None), "null"),
                     (dict(tokens=8), "tokens_per_block"), (dict(tokens=0), "tokens_per_block"),
                     (dict(tokens=24), "tokens_per_block"), (dict(tokens=8192), "tokens_per_block"),
                     (dict(heads=0), "num_heads"), (dict(heads=5000), "num_heads"),
                     (dict(dim=80), "head_size"), (dict(dim=0), "head_size"),
                     (dict(dim=2048), "head_size"), (dict(dtype=3), "dtype"),
                     (dict(dtype=-1), "dtype"), (dict(gblk=4104), "multiples of 16"),
                     (dict(mkv=-16), "multiples of 16"), (dict(mblk=1090), "multiples of 16"),
                     (dict(gids=neg.ctypes.data), "negative block id"),
                     (dict(mids=neg.ctypes.data), "negative block id"),
                     ({}, "not pinned host or device")):
        rc, msg = _blocks(fn, **kw)
        assert rc == 1 and word in msg, (kw, rc, msg)
    assert _blocks(fn, num_blocks=0)[0] == 0
    assert _blocks(fn, layers=0)[0] == 0


def _tokens(**kw):
    args = dict(n=4, key=4096, kts=256, khs=256, value=8192, vts=256, vhs=256, slots=4096, is64=1,
                mx=4096, mkv=1088, mblk=2176, blocks=3, tokens=16, heads=1, dim=128, dtype=0,
                stream=None)
    args.update(kw)
    return _lib.load().fkv_quantize_kv_tokens(*args.values()), _lib.last_error()


def test_token_calls_refuse():
    for kw, word in ((dict(n=-1), "negative count"), (dict(tokens=20), "tokens_per_block"),
                     (dict(dim=72), "head_size"), (dict(heads=0), "num_heads"),
                     (dict(dtype=7), "dtype"), (dict(mx=None), "null"), (dict(blocks=0), "num_mx"),
                     (dict(blocks=1 << 31), "num_mx"), (dict(mx=4100), "multiples of 16"),
                     (dict(mblk=100), "multiples of 16"), (dict(mkv=-32), "multiples of 16"),
                     ({}, "not device memory")):
        rc, msg = _tokens(**kw)
        assert rc == 1 and word in msg, (kw, rc, msg)


def _attend(**kw):
    args = dict(query=4096, out=8192, lse=None, query_row_stride_bytes=256,
                query_head_stride_bytes=256, out_row_stride_bytes=256, out_head_stride_bytes=256,
                mx_ptr=4096, mx_kv_stride_bytes=1088, mx_block_stride_bytes=2176,
                num_mx_blocks=3, block_table=4096, seq_lens=4096, query_starts=None,
                table_row_stride=2, table_width=2, batch=2, num_queries=2, tokens_per_block=16,
                num_heads=1, group_size=1, head_size=128, dtype=0, causal=1, scale=1.0)
    args.update(kw)
    a = _lib.Mx4AttentionArgs(**args)
    return _lib.load().fkv_mx4_attention(a, None), _lib.last_error()


def test_attention_refuses():
    assert _lib.load().fkv_mx4_attention(None, None) == 1
    for kw, word in ((dict(batch=-1), "negative count"), (dict(num_queries=-1), "negative count"),
                     (dict(tokens_per_block=8), "tokens_per_block"),
                     (dict(head_size=96), "head_size"), (dict(head_size=576), "head_size"),
                     (dict(dtype=2), "dtype"), (dict(dtype=9), "dtype"),
                     (dict(group_size=0), "group_size"), (dict(group_size=5000), "group_size"),
                     (dict(num_heads=0), "num_heads"),
                     (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
                     (dict(table_width=-1), "table_width"),
                     (dict(table_width=1 << 27), "table_width"),
                     (dict(num_queries=1 << 30), "too many"),
                     (dict(num_queries=1), "one query each"),
                     (dict(query=None), "null"), (dict(out=None), "null"),
                     (dict(seq_lens=None), "null"), (dict(block_table=None), "null"),
                     (dict(query=4104), "multiples of 16"), (dict(out=8200), "multiples of 16"),
                     (dict(query_row_stride_bytes=250), "multiples of 16"),
                     (dict(out_head_stride_bytes=8), "multiples of 16"),
                     (dict(mx_ptr=None), "null"), (dict(num_mx_blocks=0), "num_mx"),
                     (dict(mx_block_stride_bytes=17), "multiples of 16"),
                     ({}, "not device memory")):
        rc, msg = _attend(**kw)
        assert rc == 1 and word in msg, (kw, rc, msg)
    assert _attend(batch=0, num_queries=0)[0] == 0
    assert _attend(num_queries=0, query_starts=4096)[0] == 0


# -- refusals of the Python entries --------------------------------------------------

def test_python_entries_refuse_host_tensors_and_types():
    ids = torch.zeros(2, dtype=torch.int64)
    mx = torch.zeros(4096, dtype=torch.uint8)
    with pytest.raises(TypeError):
        c_ext.quantize_kv_blocks(ids.int(), ids, 0, 0, ids, mx, 0, 0, 0, 16, 1, 128,
                                 torch.bfloat16)
    with pytest.raises(RuntimeError, match="2 ids"):
        c_ext.quantize_kv_blocks(ids, ids, 0, 0, ids[:1], mx, 0, 0, 0, 16, 1, 128, torch.bfloat16)
    with pytest.raises(TypeError, match="elements"):
        c_ext.dequantize_kv_blocks(ids, ids, 0, 0, ids, mx, 0, 0, 0, 16, 1, 128, torch.int8)
    with pytest.raises(TypeError):
        c_ext.quantize_kv_blocks(ids, ids, 0, 0, ids, None, 0, 0, 0, 16, 1, 128, torch.bfloat16)
    x = torch.zeros(2, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="device tensor"):
        c_ext.quantize_kv_tokens(x, x, mx, ids)
    with pytest.raises(RuntimeError, match="device tensor"):
        c_ext.mx4_attention(x, mx, 1, ids, ids)
    with pytest.raises(TypeError):
        c_ext.mx4_attention(None, mx, 1, ids, ids)


def test_python_entries_refuse_inputs_that_require_gradients():
    x = torch.zeros(2, 1, 128, dtype=torch.bfloat16, requires_grad=True)
    plain, ids = torch.zeros(2, 1, 128, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    mx = torch.zeros(4096, dtype=torch.uint8)
    for call in (lambda: c_ext.quantize_kv_tokens(x, plain, mx, ids),
                 lambda: c_ext.mx4_attention(x, mx, 1, ids, ids)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="device tensor"):
            call()


def test_overlap_of_two_views_is_that_of_their_bytes():
    """Every pair of views of a small buffer, strides alike or not, against sets of bytes."""
    g = np.random.default_rng(5)
    buf = torch.zeros(400, dtype=torch.bfloat16)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        rows, heads, dim = (int(v) for v in g.integers(1, 5, 3))

        def view(strides):
            return buf.as_strided((rows, heads, dim), (*strides, 1), int(g.integers(0, 120)))
        strides = [tuple(int(v) for v in g.integers(0, 30, 2)) for _ in range(2)]
        x, y = view(strides[0]), view(strides[int(g.integers(0, 2))])

        def touched(t):
            return {t.storage_offset() + i * t.stride(0) + j * t.stride(1) + k
                    for i in range(rows) for j in range(heads) for k in range(dim)}
        want = bool(touched(x) & touched(y))
        assert c_ext._overlap(x, y) is want, (x.shape, x.stride(), y.stride())
        seen[want] += 1
    assert min(seen.values()) > 500
    assert not c_ext._overlap(buf[:0].view(0, 1, 4), buf[:0].view(0, 1, 4))


def test_calls_of_more_threads_than_a_launch_has_are_refused():
    """2^32 and more: 2^24 workgroups of 256."""
    lib, need = _lib.load(), ctypes.c_size_t()

    def attend(queries, heads, dim=128):
        a = _lib.Mx4AttentionArgs(query_starts=4096, batch=1, num_queries=queries, table_width=64,
                                  tokens_per_block=16, num_heads=heads, group_size=48,
                                  head_size=dim, scale=1.0)
        return lib.fkv_mx4_attention_workspace(a, need), _lib.last_error()
    # a tile of 48 rows for each query and one more, in eights: 2^14 - 8 tiles, then 2^14
    assert attend((1 << 14) - 9, 1024)[0] == 0
    for queries, heads in (((1 << 14) - 8, 1024), (1 << 20, 1024), (1 << 22, 5)):
        rc, msg = attend(queries, heads)
        assert rc == 1 and "too many" in msg
    for n in ((1 << 30) - 63, 1 << 30, (1 << 31) - 1):
        rc, msg = _tokens(n=n, dim=32, value=None)
        assert rc == 1 and "too many" in msg
    rc, msg = _tokens(n=(1 << 30) - 64, dim=32, value=None)
    assert rc == 1 and "not device memory" in msg
