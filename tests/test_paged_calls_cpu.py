"""Calls on a paged cache that have to be refused, each for its own reason, without a device."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

from flexkv_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_overlapping_caches_are_told_from_others(tmp_path):
    """Builds tests/native/overlap_check.cpp with g++ against flexkv_amd/csrc/kv_overlap.h."""
    exe = tmp_path / "overlap_check"
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "flexkv_amd", "csrc"),
           os.path.join(ROOT, "tests", "native", "overlap_check.cpp"), "-o", str(exe)]
    build = subprocess.run(cmd, capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "FAIL" not in res.stdout, res.stdout + res.stderr
    assert res.stdout.count("ok:") == 20


# -- refusals of the C entries, by their own words ------------------------------------------

# pointers in no one's memory: what is refused behind all other checks of a layer
LAYER = dict(key=1 << 20, value=1 << 24, key_block_stride_bytes=4096, key_token_stride_bytes=256,
             key_head_stride_bytes=256, value_block_stride_bytes=4096,
             value_token_stride_bytes=256, value_head_stride_bytes=256, num_blocks=3,
             tokens_per_block=16, num_heads=1, head_size=128, dtype=0)
BAD_SIZES = [
    (dict(tokens_per_block=0), "tokens_per_block must be in"),
    (dict(tokens_per_block=-3), "tokens_per_block must be in"),
    (dict(tokens_per_block=(1 << 20) + 1), "tokens_per_block must be in"),
    (dict(num_heads=0), "num_heads must be in"), (dict(num_heads=1025), "num_heads must be in"),
    (dict(head_size=0), "head_size must be a multiple of 16 bytes"),
    (dict(head_size=1032), "head_size must be a multiple of 16 bytes"),
    (dict(head_size=100), "head_size must be a multiple of 16 bytes"),
    (dict(head_size=-8), "head_size must be a multiple of 16 bytes"),
    (dict(dtype=3), "dtype must be FKV"), (dict(dtype=-1), "dtype must be FKV"),
    (dict(num_blocks=0), "num_blocks must be in"),
    (dict(num_blocks=1 << 31), "num_blocks must be in")]
BAD_MEMORY = [
    (dict(key=None), "null cache pointer"),
    (dict(key=(1 << 20) + 8), "key cache's pointer must be a multiple of 16"),
    (dict(value=(1 << 24) + 4), "value cache's pointer must be a multiple of 16"),
    *((dict([(f"{half}_{what}_stride_bytes", bad)]),
       f"the {half} cache's strides must be non-negative multiples of 16")
      for half in ("key", "value") for what in ("block", "token", "head") for bad in (-16, 24)),
    ({}, "key cache.*is not device memory")]


def _refused(rc, word):
    msg = _lib.last_error()
    assert rc == 1 and re.search(word, msg), (word, rc, msg)


def _layer(kw):
    return _lib.PagedLayer(**{**LAYER, **kw})


def _write(layer, n=4, key=4096, value=8192, stride=256, slots=4096):
    return _lib.load().fkv_write_kv_tokens(_layer(layer), n, key, stride, 256, value, 256, 256,
                                           slots, 1, None)


def _attend(layer, call=True, **kw):
    args = dict(layer=_layer(layer), query=4096, out=8192, lse=None, query_row_stride_bytes=256,
                query_head_stride_bytes=256, out_row_stride_bytes=256, out_head_stride_bytes=256,
                block_table=4096, seq_lens=4096, query_starts=None, table_row_stride=2,
                table_width=2, batch=2, num_queries=2, group_size=1, causal=1, scale=1.0)
    args = _lib.PagedAttentionArgs(**{**args, **kw})
    lib = _lib.load()
    return lib.fkv_paged_attention(args, None) if call else \
        lib.fkv_paged_attention_workspace(args, ctypes.c_size_t())


def _evict(layer, call=True, **kw):
    args = dict(layer=_layer(layer), weights=4096, new_weights=None, weights_seq_stride=32,
                weights_head_stride=32, block_table=4096, new_table=4096, seq_lens=4096,
                table_row_stride=2, new_table_row_stride=2, kept=4096, table_width=2,
                new_table_width=1, batch=2, budget=9, recent=2, weights_width=32)
    args = _lib.EvictArgs(**{**args, **kw})
    lib = _lib.load()
    return lib.fkv_evict_kv_tokens(args, None) if call else \
        lib.fkv_evict_kv_tokens_workspace(args, ctypes.c_size_t())


@pytest.mark.parametrize("layer,word", BAD_SIZES, ids=str)
def test_a_layer_of_sizes_that_cannot_be_is_refused_by_name(layer, word):
    _refused(_write(layer), word)
    for call in (True, False):
        _refused(_attend(layer, call), word)
        _refused(_evict(layer, call), word)


@pytest.mark.parametrize("layer,word", BAD_MEMORY, ids=str)
def test_a_layer_of_memory_that_cannot_be_is_refused_by_name(layer, word):
    _refused(_write(layer), word)
    _refused(_attend(layer), word)
    _refused(_evict(layer), word)


@pytest.mark.parametrize("layer,word", [
    (dict(head_size=96), "attention takes a head_size of 64, 128 or 256"),
    (dict(head_size=512), "attention takes a head_size of 64, 128 or 256"),
    (dict(dtype=2), "attention takes a bf16 or fp16 cache"),
    (dict(value=None), "null cache pointer")], ids=str)
def test_layers_that_attention_does_not_take(layer, word):
    _refused(_attend(layer), word)
    assert _evict(layer, False) == 0


def test_calls_of_more_threads_than_a_launch_has():
    """Each bound from both sides."""
    wide = dict(num_heads=1024, head_size=1024)          # 2^17 pieces of 16 bytes a token
    _refused(_write(wide, n=1 << 14), "16384 tokens of 1024 heads of 1024 are too many")
    _refused(_write(wide, n=(1 << 31) - 1), "are too many for one call")
    _refused(_write(wide, n=(1 << 14) - 1), "not device memory")
    pairs = dict(num_heads=1024)
    assert _evict(pairs, False, batch=1 << 11) == 0
    _refused(_evict(pairs, False, batch=(1 << 11) + 1), "2049 sequences of 1024 heads are too many")
    # tiles of 128 rows, one a sequence more, in rounds of 8
    many = dict(num_queries=(1 << 29) - 2048, batch=1, query_starts=4096)
    assert _attend({}, False, **many) == 0
    _refused(_attend({}, False, **{**many, "num_queries": (1 << 29) - 1024}),
             "536869888 queries of 1 K/V heads are too many")
    _refused(_attend(pairs, False, **many), "536868864 queries of 1024 K/V heads are too many")
    _refused(_attend({}, False, **{**many, "group_size": 3}), "536868864 queries of 3 heads a K/V")


def test_an_eviction_from_tables_of_no_blocks_needs_no_weights():
    none = dict(table_width=0, new_table_width=0, weights_width=0)
    assert _evict({}, False, **none) == 0
    for kw in ({}, dict(weights=None), dict(weights=None, block_table=None, new_table=None)):
        _refused(_evict({}, **none, **kw), "not device memory")
    for kw in (dict(seq_lens=None), dict(kept=None)):
        _refused(_evict({}, **none, **kw), "null pointer argument")
    for kw in (dict(weights=None), dict(block_table=None), dict(new_table=None)):
        _refused(_evict({}, **kw), "null pointer argument")


def test_keys_are_dealt_out_while_their_steps_stay_in_32_bits():
    """The steps of 32 tokens of all tiles, and with them up to 256 workgroups."""
    lib, need = _lib.load(), ctypes.c_size_t()

    def workspace(blocks):
        # groups of 32 heads of 256 elements: two tiles a sequence
        layer = _layer(dict(head_size=256, tokens_per_block=32))
        a = _lib.PagedAttentionArgs(layer=layer, batch=231, num_queries=231, group_size=32,
                                    table_width=blocks, scale=1.0)
        assert lib.fkv_paged_attention_workspace(a, need) == 0
        return need.value
    most = (2 ** 31 - 1 - 256) // 462
    assert workspace(2000) == workspace(most) > 0
    for blocks in (most + 1, (2 ** 31 - 1) // 462, (2 ** 31 - 1) // 462 + 1):
        assert workspace(blocks) == 0


@pytest.mark.parametrize("scale", [3e38, -3e38, float("inf"), float("nan")])
def test_a_scale_that_is_infinite_in_units_of_log_2_is_refused(scale):
    for call in (True, False):
        _refused(_attend({}, call, scale=scale), "scale must be finite")
    for finite in (2.0 ** 127, -(2.0 ** 127), 2.0 ** -149, 0.0):
        assert _attend({}, False, scale=finite) == 0
