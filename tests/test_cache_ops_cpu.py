"""Refusals of the cache operators (chunk attention, windowed decode
attention, eviction): every bad size, count or alignment is answered with
SKB_ERR_ARG before anything touches a GPU, so they are checked without one."""

from __future__ import annotations

import pytest

A = 1 << 20  # stands for a 256-byte aligned device address; nothing reads it


@pytest.fixture(scope="module")
def lib():
    from soraku_tts_b200 import _lib
    from soraku_tts_b200.build import build

    build()
    return _lib


CHUNK = dict(qkv=A, tokens=5, rows=2, n_heads=16, n_kv_heads=8, head_dim=128, q_norm=A, k_norm=A, eps=1e-6, rope_cos=A,
             rope_sin=A, max_pos=64, chunk_start=A, max_chunk=4, cached=A, pos=A, kv_pool=A, page_table=A, max_pages=4,
             page_size=16, n_pages=9, window=0, sinks=0, mass=None, work=A, work_bytes=1 << 40, out=A, stream=None)
DECODE = {k: v for k, v in CHUNK.items() if k not in ("tokens", "chunk_start", "max_chunk")}
EVICT = dict(mass=A, cached=A, rows=2, n_kv_heads=8, head_dim=128, kv_pool=A, page_table=A, max_pages=4, page_size=16,
             n_pages=9, budget=32, sinks=4, recent=8, kept=A, mass_out=2 * A, cached_out=2 * A, stream=None)

ATTN_BAD = [("q_norm", None), ("k_norm", None), ("rope_cos", None), ("rope_sin", None), ("cached", None), ("pos", None),
            ("kv_pool", None), ("page_table", None), ("qkv", None), ("out", None), ("head_dim", 64), ("n_heads", 0),
            ("n_heads", 17), ("n_heads", 40), ("n_kv_heads", 0), ("rows", -1), ("rows", 65536), ("max_pos", 0),
            ("max_pages", 0), ("max_pages", 1 << 27), ("page_size", 0), ("page_size", 48), ("n_pages", 0),
            ("window", -1), ("sinks", -1), ("sinks", 4), ("qkv", A + 4), ("out", A + 4), ("kv_pool", A + 8),
            ("rope_cos", A + 4), ("rope_sin", A + 4), ("q_norm", A + 4), ("k_norm", A + 4)]


@pytest.mark.parametrize("name,value", ATTN_BAD + [("chunk_start", None), ("tokens", -1), ("max_chunk", -1),
                                                   ("work", None), ("work", A + 16), ("work_bytes", 0)])
def test_chunk_attention_refuses(lib, name, value):
    args = dict(CHUNK, **{name: value})
    assert lib.lib().skb_chunk_attention(*args.values()) == lib.SKB_ERR_ARG
    assert "chunk_attention" in lib.last_error()


@pytest.mark.parametrize("name,value", ATTN_BAD)
def test_window_decode_attention_refuses(lib, name, value):
    args = dict(DECODE, **{name: value})
    assert lib.lib().skb_window_decode_attention(*args.values()) == lib.SKB_ERR_ARG
    assert "window_decode_attention" in lib.last_error()


@pytest.mark.parametrize("change", [dict(work=None), dict(work_bytes=16)])
def test_window_decode_attention_with_mass_needs_its_workspace(lib, change):
    args = dict(DECODE, mass=A, **change)
    assert lib.lib().skb_window_decode_attention(*args.values()) == lib.SKB_ERR_ARG
    assert "workspace" in lib.last_error()


@pytest.mark.parametrize("change", [
    {n: None} for n in ("mass", "cached", "kv_pool", "page_table", "kept", "mass_out", "cached_out")] + [
    dict(head_dim=64), dict(rows=-1), dict(rows=65536), dict(n_kv_heads=0), dict(max_pages=0), dict(max_pages=1 << 27),
    dict(page_size=24), dict(page_size=0), dict(n_pages=0), dict(budget=0), dict(sinks=-1), dict(recent=-1),
    dict(sinks=30, recent=3), dict(sinks=2**31 - 1, recent=2**31 - 1), dict(mass_out=A), dict(cached_out=A),
    dict(kv_pool=A + 4)])
def test_evict_cache_refuses(lib, change):
    args = dict(EVICT, **change)
    assert lib.lib().skb_evict_cache(*args.values()) == lib.SKB_ERR_ARG
    assert "evict_cache" in lib.last_error()


@pytest.mark.parametrize("offset", [4, 8, 16, 48])
def test_chunk_attention_wants_a_pool_at_32_bytes(lib, offset):
    """Its loads of cached rows are 32 bytes wide; even a call without work says so."""
    for change in ({}, dict(tokens=0), dict(rows=0)):
        args = dict(CHUNK, kv_pool=A + offset, **change)
        assert lib.lib().skb_chunk_attention(*args.values()) == lib.SKB_ERR_ARG
        assert "kv_pool" in lib.last_error()


def test_no_rows_or_no_tokens_is_no_work(lib):
    L = lib.lib()
    assert L.skb_chunk_attention(*dict(CHUNK, rows=0, qkv=None, out=None).values()) == lib.SKB_OK
    assert L.skb_chunk_attention(*dict(CHUNK, tokens=0, qkv=None, out=None).values()) == lib.SKB_OK
    assert L.skb_window_decode_attention(*dict(DECODE, rows=0, qkv=None, out=None).values()) == lib.SKB_OK
    assert L.skb_evict_cache(*dict(EVICT, rows=0).values()) == lib.SKB_OK


def test_workspace_sizes(lib):
    L = lib.lib()
    assert L.skb_chunk_attention_workspace(-1, 2, 4, 16, 8, 4, 16, 9, 0, 0, 0) == -1
    assert L.skb_chunk_attention_workspace(5, 2, 4, 16, 8, 0, 16, 9, 0, 0, 0) == -1
    assert L.skb_window_decode_workspace(2, 16, 4, 16, 0, 0, 0) == 0
    assert L.skb_window_decode_workspace(2, 16, 4, 16, 0, 0, 1) == 2 * 16 * 64 * 4
    assert L.skb_window_decode_workspace(2, 16, 4, 16, 8, 4, 1) == 2 * 16 * 12 * 4
    assert L.skb_window_decode_workspace(2, 16, 0, 16, 8, 4, 1) == -1
    # sizes that pass 32 bits are counted in 64
    big = L.skb_chunk_attention_workspace(1 << 20, 1, 1 << 20, 16, 8, 1 << 14, 64, 1 << 14, 0, 0, 0)
    assert big >= (1 << 20) * 16 * 512 + (1 << 20) * 8 * 1024
    # no more key tiles than the pool, or the windows, can fill
    by_pool = L.skb_chunk_attention_workspace(8, 64, 1, 16, 8, 1 << 10, 64, 100, 0, 0, 0)
    assert by_pool < 64 * (1 << 16) * 8 * 1024
    by_window = L.skb_chunk_attention_workspace(8, 64, 1, 16, 8, 1 << 10, 64, 1 << 16, 200, 4, 0)
    assert by_window < 64 * 1000 * 8 * 1024


def seen_tiles(cached, new, window, sinks):
    """Tiles of 128 slots that a row's new tokens see."""
    first = max(0, cached - window + 1) if window else 0
    slots = list(range(min(sinks, first))) + list(range(first, cached + new))
    return len({s // 128 for s in slots}), slots


@pytest.mark.parametrize("page", [1, 16, 32, 64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (256, 0), (256, 4), (1024, 4), (1024, 200), (2, 1), (129, 128)])
@pytest.mark.parametrize("rows", [1, 2, 9])
def test_workspace_holds_every_seen_tile_when_unseen_slots_have_no_page(lib, page, window, sinks, rows):
    """The pool holds the pages of the slots in sight and no other; all rows alike,
    at every phase of the window against the tiles."""
    size, kv_heads, new = lib.lib().skb_chunk_attention_workspace, 2, 3
    tile = kv_heads * (2 * 2 * 128 * 128 * 2 + 1024)  # keys and values as pairs of 16 bits, two numbers a slot
    for cached in range(1009, 1009 + 2 * 128, 3):
        tiles, slots = seen_tiles(cached, new, window, sinks)
        pages = rows * len({s // page for s in slots})
        # what is not key tiles: a cache of one slot has one tile a row
        rest = size(rows * new, rows, new, 4, kv_heads, 1, 1, rows, 0, 0, 0) - rows * tile
        got = size(rows * new, rows, new, 4, kv_heads, -(-(cached + new) // page), page, pages, window, sinks, 0)
        assert got >= rest + rows * tiles * tile, (cached, tiles)


def test_python_layer_refuses_before_the_gpu():
    import torch

    from soraku_tts_b200 import kernels

    f = torch.zeros
    pool, table = f(3, 2, 8, 16, 128), torch.zeros(2, 2, dtype=torch.int32)
    args = dict(n_heads=16, n_kv_heads=8, q_norm=f(128), k_norm=f(128), eps=1e-6, rope_cos=f(8, 64), rope_sin=f(8, 64),
                cached=torch.zeros(2, dtype=torch.int32), pos=torch.zeros(2, dtype=torch.int32), kv_pool=pool,
                page_table=table, page_size=16)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.window_decode_attention(f(2, 32 * 128), **args)
    with pytest.raises(ValueError, match="window"):
        kernels.window_decode_attention(f(2, 32 * 128), **dict(args, window=-1))
    with pytest.raises(ValueError, match="n_heads"):
        kernels.window_decode_attention(f(2, 32 * 128), **dict(args, n_heads=16.0))
    with pytest.raises(ValueError, match="chunk_start"):
        kernels.chunk_attention(f(2, 32 * 128), chunk_start=None, max_chunk=1, **args)
    with pytest.raises(ValueError, match="kv_pool"):
        kernels.evict_cache(f(2, 8, 32), cached=args["cached"], kv_pool=pool[0], page_table=table, page_size=16, budget=4)
    with pytest.raises(ValueError, match="budget"):
        kernels.evict_cache(f(2, 8, 32), cached=args["cached"], kv_pool=pool, page_table=table, page_size=16, budget=0)
