"""Sizes and addresses at the ends of what the cache and attention entry points take: through the C ABI, without a GPU."""
import pytest

from test_cache_attention_host import BAD_ARG, BAD_SHAPE, TOO_LARGE, _cache, _cross, _paged, lib  # noqa: F401  (lib: a fixture)

MANY = 2 ** 31 - 1


def test_rows_of_a_key_head_that_pass_32_bits(lib, pkg):  # noqa: F811
    """With starts max_new is only a bound, so it may be anything: rows a key head beyond 2^31 - 257 are refused before a launch."""
    for heads, new in ((4, MANY), (4, 2 ** 30), (4, 2 ** 30 - 128), (2, MANY), (2, MANY - 255), (200, 2 ** 25)):
        assert _paged(lib, _cache(pkg), heads=heads, qs=(heads * 64, 64), starts=1 << 22, new=new) == TOO_LARGE, (heads, new)
        assert _paged(lib, _cache(pkg, bits=16, dtype=1), heads=heads, qs=(heads * 64, 64), starts=1 << 22, new=new) == TOO_LARGE, (heads, new)
    for heads, kv, queries in ((4, 2, 2 ** 30), (2, 2, MANY), (200, 2, 2 ** 25)):
        assert _cross(lib, batch=1, queries=queries, heads=heads, kv=kv, qs=(0, 0, 0)) == TOO_LARGE


def test_keys_that_pass_32_bits_in_whole_tiles(lib, pkg):  # noqa: F811
    for page, width in ((16, 2 ** 27 - 7), (16, 2 ** 27 - 5), (16, 2 ** 27), (32, 2 ** 26 - 3)):
        assert _paged(lib, _cache(pkg, page_size=page), width=width) == TOO_LARGE, (page, width)
    for states in (2 ** 31 - 127, 2 ** 31 - 65, 2 ** 31 - 1):
        assert _cross(lib, states=states, ks=(0, 0, 64), vs=(0, 0, 64)) == BAD_SHAPE, states


def test_outputs_over_the_cache_or_the_tables_are_refused(lib, pkg):  # noqa: F811
    at = 1 << 24
    size = 4 * 2 * 16                                                    # rows of the cache
    ends = dict(k_pages=32 * size, v_pages=32 * size, k_stats=4 * size, v_stats=4 * size, codebooks=4 * 2 * 16)
    for name, size_of in ends.items():
        for out in (at, at + size_of - 16, at - 2 * 4 * 128 + 16):
            assert _paged(lib, _cache(pkg, **{name: at}), out=out) == BAD_ARG and b"over the cache" in lib.arcq_last_error_string(), (name, out - at)
    for name in ("k_pages", "v_pages"):
        for out in (at, at + 128 * size - 16):
            assert _paged(lib, _cache(pkg, bits=16, dtype=1, **{name: at}), out=out) == BAD_ARG and b"over the cache" in lib.arcq_last_error_string()
    for name in ("table", "lengths", "starts"):
        assert _paged(lib, _cache(pkg), **{name: at}, out=at) == BAD_ARG and b"out lies over the page table" in lib.arcq_last_error_string()
    for name in ("lengths", "mask"):
        assert _cross(lib, **{name: at + 4}, out=at) == BAD_ARG and b"out lies over the lengths" in lib.arcq_last_error_string()
    # a cache of more bytes than 64 bits count
    assert _paged(lib, _cache(pkg, pages=MANY, heads=65535, page_size=1 << 20), heads=65535, out=1 << 40, qs=(65535 * 64, 64)) == BAD_ARG
