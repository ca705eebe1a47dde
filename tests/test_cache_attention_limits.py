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
