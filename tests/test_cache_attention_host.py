"""What the cache and attention entry points refuse before anything is launched: through the C ABI, without a GPU."""
import ctypes

import pytest
import torch

BAD_ARG, BAD_SHAPE, UNSUPPORTED, ALIGN, TOO_LARGE = -1, -2, -3, -4, -6


def _cache(pkg, **kw):
    p = 1 << 20                                  # stands for device memory: every call here is refused, or has nothing to do, before it is used
    d = dict(k_pages=p, v_pages=p, k_stats=p, v_stats=p, codebooks=p, pages=4, heads=2, page_size=16, bits=4, dtype=0)
    return pkg._cabi.KvCache(**{**d, **kw})


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


@pytest.fixture()
def lib(pkg):
    return pkg._cabi.load()


def _write(lib, c, th=1 << 20, k=1 << 20, v=1 << 20, dt=1, tokens=3, ks=(128, 64), vs=(128, 64), slots=1 << 20):
    return lib.arcq_kv_cache_write(ctypes.byref(c), th, k, v, dt, tokens, _i64(*ks), _i64(*vs), slots, None)


def _read(lib, c, slots=1 << 20, tokens=3, k=1 << 20, v=1 << 20, dt=1):
    return lib.arcq_kv_cache_read(ctypes.byref(c), slots, tokens, k, v, dt, None)


def _paged(lib, c, q=1 << 20, dt=1, rows=2, qs=(256, 64), heads=4, batch=2, table=1 << 20, width=3, lengths=1 << 20, starts=None, new=1, causal=1,
           scale=0.125, out=1 << 21, work=1 << 20):
    return lib.arcq_paged_attention(ctypes.byref(c), q, dt, rows, _i64(*qs), heads, batch, table, width, lengths, starts, new, causal, scale, out, work, 1 << 20, None)


def _cross(lib, q=1 << 20, k=1 << 20, v=1 << 20, dt=1, batch=2, queries=3, states=5, heads=4, kv=2, qs=(768, 256, 64), ks=(640, 128, 64),
           vs=(640, 128, 64), lengths=None, mask=None, scale=0.125, out=1 << 21, work=1 << 20):
    return lib.arcq_cross_attention(q, k, v, dt, batch, queries, states, heads, kv, _i64(*qs), _i64(*ks), _i64(*vs), lengths, mask, 5, scale, out, work, 1 << 20, None)


@pytest.mark.parametrize("change,code", [
    (dict(bits=5), BAD_ARG), (dict(bits=8), BAD_ARG), (dict(heads=0), BAD_SHAPE), (dict(pages=-1), BAD_SHAPE), (dict(page_size=8), UNSUPPORTED),
    (dict(page_size=48), UNSUPPORTED), (dict(page_size=1 << 21), UNSUPPORTED), (dict(k_pages=None), BAD_ARG), (dict(v_stats=None), BAD_ARG),
    (dict(codebooks=None), BAD_ARG), (dict(v_pages=(1 << 20) + 8), ALIGN), (dict(k_stats=(1 << 20) + 4), ALIGN), (dict(bits=16, dtype=0), BAD_ARG)])
def test_caches_that_are_refused(lib, pkg, change, code):
    c = _cache(pkg, **change)
    assert _write(lib, c) == code and _read(lib, c) == code and _paged(lib, c) == code
    assert lib.arcq_last_error_string() != b""


def test_writes_and_reads_that_are_refused(lib, pkg):
    c = _cache(pkg)
    assert _write(lib, c, th=None) == BAD_ARG and _write(lib, c, k=None) == BAD_ARG and _write(lib, c, slots=None) == BAD_ARG
    assert _write(lib, c, dt=3) == BAD_ARG and _write(lib, c, tokens=-1) == BAD_SHAPE and _write(lib, c, tokens=1 << 31) == BAD_SHAPE
    assert _write(lib, c, k=(1 << 20) + 2) == ALIGN and _write(lib, c, ks=(128, 68)) == ALIGN and _write(lib, c, vs=(100, 64)) == ALIGN
    assert _write(lib, _cache(pkg, bits=16, dtype=1), dt=2) == BAD_ARG
    assert _read(lib, c, dt=7) == BAD_ARG and _read(lib, c, k=None) == BAD_ARG and _read(lib, c, v=(1 << 20) + 8) == ALIGN and _read(lib, c, tokens=-2) == BAD_SHAPE
    assert _write(lib, c, tokens=0) == 0 and _read(lib, c, tokens=0) == 0
    assert lib.arcq_kv_cache_read(None, None, 0, None, None, 1, None) == BAD_ARG


def test_attention_that_is_refused(lib, pkg):
    c = _cache(pkg)
    assert _paged(lib, c, dt=0) == BAD_ARG and _paged(lib, c, heads=3) == BAD_SHAPE and _paged(lib, c, heads=0) == BAD_SHAPE
    assert _paged(lib, c, rows=3) == BAD_SHAPE and _paged(lib, c, batch=-1) == BAD_SHAPE and _paged(lib, c, width=1 << 31) == TOO_LARGE
    assert _paged(lib, c, lengths=None) == BAD_ARG and _paged(lib, c, table=None) == BAD_ARG and _paged(lib, c, q=None) == BAD_ARG
    assert _paged(lib, c, q=(1 << 20) + 8) == ALIGN and _paged(lib, c, qs=(256, 60)) == ALIGN and _paged(lib, c, out=(1 << 20) + 2) == ALIGN
    for s in (0.0, -0.125, float("inf"), float("nan"), 3e38):
        assert _paged(lib, c, scale=s) == BAD_ARG and _cross(lib, scale=s) == BAD_ARG
    assert _paged(lib, _cache(pkg, bits=16, dtype=2)) == BAD_ARG
    assert _paged(lib, c, batch=0, rows=0) == 0 and _paged(lib, c, rows=0, starts=1 << 20) == 0
    assert _cross(lib, dt=0) == BAD_ARG and _cross(lib, kv=3) == BAD_SHAPE and _cross(lib, queries=-1) == BAD_SHAPE and _cross(lib, states=-1) == BAD_SHAPE
    assert _cross(lib, k=None) == BAD_ARG and _cross(lib, lengths=1 << 20, mask=1 << 20) == BAD_ARG
    assert _cross(lib, v=(1 << 20) + 2) == ALIGN and _cross(lib, ks=(641, 128, 64)) == ALIGN
    assert _paged(lib, c, work=(1 << 20) + 8) == ALIGN and _cross(lib, work=(1 << 20) + 4) == ALIGN
    assert _cross(lib, batch=0) == 0 and _cross(lib, queries=0) == 0


def test_sizes_whose_products_pass_64_bits(lib, pkg):
    c = _cache(pkg, heads=4, page_size=16)
    assert _write(lib, c, tokens=1 << 62) == BAD_SHAPE and _read(lib, c, tokens=1 << 62) == BAD_SHAPE
    assert _paged(lib, c, width=1 << 60) == TOO_LARGE and _paged(lib, c, new=1 << 62) == BAD_SHAPE
    assert _cross(lib, queries=1 << 62) == BAD_SHAPE and _cross(lib, batch=1 << 62) == BAD_SHAPE and _cross(lib, states=1 << 62) == BAD_SHAPE


def test_outputs_over_inputs_are_refused(lib, pkg):
    c, at = _cache(pkg), 1 << 20
    q_end = at + 2 * (256 + 3 * 64 + 64)                                 # two rows of four heads
    for out in (at, q_end - 16, at - 2 * 4 * 128 + 16):
        assert _paged(lib, c, out=out) == BAD_ARG and b"over the queries" in lib.arcq_last_error_string()
    for out in (at, at + 16):
        for other in ("q", "k", "v"):
            where = {n: 1 << 22 for n in "qkv"}
            assert _cross(lib, **{**where, other: at}, out=out) == BAD_ARG and b"out lies over" in lib.arcq_last_error_string()
    back = at + 2 * 256                                                  # rows one after the other downwards
    assert _paged(lib, c, q=back, qs=(-256, 64), out=at) == BAD_ARG and b"over the queries" in lib.arcq_last_error_string()


def test_operators_refuse_tensors_of_the_host(pkg):
    x = torch.zeros(2, 4, 64, dtype=torch.float16)
    pages = torch.zeros(2, 4, 16, 64, dtype=torch.float16)
    i32 = torch.zeros(2, dtype=torch.int32)
    for f in (lambda: pkg.ops.paged_attention(x, pages, pages, i32[None], i32[:1]), lambda: pkg.ops.cross_attention(x[None], x[None], x[None]),
              lambda: pkg.ops.kv_cache_write(x, x, i32.long(), pages, pages), lambda: pkg.ops.kv_cache_read(i32.long(), pages, pages)):
        with pytest.raises(RuntimeError):
            f()
