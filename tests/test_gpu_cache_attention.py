"""The paged key/value cache, attention over it and attention to an encoder's states, against plain evaluations in 64 bits.

Bounds of the attentions, per output, are those of the roundings that the kernels make (u = 2^-11 for fp16, 2^-8 for bf16):
  packed keys and values   a level rounded to fp16, up or down (two half steps), or to the nearest with one fma behind it:
                           u16 * (2 |scale * level| + |x|) at most; center and scale * level come together in fp32, 2^-20 of the center
  a score                  the keys' errors times |q|, and 64 products summed in fp32 (2^-23 each, the tensor cores may truncate)
  a weight                 twice the largest score error of the row, the exponential (2^-20 with its argument), one rounding to 16 bits
                           (in fp16 2^-25 at least) before the second product
  the sum over n keys      n * 2^-23; the output's rounding u."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _levels(bits, dev):
    at = (torch.arange(2 ** bits, dtype=torch.float64) + 0.5) / 2 ** bits
    lv = torch.special.ndtri(at)
    lv = torch.stack([lv, 1.1 * lv + 0.02]).float()
    return lv.to(dev), ((lv[:, 1:] + lv[:, :-1]) / 2).to(dev)


def _empty_cache(pages, heads, page, bits, dtype, dev):
    if bits == 16:
        return dict(k_pages=torch.zeros(pages, heads, page, 64, dtype=dtype, device=dev),
                    v_pages=torch.zeros(pages, heads, page, 64, dtype=dtype, device=dev)), None
    cb, th = _levels(bits, dev)
    c = dict(codebooks=cb)
    for n in "kv":
        c[n + "_pages"] = torch.zeros(pages, heads, page, 8 * bits, dtype=torch.uint8, device=dev)
        c[n + "_stats"] = torch.zeros(pages, heads, page, 2, dtype=torch.float16, device=dev)
    return c, th


def _cached(pkg, c, which, rows):
    """Values [n, heads, 64] in 64 bits of cache rows (page, place) [n, 2], and what their roundings to fp16 may be off by."""
    i = "kv".index(which)
    got = c[which + "_pages"][rows[:, 0], :, rows[:, 1]]
    if got.dtype != torch.uint8 or got.shape[0] == 0:
        got = got if got.dtype != torch.uint8 else got.new_zeros(0, got.shape[1], 64)
        return got.double(), torch.zeros_like(got, dtype=torch.float64)
    n, heads, width = got.shape
    codes = pkg.ops.unpack_codes_u8(got.reshape(n * heads, width).contiguous(), width // 8, 64).long().reshape(n, heads, 64)
    st = c[which + "_stats"][rows[:, 0], :, rows[:, 1]].double()
    part = st[..., 1:] * c["codebooks"][i].double()[codes]
    x = st[..., :1] + part
    return x, U[torch.float16] * (2 * part.abs() + x.abs()) + 2.0 ** -20 * st[..., :1].abs()


def _attend(q, k, dk, v, dv, seen, scale, dtype, packed):
    """One sequence: q [n, H, 64], k, v (and their errors) [S, Hk, 64], seen [n, S]: output and bound."""
    n, H, _ = q.shape
    S, Hk = k.shape[:2]
    out = torch.zeros(n, H, 64, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(out)
    up = U[torch.float16 if packed else dtype]
    for h in range(H):
        kk, vv, ek, ev = (t[:, h // (H // Hk)] for t in (k, v, dk, dv))
        qq = q[:, h].double()
        if S == 0:
            continue
        s = scale * qq @ kk.t()
        ds = scale * qq.abs() @ (ek + 64 * 2.0 ** -23 * kk.abs()).t() + s.abs() * 2.0 ** -22
        if packed and dtype == torch.bfloat16:
            ds = ds + scale * 2.0 ** -27 * qq.abs().amax(-1, keepdim=True) * kk.abs().sum(-1)      # values far below the row's largest
        s = s.masked_fill(~seen, float("-inf"))
        some = seen.any(-1)
        if not bool(some.any()):
            continue
        w = torch.softmax(s[some], -1)
        D = ds[some].masked_fill(~seen[some], 0.0).amax(-1, keepdim=True)
        o = w @ vv
        rel = torch.expm1(2 * D) + up + 2.0 ** -20 + S * 2.0 ** -23
        tiny = 2.0 ** -25 if up == U[torch.float16] else 0.0
        out[some, h] = o
        off[some, h] = 1.05 * (rel * (w @ vv.abs()) + w @ ev + tiny * (seen[some].double() @ vv.abs()) + U[dtype] * o.abs()) + 2.0 ** -24
    return out, off


def _filled(pkg, gen, pages, heads, page, bits, dtype, dev, spread=1.0):
    c, th = _empty_cache(pages, heads, page, bits, dtype, dev)
    T = pages * page
    x = [(spread * (torch.randn(T, heads, 64, generator=gen) + 0.5 * torch.randn(heads, 64, generator=gen))).to(dtype).to(dev) for _ in range(2)]
    pkg.ops.kv_cache_write(x[0], x[1], torch.arange(T, device=dev), thresholds=th, **c)
    return c


def _paged_check(pkg, dev, bits, dtype, heads, kv_heads, page, lengths, new, seed=0, causal=True, scale=None, spread=1.0, bad_pages=(), strided=False):
    gen = torch.Generator().manual_seed(seed)
    B = len(lengths)
    width = max(1, max(-(-n // page) for n in lengths))
    pages = B * width + 2
    c = _filled(pkg, gen, pages, kv_heads, page, bits, dtype, dev, spread)
    table = torch.randperm(pages, generator=gen)[:B * width].reshape(B, width).to(torch.int32)
    for b, j, value in bad_pages:
        table[b, j] = value
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    total = int(starts[-1])
    q = (1.3 * torch.randn(total + 3, heads + (2 if strided else 0), 64, generator=gen)).to(dtype).to(dev)
    q = q[:, 1:1 + heads] if strided else q
    out = torch.full(q.shape, 7.0, dtype=dtype, device=dev)
    got = pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev), starts.to(dev),
                                  max(new), k_stats=c.get("k_stats"), v_stats=c.get("v_stats"), codebooks=c.get("codebooks"), causal=causal,
                                  scale=scale, out=out)
    assert got is out
    assert bool((out[total:] == 7.0).all())                       # rows behind the last sequence
    worst = 0.0
    for b in range(B):
        L, n = lengths[b], new[b]
        if n == 0:
            continue
        j = torch.arange(L)
        page_of = table[b][j // page].long()
        there = (page_of >= 0) & (page_of < pages)
        rows = torch.stack([page_of.clamp(0, pages - 1), j % page], 1).to(dev)
        (k, dk), (v, dv) = (_cached(pkg, c, w, rows) for w in "kv")
        seen = there[None, :].expand(n, L)
        if causal:
            seen = seen & (j[None, :] <= (L - n + torch.arange(n))[:, None])
        lo = int(starts[b])
        want, off = _attend(q[lo:lo + n], k, dk, v, dv, seen.to(dev), scale or 0.125, dtype, bits != 16)
        err = (out[lo:lo + n].double() - want).abs()
        assert bool((err <= off).all()), (b, L, n, float((err - off).max()), float((err / off).max()))
        worst = max(worst, float((err / off).max()))
    assert pkg.ops.device_status() == 0
    return worst


# ---------------------------------------------------------------- cache
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [2, 3, 4])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 16), (7, 3, 16), (130, 12, 64), (3001, 6, 32), (9973, 8, 256)])
def test_written_codes_are_the_quantizers(pkg, cuda_device, bits, dtype, tokens, heads, page):
    gen = torch.Generator().manual_seed(tokens + bits)
    pages = -(-tokens // page) + 2
    c, th = _empty_cache(pages, heads, page, bits, dtype, cuda_device)
    qkv = (torch.randn(tokens, 3 * heads, 64, generator=gen) * torch.rand(tokens, 1, 1, generator=gen) + 0.2).to(dtype).to(cuda_device)
    qkv[0, heads] = 0.25                                           # a group of equal values
    k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
    slots = torch.randperm(pages * page, generator=gen)[:tokens].to(cuda_device)
    pkg.ops.kv_cache_write(k, v, slots, thresholds=th, **c)
    at = (slots // page, slice(None), slots % page)
    for i, (n, x) in enumerate((("k", k), ("v", v))):
        packed, mu, sg, cs = pkg.ops.quantize_activation(x.reshape(tokens, heads * 64).contiguous(), th[i].contiguous(), c["codebooks"][i].contiguous(), bits, 64)
        assert torch.equal(c[n + "_pages"][at], packed.reshape(tokens, heads, 8 * bits))
        st = c[n + "_stats"][at].double()
        center = mu.double() - sg.double() * cs.double() / 64
        # the center is one fma of the quantizer's statistics in fp32, then rounded to fp16
        assert bool(((st[..., 0] - center).abs() <= U[torch.float16] * center.abs() + 2.0 ** -24 * (mu.double().abs() + center.abs()) + 2.0 ** -25).all())
        assert torch.equal(c[n + "_stats"][at][..., 1], sg.half())
    # nothing else was written
    keep = torch.ones(pages * page, dtype=torch.bool, device=cuda_device)
    keep[slots] = False
    rest = keep.nonzero()[:, 0]
    assert not bool(c["k_pages"][rest // page, :, rest % page].any()) and not bool(c["v_stats"][rest // page, :, rest % page].any())
    # read back
    for out in (torch.float32, torch.float16, torch.bfloat16):
        got = pkg.ops.kv_cache_read(slots, out_dtype=out, **c)
        for n, g in zip("kv", got):
            x, _ = _cached(pkg, c, n, torch.stack([slots // page, slots % page], 1))
            assert g.dtype == out and tuple(g.shape) == (tokens, heads, 64)
            once = 2.0 ** -24 if out != torch.float32 else 0.0      # the fma in fp32 is rounded before the output type is
            assert bool(((g.double() - x).abs() <= (U[out] + once) * x.abs() + 2.0 ** -25).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_pages_in_16_bits_are_copies(pkg, cuda_device, dtype):
    c, _ = _empty_cache(5, 3, 32, 16, dtype, cuda_device)
    x = torch.randn(100, 8, 64).to(dtype).to(cuda_device)
    x[3, 1, 5] = float("nan")
    k, v = x[:, :3], x[:, 4:7]
    slots = torch.randperm(160)[:100].to(cuda_device)
    pkg.ops.kv_cache_write(k, v, slots, **c)
    got = pkg.ops.kv_cache_read(slots, out_dtype=dtype, **c)
    assert torch.equal(got[0].view(torch.int16), k.contiguous().view(torch.int16)) and torch.equal(got[1].view(torch.int16), v.contiguous().view(torch.int16))
    assert torch.equal(pkg.ops.kv_cache_read(slots, out_dtype=torch.float32, **c)[1], v.float())


@pytest.mark.parametrize("bits", [4, 16])
def test_slots_that_do_not_exist(pkg, cuda_device, bits):
    c, th = _empty_cache(4, 2, 16, bits, torch.float16, cuda_device)
    x = torch.randn(6, 2, 64).half().to(cuda_device)
    slots = torch.tensor([3, -1, 64, 2 ** 40, -2 ** 40, 63], device=cuda_device)
    pkg.ops.kv_cache_write(x, x, slots, thresholds=th, **c)
    k, v = pkg.ops.kv_cache_read(slots, **c)
    assert not bool(k[1:5].any()) and not bool(v[1:5].any()) and bool(k[0].any()) and bool(v[5].any())
    everything = pkg.ops.kv_cache_read(torch.arange(64, device=cuda_device), **c)[0]
    assert int(everything.any(-1).any(-1).sum()) == 2


def test_values_at_the_ends_of_fp16(pkg, cuda_device):
    """Statistics beyond fp16's range are held at its end; what is read is finite."""
    c, th = _empty_cache(1, 1, 16, 4, torch.float32, cuda_device)
    x = torch.full((2, 1, 64), 3e6, device=cuda_device)
    x[1, 0, ::2] = -3e6
    pkg.ops.kv_cache_write(x, x, torch.arange(2, device=cuda_device), thresholds=th, **c)
    assert bool(torch.isfinite(c["k_stats"]).all())
    assert bool(torch.isfinite(pkg.ops.kv_cache_read(torch.arange(2, device=cuda_device), out_dtype=torch.float32, **c)[0]).all())


# ---------------------------------------------------------------- attention over pages
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [2, 3, 4, 16])
@pytest.mark.parametrize("heads,kv_heads,page,lengths", [
    (1, 1, 16, [1]), (6, 6, 16, [333]), (12, 4, 64, [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 500]), (8, 1, 128, [1000, 2, 700]),
    (36, 2, 32, [255, 257, 40])])
def test_one_new_token(pkg, cuda_device, bits, dtype, heads, kv_heads, page, lengths):
    _paged_check(pkg, cuda_device, bits, dtype, heads, kv_heads, page, lengths, [1] * len(lengths))


@pytest.mark.parametrize("bits,dtype", [(4, torch.float16), (4, torch.bfloat16), (3, torch.float16), (2, torch.bfloat16), (16, torch.float16), (16, torch.bfloat16)])
@pytest.mark.parametrize("heads,kv_heads,page,lengths,new", [
    (2, 2, 16, [5, 200, 3], [5, 77, 3]),                     # prompts, and pieces behind a context
    (6, 2, 32, [130, 130, 129, 1, 700], [1, 130, 128, 1, 257]),
    (4, 4, 64, [10, 0, 90, 40], [20, 3, 0, 40]),             # more new tokens than there are; none
    (12, 1, 256, [900], [40])])
def test_new_tokens_in_pieces(pkg, cuda_device, bits, dtype, heads, kv_heads, page, lengths, new):
    _paged_check(pkg, cuda_device, bits, dtype, heads, kv_heads, page, lengths, new, seed=3)
    _paged_check(pkg, cuda_device, bits, dtype, heads, kv_heads, page, lengths, new, seed=4, causal=False, scale=0.3, strided=True)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("new", [3, 40, 140])
def test_more_sequences_than_multiprocessors(pkg, cuda_device, bits, new):
    """Every block then has all keys of its rows, a ring of tiles deep."""
    lengths = [200 + (37 * i) % 900 for i in range(170)]
    _paged_check(pkg, cuda_device, bits, torch.float16, 1, 1, 64, lengths, [min(new, 1 + (11 * i) % (new + 9)) for i in range(170)], seed=14)
    _cross_check(pkg, cuda_device, torch.bfloat16, 170, new, 900, 1, 1, "mask", seed=15)


@pytest.mark.parametrize("bits,dtype", [(4, torch.float16), (16, torch.bfloat16)])
def test_long_contexts(pkg, cuda_device, bits, dtype):
    _paged_check(pkg, cuda_device, bits, dtype, 3, 3, 64, [20011, 4097], [1, 1], seed=5)
    _paged_check(pkg, cuda_device, bits, dtype, 3, 1, 128, [6000, 3333], [300, 129], seed=6)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("new", [1, 150])
def test_pages_that_do_not_exist_are_not_seen(pkg, cuda_device, bits, new):
    bad = [(0, 0, -1), (0, 2, 10 ** 9), (1, 1, -2 ** 31), (2, 0, 99999), (2, 1, -5), (2, 2, -5), (2, 3, -7), (2, 4, 2 ** 31 - 1)]
    _paged_check(pkg, cuda_device, bits, torch.float16, 4, 2, 32, [150, 160, 160], [new] * 3, seed=7, bad_pages=bad)


@pytest.mark.parametrize("spread", [1e-3, 300.0])
@pytest.mark.parametrize("bits,dtype", [(4, torch.float16), (4, torch.bfloat16), (16, torch.bfloat16)])
def test_small_and_large_values(pkg, cuda_device, bits, dtype, spread):
    scale = 0.125 if spread < 1 else 1e-3
    _paged_check(pkg, cuda_device, bits, dtype, 2, 2, 16, [300, 90], [1, 90], seed=8, spread=spread, scale=scale)


@pytest.mark.parametrize("new", [1, 140])
def test_queries_of_bf16_over_packed_keys_in_any_range(pkg, cuda_device, new):
    """fp16 products with bf16 queries: each row is scaled by a power of two, so its size does not matter."""
    gen = torch.Generator().manual_seed(1)
    c = _filled(pkg, gen, 8, 2, 32, 4, torch.bfloat16, cuda_device)
    table = torch.arange(8, dtype=torch.int32, device=cuda_device)[None]
    L = torch.tensor([250], dtype=torch.int32, device=cuda_device)
    starts = torch.tensor([0, new], dtype=torch.int32, device=cuda_device)
    q = torch.randn(new, 4, 64, generator=gen).bfloat16().to(cuda_device)
    args = dict(k_stats=c["k_stats"], v_stats=c["v_stats"], codebooks=c["codebooks"])
    want = pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, L, starts, new, **args)
    for e in (-60, -20, 20, 60):
        got = pkg.ops.paged_attention(q * 2.0 ** e, c["k_pages"], c["v_pages"], table, L, starts, new, scale=0.125 * 2.0 ** -e, **args)
        assert torch.equal(got, want), e


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("new", [1, 130])
def test_what_is_not_seen_has_no_effect(pkg, cuda_device, bits, new):
    gen = torch.Generator().manual_seed(2)
    c = _filled(pkg, gen, 10, 2, 32, bits, torch.float16, cuda_device)
    table = torch.tensor([[3, 1, 4, 0, 9, 7]], dtype=torch.int32, device=cuda_device)
    length = torch.tensor([150], dtype=torch.int32, device=cuda_device)
    starts = torch.tensor([0, new], dtype=torch.int32, device=cuda_device)
    q = torch.randn(new, 4, 64, generator=gen).half().to(cuda_device)
    args = {n: c.get(n) for n in ("k_stats", "v_stats", "codebooks")}
    want = pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, length, starts, new, **args)
    bad = float("nan")
    for n in "kv":
        t = c[n + "_stats"] if bits != 16 else c[n + "_pages"]
        t[9, :, 22:] = bad                                     # the page that the sequence ends in
        t[7] = float("inf")
        t[2] = bad
    assert torch.equal(pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, length, starts, new, **args), want)


def test_every_sequence_by_itself_and_without_starts(pkg, cuda_device):
    """A row's result does not depend on the other sequences; without starts there are max_new rows each."""
    gen = torch.Generator().manual_seed(3)
    c = _filled(pkg, gen, 12, 3, 16, 4, torch.float16, cuda_device)
    args = {n: c.get(n) for n in ("k_stats", "v_stats", "codebooks")}
    table = torch.arange(12, dtype=torch.int32, device=cuda_device).reshape(3, 4)
    lengths = torch.tensor([64, 17, 40], dtype=torch.int32, device=cuda_device)
    for n in (1, 2, 16):
        q = torch.randn(3 * n, 6, 64, generator=gen).half().to(cuda_device)
        both = pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, lengths, None, n, **args)
        starts = torch.arange(0, 3 * n + 1, n, dtype=torch.int32, device=cuda_device)
        assert torch.equal(both, pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, lengths, starts, n, **args))
        # bounds of the lengths do not change a sequence's result either
        for b in range(3):
            alone = pkg.ops.paged_attention(q[b * n:(b + 1) * n], c["k_pages"], c["v_pages"], table[b:b + 1].contiguous(), lengths[b:b + 1], None, n, **args)
            assert float((alone.double() - both[b * n:(b + 1) * n].double()).abs().max()) <= 2.0 ** -9


def test_lengths_and_starts_that_promise_too_much(pkg, cuda_device):
    gen = torch.Generator().manual_seed(4)
    c = _filled(pkg, gen, 4, 1, 16, 4, torch.float16, cuda_device)
    args = {n: c.get(n) for n in ("k_stats", "v_stats", "codebooks")}
    table = torch.arange(4, dtype=torch.int32, device=cuda_device).reshape(2, 2)
    q = torch.randn(4, 1, 64, generator=gen).half().to(cuda_device)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    out = torch.full_like(q, 5.0)
    # more tokens than the table has pages for: the table's; negative lengths: none
    pkg.ops.paged_attention(q[:2], c["k_pages"], c["v_pages"], table, torch.tensor([10 ** 6, -3], **i32), None, 1, out=out[:2], **args)
    full = pkg.ops.paged_attention(q[:1], c["k_pages"], c["v_pages"], table[:1], torch.tensor([32], **i32), None, 1, **args)
    assert torch.equal(out[:1], full) and not bool(out[1].any()) and bool((out[2:] == 5.0).all())
    # starts beyond the rows of q, before them, or backwards: only rows that exist
    for starts in ([0, 2, 10 ** 9], [3, 2, 4], [-5, 1, 2], [2 ** 31 - 1, 4, 4]):
        out.fill_(5.0)
        pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, torch.tensor([20, 20], **i32), torch.tensor(starts, **i32), 4, out=out, **args)
        torch.cuda.synchronize()
    # more new tokens than max_new: the first max_new
    out.fill_(5.0)
    pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, torch.tensor([20, 20], **i32), torch.tensor([0, 3, 4], **i32), 2, out=out, **args)
    assert bool((out[2] == 5.0).all()) and not bool((out[1] == 5.0).all()) and not bool((out[3] == 5.0).all())


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("new", [1, 200])
def test_offsets_beyond_32_bits(pkg, cuda_device, bits, new):
    heads, page = 8, 256
    row = 128 if bits == 16 else 32
    pages = 2 ** 32 // (heads * page * row) + 40
    c = dict(codebooks=None, k_stats=None, v_stats=None)
    th = None
    if bits == 16:
        for n in "kv":
            c[n + "_pages"] = torch.empty(pages, heads, page, 64, dtype=torch.float16, device=cuda_device)
    else:
        c["codebooks"], th = _levels(bits, cuda_device)
        for n in "kv":
            c[n + "_pages"] = torch.empty(pages, heads, page, row, dtype=torch.uint8, device=cuda_device)
            c[n + "_stats"] = torch.empty(pages, heads, page, 2, dtype=torch.float16, device=cuda_device)
    far = torch.tensor([pages - 1, 3, pages - 7], device=cuda_device)
    slots = (far[:, None] * page + torch.arange(page, device=cuda_device)).reshape(-1)
    x = [torch.randn(3 * page, heads, 64, device=cuda_device).half() for _ in range(2)]
    pkg.ops.kv_cache_write(x[0], x[1], slots, thresholds=th, **c)
    got = pkg.ops.kv_cache_read(slots, **c)
    near, _ = _empty_cache(3, heads, page, bits, torch.float16, cuda_device)
    pkg.ops.kv_cache_write(x[0], x[1], torch.arange(3 * page, device=cuda_device), thresholds=th, **near)
    want = pkg.ops.kv_cache_read(torch.arange(3 * page, device=cuda_device), **near)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = torch.randn(new, heads, 64, device=cuda_device).half()
    L = torch.tensor([3 * page - 5], dtype=torch.int32, device=cuda_device)
    args = {n: c[n] for n in ("k_stats", "v_stats", "codebooks")}
    nargs = {n: near.get(n) for n in ("k_stats", "v_stats", "codebooks")}
    a = pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], far[None].to(torch.int32), L, None, new, **args)
    b = pkg.ops.paged_attention(q, near["k_pages"], near["v_pages"], torch.arange(3, dtype=torch.int32, device=cuda_device)[None], L, None, new, **nargs)
    assert torch.equal(a, b)


# ---------------------------------------------------------------- attention to an encoder's states
def _cross_check(pkg, dev, dtype, B, n, S, heads, kv_heads, form, seed=0, spread=1.0, scale=None):
    gen = torch.Generator().manual_seed(seed)
    q = (1.3 * torch.randn(B, n, heads, 64, generator=gen)).to(dtype).to(dev)
    kv = (spread * torch.randn(B, S, 2 * kv_heads, 64, generator=gen)).to(dtype).to(dev)
    k, v = kv[:, :, :kv_heads], kv[:, :, kv_heads:]
    seen = torch.ones(B, S, dtype=torch.bool)
    args = {}
    if form == "lengths":
        lengths = torch.randint(0, S + 1, (B,), generator=gen)
        lengths[0] = S
        if B > 1:
            lengths[-1] = 0
        seen = torch.arange(S)[None] < lengths[:, None]
        args["lengths"] = lengths.to(torch.int32).to(dev)
    if form == "mask":
        seen = torch.rand(B, S, generator=gen) < 0.6
        seen[-1] = False
        args["mask"] = seen.to(dev)
    hidden = ~seen.to(dev)
    kv.masked_fill_(hidden[:, :, None, None], float("nan"))
    out = pkg.ops.cross_attention(q, k, v, scale=scale, **args)
    assert out.shape == q.shape and out.dtype == dtype
    zero = torch.zeros(S, kv_heads, 64, dtype=torch.float64, device=dev)
    for b in range(B):
        kk, vv = (t[b].double().masked_fill(hidden[b][:, None, None], 0.0) for t in (k, v))
        want, off = _attend(q[b], kk, zero, vv, zero, seen[b].to(dev)[None].expand(n, S), scale or 0.125, dtype, False)
        err = (out[b].double() - want).abs()
        assert bool((err <= off).all()), (b, float((err / off).max()))
    assert pkg.ops.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", ["none", "lengths", "mask"])
@pytest.mark.parametrize("B,n,S,heads,kv_heads", [(1, 1, 1, 1, 1), (5, 1, 197, 6, 6), (3, 2, 16, 8, 2), (2, 40, 577, 12, 12), (2, 129, 65, 4, 1),
                                                  (3, 300, 333, 3, 3), (1, 5, 2309, 2, 2), (2, 128, 128, 2, 2)])
def test_cross_attention(pkg, cuda_device, dtype, form, B, n, S, heads, kv_heads):
    _cross_check(pkg, cuda_device, dtype, B, n, S, heads, kv_heads, form, seed=n + S)


@pytest.mark.parametrize("n", [1, 140])
def test_cross_attention_of_large_scores(pkg, cuda_device, n):
    _cross_check(pkg, cuda_device, torch.float16, 2, n, 200, 2, 2, "mask", seed=9, spread=20.0)
    _cross_check(pkg, cuda_device, torch.bfloat16, 2, n, 200, 2, 2, "lengths", seed=10, spread=1e-3)


@pytest.mark.parametrize("n", [1, 130])
def test_no_states(pkg, cuda_device, n):
    q = torch.randn(2, n, 4, 64, device=cuda_device).half()
    k = torch.empty(2, 0, 4, 64, device=cuda_device).half()
    assert not bool(pkg.ops.cross_attention(q, k, k).any())
    assert pkg.ops.cross_attention(q[:0], k[:0], k[:0]).shape == (0, n, 4, 64)
    assert pkg.ops.cross_attention(q[:, :0], k, k).shape == (2, 0, 4, 64)


@pytest.mark.parametrize("n", [1, 130])
def test_layouts_of_cross_attention(pkg, cuda_device, n):
    """Heads before tokens, shared and unaligned tensors: what the contiguous ones give."""
    gen = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(2, t, 4, 64, generator=gen).half().to(cuda_device) for t in (n, 77, 77))
    want = pkg.ops.cross_attention(q, k, v)
    swapped = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(pkg.ops.cross_attention(*swapped), want)
    odd = []
    for t in (q, k, v):
        b = torch.empty(t.numel() + 3, dtype=t.dtype, device=cuda_device)[3:].view(t.shape)
        b.copy_(t)
        odd.append(b)
    assert torch.equal(pkg.ops.cross_attention(*odd), want)
    one = k[:1].expand(2, -1, -1, -1)
    assert torch.equal(pkg.ops.cross_attention(q, one, one), pkg.ops.cross_attention(q, one.contiguous(), one.contiguous()))
    mask = (torch.rand(77, 2, generator=gen) < 0.5).to(cuda_device).t()
    assert torch.equal(pkg.ops.cross_attention(q, k, v, mask=mask), pkg.ops.cross_attention(q, k, v, mask=mask.contiguous()))


# ---------------------------------------------------------------- together, streams, graphs, refusals
@pytest.mark.parametrize("bits", [4, 16])
def test_a_decoder_layer_prompt_then_token_by_token(pkg, cuda_device, bits):
    """A prompt at once and its last tokens one by one, captured: the same states, and the encoder's states attended to on the way."""
    gen = torch.Generator().manual_seed(12)
    B, H, Hk, page, P, n = 3, 6, 2, 16, 70, 5
    dev = cuda_device
    qkv = torch.randn(B, P + n, H + 2 * Hk, 64, generator=gen).half().to(dev)
    kv = torch.randn(B, 197, 2 * H, 64, generator=gen).half().to(dev)
    c, th = _empty_cache(B * 5 + 1, Hk, page, bits, torch.float16, dev)
    table = torch.randperm(B * 5 + 1, generator=gen)[:B * 5].reshape(B, 5).to(torch.int32).to(dev)
    args = {m: c.get(m) for m in ("k_stats", "v_stats", "codebooks")}

    def slots(at):                                                    # [B, tokens] positions -> slots
        return (table.long().gather(1, at // page) * page + at % page).reshape(-1)

    def step(x, at, lengths):                                         # x [B, t, heads, 64]
        t = x.shape[1]
        x = x.reshape(B * t, H + 2 * Hk, 64)
        pkg.ops.kv_cache_write(x[:, H:H + Hk], x[:, H + Hk:], slots(at), thresholds=th, **c)
        y = pkg.ops.paged_attention(x[:, :H], c["k_pages"], c["v_pages"], table, lengths, None, t, **args)
        return pkg.ops.cross_attention(y.reshape(B, t, H, 64), kv[:, :, :H], kv[:, :, H:]), y

    pos = torch.arange(P + n, device=dev)[None].expand(B, -1)
    i32 = dict(dtype=torch.int32, device=dev)
    whole, mid = step(qkv, pos, torch.full((B,), P + n, **i32))
    # the same in pieces: prompt, then a captured step replayed
    step(qkv[:, :P], pos[:, :P], torch.full((B,), P, **i32))
    x, at, lengths = qkv[:, P:P + 1].clone(), pos[:, P:P + 1].clone(), torch.full((B,), P + 1, **i32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, at, lengths)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, mid1 = step(x, at, lengths)
    for i in range(n):
        x.copy_(qkv[:, P + i:P + i + 1])
        at.fill_(P + i)
        lengths.fill_(P + i + 1)
        g.replay()
        a, b = mid1.reshape(B, H, 64), mid.reshape(B, P + n, H, 64)[:, P + i]
        # both within the bound of their roundings: probabilities and the output, 2^-11 each, of outputs below 4
        assert float((a.double() - b.double()).abs().max()) <= 4 * 4 * 2.0 ** -11
        assert float((out[:, 0].double() - whole[:, P + i].double()).abs().max()) <= 4 * 4 * 2.0 ** -11
    assert pkg.ops.device_status() == 0


def test_calls_on_two_streams_at_once(pkg, cuda_device):
    gen = torch.Generator().manual_seed(13)
    c = _filled(pkg, gen, 40, 4, 64, 4, torch.float16, cuda_device)
    args = {n: c.get(n) for n in ("k_stats", "v_stats", "codebooks")}
    i32 = dict(dtype=torch.int32, device=cuda_device)
    table = torch.arange(40, **i32).reshape(2, 20)
    lengths = torch.tensor([1280, 900], **i32)
    q = [torch.randn(2 * n, 8, 64, generator=gen).half().to(cuda_device) for n in (1, 200)]

    def run(i):
        return pkg.ops.paged_attention(q[i], c["k_pages"], c["v_pages"], table, lengths, None, (1, 200)[i], **args)
    want = [run(0), run(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for r in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, run(i)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)
    assert pkg.ops.device_status() == 0


def test_what_is_refused(pkg, cuda_device):
    dev, ops = cuda_device, pkg.ops
    c, th = _empty_cache(4, 2, 16, 4, torch.float16, dev)
    args = {n: c[n] for n in ("k_stats", "v_stats", "codebooks")}
    i32 = dict(dtype=torch.int32, device=dev)
    q, table, lengths = torch.zeros(2, 4, 64, device=dev).half(), torch.zeros(2, 2, **i32), torch.ones(2, **i32)
    k = torch.zeros(3, 2, 64, device=dev).half()
    slots = torch.arange(3, device=dev)

    def paged(q=q, table=table, lengths=lengths, starts=None, n=1, kp=c["k_pages"], vp=c["v_pages"], **kw):
        return ops.paged_attention(q, kp, vp, table, lengths, starts, n, **{**args, **kw})
    paged()
    bad = [lambda: paged(q=q.float()), lambda: paged(q=q[:, :3]), lambda: paged(q=q[:, :, :32]), lambda: paged(q=q.cpu()), lambda: paged(table=table.long()),
           lambda: paged(lengths=lengths[:1]), lambda: paged(n=2), lambda: paged(starts=torch.zeros(2, **i32)), lambda: paged(k_stats=None),
           lambda: paged(codebooks=c["codebooks"][:, :8]), lambda: paged(scale=0.0), lambda: paged(scale=float("nan")), lambda: paged(scale=-1.0),
           lambda: paged(out=torch.empty_like(q).bfloat16()), lambda: paged(out=torch.empty(2, 5, 64, device=dev).half()), lambda: paged(n=-1),
           lambda: paged(kp=c["k_pages"][:, :, :8].contiguous(), vp=c["v_pages"][:, :, :8].contiguous()),
           lambda: paged(kp=c["k_pages"].transpose(1, 2)), lambda: paged(kp=c["k_pages"].half()),
           lambda: paged(q=q.clone().requires_grad_()),
           lambda: ops.paged_attention(q.bfloat16(), torch.zeros(4, 2, 16, 64, device=dev).half(), torch.zeros(4, 2, 16, 64, device=dev).half(), table, lengths),
           lambda: ops.kv_cache_write(k, k, slots.int(), thresholds=th, **c), lambda: ops.kv_cache_write(k, k[:2], slots, thresholds=th, **c),
           lambda: ops.kv_cache_write(k, k, slots[:2], thresholds=th, **c), lambda: ops.kv_cache_write(k, k, slots, **c),
           lambda: ops.kv_cache_write(k, k, slots, thresholds=th[:, :3], **c), lambda: ops.kv_cache_write(k[:, :1], k[:, :1], slots, thresholds=th, **c),
           lambda: ops.kv_cache_write(k, k.float(), slots, thresholds=th, **c), lambda: ops.kv_cache_write(k.cpu(), k.cpu(), slots, thresholds=th, **c),
           lambda: ops.kv_cache_read(slots, out_dtype=torch.int8, **c), lambda: ops.kv_cache_read(slots[None], **c),
           lambda: ops.cross_attention(q[None], k[None], k[None, :2]), lambda: ops.cross_attention(q[None], k[None].bfloat16(), k[None]),
           lambda: ops.cross_attention(q[None], k[None, :, :, :32], k[None, :, :, :32]), lambda: ops.cross_attention(q[None, :, :3], k[None], k[None]),
           lambda: ops.cross_attention(q[None], k[None], k[None], lengths=torch.ones(1, **i32), mask=torch.ones(1, 3, device=dev).bool()),
           lambda: ops.cross_attention(q[None], k[None], k[None], mask=torch.ones(1, 4, device=dev).bool()),
           lambda: ops.cross_attention(q[None], k[None], k[None], mask=torch.ones(1, 3, device=dev)),
           lambda: ops.cross_attention(q[None], k[None].clone().requires_grad_(), k[None])]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was taken")
    with torch.no_grad():
        paged(q=q.clone().requires_grad_())
    torch.cuda.synchronize()
    assert ops.device_status() == 0


# ---------------------------------------------------------------- both kernels on either side of where one takes over from the other
@pytest.mark.parametrize("bits,dtype", [(4, torch.float16), (3, torch.bfloat16), (2, torch.float16), (16, torch.float16), (16, torch.bfloat16)])
@pytest.mark.parametrize("new,heads,kv_heads", [(8, 2, 2), (4, 6, 2), (9, 2, 2), (16, 2, 2), (17, 1, 1), (32, 2, 2), (11, 3, 1), (33, 1, 1), (128, 1, 1), (129, 1, 1)])
def test_rows_of_a_key_head(pkg, cuda_device, bits, dtype, new, heads, kv_heads):
    """Few sequences with narrow tables, and many keys in all (one long sequence): up to 32 rows the kernels share such calls out between them."""
    _paged_check(pkg, cuda_device, bits, dtype, heads, kv_heads, 32, [300, 45], [new, min(new, 3)], seed=21)
    _paged_check(pkg, cuda_device, bits, dtype, heads, kv_heads, 64, [500] + [90] * 9, [new] * 10, seed=22, causal=False)
    far = 17000 if bits != 16 else 42000                               # keys times key heads: 136 000, 336 000
    gen = torch.Generator().manual_seed(23)
    B = 8 // kv_heads
    c = _filled(pkg, gen, 20, kv_heads, 64, bits, dtype, cuda_device)
    width = -(-far // 64)
    table = torch.full((B, width), -1, dtype=torch.int32)              # pages that do not exist but for some, up to the last
    places = torch.cat([torch.tensor([0, 1, width - 1]), 2 + torch.randperm(width - 3, generator=gen)[:13]]).sort().values
    for b in range(B):
        table[b, places] = torch.randperm(20, generator=gen)[:16].to(torch.int32)
    lengths = torch.tensor([far - 7 * b for b in range(B)], dtype=torch.int32)
    q = (1.3 * torch.randn(B * new, heads, 64, generator=gen)).to(dtype).to(cuda_device)
    out = pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table.to(cuda_device), lengths.to(cuda_device), None, new,
                                  **{n: c.get(n) for n in ("k_stats", "v_stats", "codebooks")})
    for b in range(B):
        j = (places[:, None] * 64 + torch.arange(64)).reshape(-1)
        j = j[j < lengths[b]]
        rows = torch.stack([table[b, j // 64].long(), j % 64], 1).to(cuda_device)
        (k, dk), (v, dv) = (_cached(pkg, c, w, rows) for w in "kv")
        seen = (j[None, :] <= (lengths[b] - new + torch.arange(new))[:, None]).to(cuda_device)
        want, off = _attend(q[b * new:(b + 1) * new], k, dk, v, dv, seen, 0.125, dtype, bits != 16)
        err = (out[b * new:(b + 1) * new].double() - want).abs()
        assert bool((err <= off).all()), (b, float((err / off).max()))
    assert pkg.ops.device_status() == 0


@pytest.mark.parametrize("bits,dtype", [(4, torch.bfloat16), (3, torch.float16), (2, torch.float16), (16, torch.float16)])
def test_units_that_are_cut_and_that_are_not(pkg, cuda_device, bits, dtype):
    """Contexts on both sides of where units are cut between blocks, with sequences of a token and of none between long ones."""
    for longest in (1150, 1153, 2600):
        _paged_check(pkg, cuda_device, bits, dtype, 4, 2, 16, [longest, 1, 0, 31, longest - 40, 33, 1], [1, 1, 1, 1, 2, 0, 1], seed=24)


@pytest.mark.parametrize("bits", [4, 16])
def test_more_sequences_than_threads(pkg, cuda_device, bits):
    lengths = [(7 * i) % 50 for i in range(900)]
    _paged_check(pkg, cuda_device, bits, torch.float16, 1, 1, 16, lengths, [i % 2 if i % 40 < 30 else 0 for i in range(900)], seed=25)
    _cross_check(pkg, cuda_device, torch.float16, 900, 1, 40, 1, 1, "lengths", seed=26)


def test_empty_caches_tables_and_batches(pkg, cuda_device):
    i32 = dict(dtype=torch.int32, device=cuda_device)
    for bits in (4, 16):
        c, th = _empty_cache(0, 2, 16, bits, torch.float16, cuda_device)
        args = {n: c.get(n) for n in ("k_stats", "v_stats", "codebooks")}
        x = torch.randn(3, 2, 64, device=cuda_device).half()
        slots = torch.arange(3, device=cuda_device)
        pkg.ops.kv_cache_write(x, x, slots, thresholds=th, **c)
        assert not any(bool(t.any()) for t in pkg.ops.kv_cache_read(slots, **c))
        for new in (1, 40):
            q = torch.randn(2 * new, 4, 64, device=cuda_device).half()
            for table in (torch.zeros(2, 3, **i32), torch.zeros(2, 0, **i32)):
                got = pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, torch.tensor([30, 5], **i32), None, new, **args)
                assert not bool(got.any())
            assert pkg.ops.paged_attention(q[:0], c["k_pages"], c["v_pages"], torch.zeros(0, 3, **i32), torch.zeros(0, **i32), None, new, **args).shape == (0, 4, 64)
    assert pkg.ops.device_status() == 0


def test_the_same_slot_twice(pkg, cuda_device):
    """One of the tokens, or parts of both: statistics and codes of either, and no other slot."""
    c, th = _empty_cache(2, 1, 16, 4, torch.float16, cuda_device)
    x = torch.randn(4000, 1, 64, generator=torch.Generator().manual_seed(5)).half().to(cuda_device)
    pkg.ops.kv_cache_write(x, x, torch.full((4000,), 17, device=cuda_device), thresholds=th, **c)
    got = pkg.ops.kv_cache_read(torch.arange(32, device=cuda_device), **c)
    assert bool(torch.isfinite(got[0]).all()) and int(got[0].any(-1).sum()) == 1 and int(got[1].any(-1).sum()) == 1


@pytest.mark.parametrize("bits", [4, 16])
def test_two_captured_graphs_at_once(pkg, cuda_device, bits):
    """Each graph keeps workspaces of its own: replayed side by side, with new lengths, both give what an eager call gives."""
    gen = torch.Generator().manual_seed(31)
    c = _filled(pkg, gen, 64, 2, 64, bits, torch.float16, cuda_device)
    args = {n: c.get(n) for n in ("k_stats", "v_stats", "codebooks")}
    i32 = dict(dtype=torch.int32, device=cuda_device)
    table = torch.randperm(64, generator=gen).to(torch.int32).to(cuda_device).reshape(2, 32)
    calls = []
    for new in (1, 2):
        q = torch.randn(2 * new, 8, 64, generator=gen).half().to(cuda_device)
        lengths = torch.tensor([2000, 1500], **i32)
        run = lambda q=q, lengths=lengths, new=new: pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, lengths, None, new, **args)   # noqa: E731
        run()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = run()
        calls.append((g, run, got, lengths, torch.cuda.Stream()))
    for values in ([2000, 1500], [2048, 3], [700, 0], [1, 2047]):
        want = []
        for g, run, got, lengths, s in calls:
            lengths.copy_(torch.tensor(values, dtype=torch.int32))
            want.append(run())
        torch.cuda.synchronize()
        for _ in range(4):
            for g, run, got, lengths, s in calls:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(call[2], w) for call, w in zip(calls, want))
    assert pkg.ops.device_status() == 0


@pytest.mark.parametrize("polls", [0, 1, 3])
@pytest.mark.parametrize("bits,B,n,S", [(16, 1, 40, 900), (16, 2, 300, 400), (4, 1, 40, 900), (4, 90, 200, 300)])
def test_waits_of_the_tile_kernel_that_run_out(pkg, cuda_device, bits, B, n, S, polls):
    """The kernel ends, a result that is not the whole one has left its code in the status word, and the next launch is none the worse."""
    gen = torch.Generator().manual_seed(32)
    c = _filled(pkg, gen, 2 * B + 8, 1, 512, bits, torch.float16, cuda_device)
    args = {m: c.get(m) for m in ("k_stats", "v_stats", "codebooks")}
    table = torch.arange(2 * B, dtype=torch.int32, device=cuda_device).reshape(B, 2)
    q = torch.randn(B * n, 1, 64, generator=gen).half().to(cuda_device)
    run = lambda: pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, torch.full((B,), S, dtype=torch.int32, device=cuda_device), None, n, **args)   # noqa: E731
    want = run()
    for _ in range(3):
        with pkg._cabi.option("ARCQ_POLL_LIMIT", polls):
            got = run()
        status = pkg.ops.device_status()
        assert status == 0x502 or (polls > 0 and status == 0 and torch.equal(got, want))
    assert torch.equal(run(), want) and pkg.ops.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,S", [(33, 128), (40, 129), (128, 768), (77, 769), (100, 385)])
def test_blocks_of_one_stream_and_of_two(pkg, cuda_device, dtype, n, S):
    """More key heads than multiprocessors, up to 128 rows: states on both sides of where one kernel takes over, and pieces over pages."""
    _cross_check(pkg, cuda_device, dtype, 160, n, S, 1, 1, "mask", seed=41)
    _cross_check(pkg, cuda_device, dtype, 80, n // 2, S, 4, 2, "lengths", seed=42)
    lengths = [max(1, S - (31 * i) % (S + 20)) for i in range(160)]
    _paged_check(pkg, cuda_device, 16, dtype, 1, 1, 64, lengths, [min(n, 1 + (13 * i) % (n + 3)) for i in range(160)], seed=43)


@pytest.mark.parametrize("bits,dtype", [(4, torch.float16), (3, torch.bfloat16), (16, torch.float16), (16, torch.bfloat16)])
@pytest.mark.parametrize("B,kv_heads,new", [(50, 12, 16), (50, 12, 1), (300, 6, 8), (340, 6, 17), (120, 5, 33), (40, 12, 64), (1900, 1, 3)])
@pytest.mark.parametrize("longest", [1, 130])
def test_many_short_units(pkg, cuda_device, bits, dtype, B, kv_heads, new, longest):
    """Units that warps have whole, more and fewer than warps, of different lengths, some without queries or keys."""
    lengths = [(longest - (7 * i) % (longest + 1)) for i in range(B)]
    _paged_check(pkg, cuda_device, bits, dtype, kv_heads, kv_heads, 16, lengths, [0 if i % 9 == 4 else 1 + (5 * i) % new for i in range(B)], seed=61)


@pytest.mark.parametrize("bits,dtype", [(4, torch.float16), (16, torch.bfloat16)])
@pytest.mark.parametrize("B,heads,kv_heads", [(2, 100, 100), (24, 14, 7), (64, 6, 3), (65, 6, 3)])
def test_sequences_in_the_order_of_their_work(pkg, cuda_device, bits, dtype, B, heads, kv_heads):
    """A few rounds of blocks, sequences of equal and of different work, some without queries or keys."""
    lengths = [0 if i % 13 == 5 else 150 + 90 * (i * 5 % 7) for i in range(B)]
    _paged_check(pkg, cuda_device, bits, dtype, heads, kv_heads, 64, lengths, [0 if i % 11 == 3 else 1 + 37 * (i * 3 % 5) for i in range(B)], seed=51)
    if bits == 16:
        _cross_check(pkg, cuda_device, dtype, B, 70, 400, heads, kv_heads, "lengths", seed=52)


@pytest.mark.parametrize("polls", [0, 1, 3])
@pytest.mark.parametrize("B,n,S", [(1, 40, 100), (200, 40, 700)])
def test_waits_of_one_stream_that_run_out(pkg, cuda_device, polls, B, n, S):
    gen = torch.Generator().manual_seed(33)
    q, k = (torch.randn(B, t, 1, 64, generator=gen).half().to(cuda_device) for t in (n, S))
    want = pkg.ops.cross_attention(q, k, k)
    for _ in range(3):
        with pkg._cabi.option("ARCQ_POLL_LIMIT", polls):
            got = pkg.ops.cross_attention(q, k, k)
        status = pkg.ops.device_status()
        assert status == 0x502 or (polls > 0 and status == 0 and torch.equal(got, want))
    assert torch.equal(pkg.ops.cross_attention(q, k, k), want) and pkg.ops.device_status() == 0


@pytest.mark.parametrize("bits", [4, 16])
def test_a_threads_first_calls_are_captured(pkg, cuda_device, bits):
    """Nothing has been set up in the thread: every kernel's first launch there goes into a graph, on a stream of its own."""
    import threading
    gen = torch.Generator().manual_seed(71)
    c = _filled(pkg, gen, 40, 2, 64, bits, torch.float16, cuda_device)
    args = {n: c.get(n) for n in ("k_stats", "v_stats", "codebooks")}
    i32 = dict(dtype=torch.int32, device=cuda_device)
    table, lengths = torch.arange(40, **i32).reshape(2, 20), torch.tensor([1280, 77], **i32)
    qs = {n: torch.randn(2 * n, 4, 64, generator=gen).half().to(cuda_device) for n in (1, 30, 200)}
    states = torch.randn(2, 90, 4, 64, generator=gen).half().to(cuda_device)

    def run():
        outs = [pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, lengths, None, n, **args) for n, q in qs.items()]
        return outs + [pkg.ops.cross_attention(q.reshape(2, n, 4, 64), states, states) for n, q in qs.items()]
    results = []

    def capture():
        try:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, capture_error_mode="thread_local"):
                outs = run()
            g.replay()
            torch.cuda.synchronize()
            results.append((g, outs))
        except Exception as e:                                          # noqa: BLE001  (shown by the test's own thread)
            results.append(e)
    torch.cuda.synchronize()
    t = threading.Thread(target=capture)
    t.start()
    t.join()
    assert isinstance(results[0], tuple), results[0]
    assert all(torch.equal(a, b) for a, b in zip(results[0][1], run())) and pkg.ops.device_status() == 0


def test_registers_and_workspaces_that_are_too_few(pkg, cuda_device):
    import ctypes
    import threading
    q = torch.randn(1, 200, 2, 64, device=cuda_device).half()
    k = torch.randn(1, 300, 2, 64, device=cuda_device).half()
    results = []

    def run():                                                         # the kernel is asked once a thread
        try:
            results.append(pkg.ops.cross_attention(q, k, k))
        except RuntimeError as e:
            results.append(str(e))
    for regs in (120, 128, 0):
        with pkg._cabi.option("ARCQ_LAUNCH_REGS", regs):
            t = threading.Thread(target=run)
            t.start()
            t.join()
        assert torch.is_tensor(results[-1]) if regs != 120 else "compiled for 120 registers" in results[-1]
    lib = pkg._cabi.load()
    need = lib.arcq_attention_workspace(1, 1, 2, 2)
    work, out = torch.empty(need, dtype=torch.uint8, device=cuda_device), torch.full((1, 1, 2, 64), 3.0, device=cuda_device).half()
    strides = [(ctypes.c_int64 * 3)(*t.stride()[:3]) for t in (q, k, k)]
    call = lambda bytes_, at: lib.arcq_cross_attention(q.data_ptr(), k.data_ptr(), k.data_ptr(), 1, 1, 1, 300, 2, 2, *strides, None, None, 0, 0.125,   # noqa: E731
                                                       out.data_ptr(), at, bytes_, None)
    assert call(need - 1, work.data_ptr()) == -1 and call(need, None) == -1 and bool((out == 3.0).all())
    assert call(need, work.data_ptr()) == 0
    torch.cuda.synchronize()
    assert not bool((out == 3.0).all()) and pkg.ops.device_status() == 0
    with pytest.raises(RuntimeError, match="out lies over"):
        pkg.ops.cross_attention(q, k, k, out=q)
