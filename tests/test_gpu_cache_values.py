"""What the values in a cache may be: NaN and infinities, magnitudes far apart, and roundings that have to cancel."""
import pytest
import torch

from test_gpu_cache_attention import U, _cached, _empty_cache, _levels

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def _pages_args(c):
    return {n: c.get(n) for n in ("k_stats", "v_stats", "codebooks")}


# ---------------------------------------------------------------- NaN and infinities
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [2, 3, 4])
@pytest.mark.parametrize("tokens", [40, 1300])                      # eight lanes a group, and a lane
def test_groups_that_are_not_finite_are_read_back_as_nan(pkg, cuda_device, bits, dtype, tokens):
    gen = torch.Generator().manual_seed(tokens + bits)
    pages = -(-tokens // 16)
    x = [torch.randn(tokens, 2, 64, generator=gen).to(dtype).to(cuda_device) for _ in range(2)]
    hit = [torch.zeros(tokens, 2, dtype=torch.bool, device=cuda_device) for _ in range(2)]
    bad = [t.clone() for t in x]
    for which, token, head, at in ((0, 3, 0, {5: NAN}), (0, 17, 1, {63: INF}), (0, tokens - 1, 0, {0: -INF}), (1, 3, 1, {9: INF, 10: -INF}),
                                   (1, 4, 0, dict.fromkeys(range(64), INF)), (1, 21, 0, dict.fromkeys(range(64), NAN)), (1, 22, 1, {31: -INF, 32: NAN})):
        for i, value in at.items():
            bad[which][token, head, i] = value
        hit[which][token, head] = True
    slots = torch.randperm(pages * 16, generator=gen)[:tokens].to(cuda_device)
    got = []
    for k, v in (x, bad):
        c, th = _empty_cache(pages, 2, 16, bits, dtype, cuda_device)
        pkg.ops.kv_cache_write(k, v, slots, thresholds=th, **c)
        got.append(pkg.ops.kv_cache_read(slots, out_dtype=torch.float32, **c))
    for clean, y, h in zip(*got, hit):
        assert bool(torch.isnan(y[h]).all()), y[h][~torch.isnan(y[h])]
        assert torch.equal(y[~h], clean[~h])


def _plain(q, k, v, seen):
    """One head in 64 bits: q [n, 64], k, v [S, 64], seen [n, S] -> [n, 64]; values that are not seen do not count."""
    s = (0.125 * q.double() @ k.double().t()).masked_fill(~seen, -INF)
    w = torch.softmax(s, -1)
    return torch.stack([w[i][seen[i]] @ v.double()[seen[i]] for i in range(q.shape[0])])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [2, 3, 4, 16])
@pytest.mark.parametrize("new", [1, 2, 130])                         # few rows, and the tile kernel
@pytest.mark.parametrize("which,value", [("k", NAN), ("k", INF), ("v", NAN), ("v", INF), ("v", -INF)])
def test_what_is_not_finite_and_seen_shows(pkg, cuda_device, bits, dtype, new, which, value):
    """NaN and infinities where the formula has them, and nowhere else: not with another key head and not in another sequence."""
    gen = torch.Generator().manual_seed(new)
    H, Hk, page, L, at = 4, 2, 16, 150, 20                             # every query sees token 20
    pages = 20
    x = {n: (0.5 * torch.randn(pages * page, Hk, 64, generator=gen)).to(dtype).to(cuda_device) for n in "kv"}
    table = torch.randperm(pages, generator=gen).to(torch.int32).reshape(2, 10)
    slot = int(table[0, at // page]) * page + at % page
    q = (0.5 * torch.randn(2 * new, H, 64, generator=gen)).to(dtype).to(cuda_device)
    lengths = torch.full((2,), L, dtype=torch.int32, device=cuda_device)
    outs = []
    for planted in (False, True):
        if planted:
            x[which][slot, 0, 7] = value
        c, th = _empty_cache(pages, Hk, page, bits, dtype, cuda_device)
        pkg.ops.kv_cache_write(x["k"], x["v"], torch.arange(pages * page, device=cuda_device), thresholds=th, **c)
        outs.append(pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table.to(cuda_device), lengths, None, new, **_pages_args(c)))
    clean, got = outs
    assert torch.equal(got[new:], clean[new:]) and torch.equal(got[:new, 2:], clean[:new, 2:])
    j = torch.arange(L)
    rows = torch.stack([table[0][j // page].long(), j % page], 1).to(cuda_device)
    k, v = (_cached(pkg, c, n, rows)[0][:, 0] for n in "kv")
    seen = (j[None] <= (L - new + torch.arange(new))[:, None]).to(cuda_device)
    for h in range(2):
        want = _plain(q[:new, h], k, v, seen)
        assert not bool(torch.isfinite(want).all()) or (bits, which, value) == (16, "k", INF)      # a score of -inf has no weight
        y = got[:new, h].double()
        assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y[torch.isinf(want)], want[torch.isinf(want)])
        fine = torch.isfinite(want)
        # scores below 8 * 64 / 8 * 2^-10 off, roundings of weights and outputs: far below a tenth of values of 0.5
        assert bool(((y - want)[fine].abs() <= 0.05).all())
    assert pkg.ops.device_status() == 0


@pytest.mark.parametrize("bits", [2, 3, 4, 16])
@pytest.mark.parametrize("new", [2, 9, 130])
def test_a_later_key_that_is_nan_has_no_effect_on_earlier_queries(pkg, cuda_device, bits, new):
    gen = torch.Generator().manual_seed(5)
    x = [torch.randn(160, 1, 64, generator=gen).half().to(cuda_device) for _ in range(2)]
    q = torch.randn(new, 2, 64, generator=gen).half().to(cuda_device)
    table = torch.arange(10, dtype=torch.int32, device=cuda_device)[None]
    length = torch.tensor([150], dtype=torch.int32, device=cuda_device)
    outs = []
    for planted in (False, True):
        if planted:
            x[0][149, 0, 3] = NAN
        c, th = _empty_cache(10, 1, 16, bits, torch.float16, cuda_device)
        pkg.ops.kv_cache_write(x[0], x[1], torch.arange(160, device=cuda_device), thresholds=th, **c)
        outs.append(pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, length, None, new, **_pages_args(c)))
    assert torch.equal(outs[1][:-1], outs[0][:-1]) and bool(torch.isnan(outs[1][-1]).all())


# ---------------------------------------------------------------- roundings of levels
@pytest.mark.parametrize("bits", [2, 3, 4])
@pytest.mark.parametrize("keys", [1, 2, 3, 8, 16, 24, 32])
def test_roundings_of_levels_have_no_direction(pkg, cuda_device, bits, keys):
    """Few rows over packed pages: a level is rounded to fp16 up or down by fixed shares t of the way between its neighbours, which is off by
    1/2 - t units on average.  Shares lie evenly about 1/2 from the first keys on: 1/16 for single keys at most, 0 for sets of four and more.

    Queries of zero weigh all keys alike, centers are 0, scales 1: an output is the mean of its keys' levels.  Its error in units of the
    levels' last places, averaged over 100 codebooks of 2^bits levels each: 0.29 / 20 (2 bits) from the average, four times that allowed."""
    gen = torch.Generator().manual_seed(100 * bits + keys)
    pages, heads, total, count = 2, 12, 0.0, 0
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    length = torch.tensor([keys], dtype=torch.int32, device=cuda_device)
    q = torch.zeros(1, heads, 64, device=cuda_device).half()
    rows = torch.stack([torch.arange(keys) // 16, torch.arange(keys) % 16], 1).to(cuda_device)
    for _ in range(100):
        c, _ = _empty_cache(pages, heads, 16, bits, torch.float16, cuda_device)
        c["codebooks"] = (0.3 + 2 * torch.rand(2, 2 ** bits, generator=gen)).to(cuda_device)
        for n in "kv":
            c[n + "_pages"].copy_(torch.randint(0, 256, c[n + "_pages"].shape, generator=gen).to(torch.uint8))
            c[n + "_stats"][..., 1] = 1.0
        got = pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, length, None, 1, **_pages_args(c))[0].double()
        v = _cached(pkg, c, "v", rows)[0]
        unit = torch.exp2(torch.floor(torch.log2(v)) - 10).mean(0)
        total += float(((got - v.mean(0)) / unit).sum())
        count += got.numel()
    assert abs(total / count) <= (1 / 16 if keys < 4 else 0.0) + 4 * 0.29 / 20


# ---------------------------------------------------------------- values of very different sizes
@pytest.mark.parametrize("bits", [2, 3, 4])
@pytest.mark.parametrize("new", [1, 2])
@pytest.mark.parametrize("L,at", [(20, 0), (32, 31), (32, 5), (77, 76), (77, 33)])
def test_a_large_value_that_hardly_counts_costs_the_others_nothing(pkg, cuda_device, bits, new, L, at):
    """Few rows: one value ten million times the others, with a weight of e^-60 or not seen at all (the last token, by the query before it).

    Keys of the others are 0 as good as exactly, so they weigh alike, 1 / n each.  The bound: a level's rounding (`_cached`), a weight times scale
    rounded to fp16 (2^-11, or 2^-25 of the largest of the call's steps, exponents a step has up to 2^6 apart and a maximum's lag of 2^8 on
    the safe side: n 2^-18 of it), scores 2^-12, sums n 2^-23, and the output's rounding, subnormal below 2^-14."""
    gen = torch.Generator().manual_seed(L + at)
    sign = torch.where(torch.rand(64, generator=gen) < 0.5, -1.0, 1.0)
    k = torch.zeros(128, 1, 64)
    k[at] = -8 * sign
    v = 0.003 * torch.randn(128, 1, 64, generator=gen)
    v[at] = 2.5e4 * torch.randn(64, generator=gen).clamp(-2, 2)
    k, v = k.half().to(cuda_device), v.half().to(cuda_device)
    c, th = _empty_cache(8, 1, 16, bits, torch.float16, cuda_device)
    pkg.ops.kv_cache_write(k, v, torch.arange(128, device=cuda_device), thresholds=th, **c)
    q = (2 * sign).expand(new, 1, 64).half().contiguous().to(cuda_device)
    table = torch.arange(8, dtype=torch.int32, device=cuda_device)[None]
    got = pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, torch.tensor([L], dtype=torch.int32, device=cuda_device), None, new, **_pages_args(c))
    j = torch.arange(L)
    rows = torch.stack([j // 16, j % 16], 1).to(cuda_device)
    (kk, _), (vv, ev) = ((a[:, 0], b[:, 0]) for a, b in (_cached(pkg, c, n, rows) for n in "kv"))
    scale = c["v_stats"][:, 0, :, 1].reshape(-1)[:L].double()
    for i in range(new):
        seen = (j <= L - new + i).to(cuda_device)
        w = torch.softmax((0.125 * q[i, 0].double() @ kk.t()).masked_fill(~seen, -INF), -1)
        assert float(w[at]) < 1e-20
        want = w @ vv
        off = w @ ev + (2.0 ** -11 + 2.0 ** -12 + L * 2.0 ** -23) * (w @ vv.abs())
        off = off + L * 2.0 ** -18 * (w * scale).max() * c["codebooks"][1].abs().max() + U[torch.float16] * want.abs() + 2.0 ** -25
        err = (got[i, 0].double() - want).abs()
        assert bool((err <= 1.05 * off).all()), (i, float((err / off).max()))


@pytest.mark.parametrize("new", [1, 140])
def test_queries_of_bf16_at_the_ends_of_their_range(pkg, cuda_device, new):
    """Over packed keys a row of queries is scaled into fp16's range by a power of two; 2^120 needs more than 2^-100, and 2^-100 more than 2^100."""
    gen = torch.Generator().manual_seed(1)
    c, th = _empty_cache(8, 2, 32, 4, torch.bfloat16, cuda_device)
    x = [torch.randn(256, 2, 64, generator=gen).bfloat16().to(cuda_device) for _ in range(2)]
    pkg.ops.kv_cache_write(x[0], x[1], torch.arange(256, device=cuda_device), thresholds=th, **c)
    table = torch.arange(8, dtype=torch.int32, device=cuda_device)[None]
    length = torch.tensor([250], dtype=torch.int32, device=cuda_device)
    q = torch.randn(new, 4, 64, generator=gen).bfloat16().to(cuda_device)

    def run(e):
        return pkg.ops.paged_attention(q * 2.0 ** e, c["k_pages"], c["v_pages"], table, length, None, new, scale=0.125 * 2.0 ** -e, **_pages_args(c))
    want = run(0)
    assert bool(torch.isfinite(want).all())
    for e in (-100, 100, 120):
        assert torch.equal(run(e), want), e


@pytest.mark.parametrize("bits", [2, 3, 4])
@pytest.mark.parametrize("new", [2, 9, 40, 130, 300])
@pytest.mark.parametrize("at", [-1, -2, "half"])
@pytest.mark.parametrize("both", [False, True])
def test_a_later_value_that_is_nan_has_no_effect_on_earlier_queries(pkg, cuda_device, bits, new, at, both):
    """Packed pages: the queries that see a value with a NaN are NaN, the others are what they are without it."""
    at = 349 - (new // 2 if at == "half" else -at - 1)
    gen = torch.Generator().manual_seed(5)
    x = [torch.randn(352, 1, 64, generator=gen).half().to(cuda_device) for _ in range(2)]
    q = torch.randn(new, 2, 64, generator=gen).half().to(cuda_device)
    table = torch.arange(22, dtype=torch.int32, device=cuda_device)[None]
    length = torch.tensor([350], dtype=torch.int32, device=cuda_device)
    outs = []
    for planted in (False, True):
        if planted:
            x[1][at, 0, 3] = INF
            if both:
                x[1][349, 0, 9] = NAN
        c, th = _empty_cache(22, 1, 16, bits, torch.float16, cuda_device)
        pkg.ops.kv_cache_write(x[0], x[1], torch.arange(352, device=cuda_device), thresholds=th, **c)
        outs.append(pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, length, None, new, **_pages_args(c)))
    sees = torch.arange(new) >= at - (350 - new)
    assert bool(torch.isnan(outs[1][sees.to(cuda_device)]).all())
    earlier = (~sees).to(cuda_device)
    # the few-row kernel's exponents may be taken against another maximum: two roundings of weights and outputs below 4
    assert bool(((outs[1][earlier].double() - outs[0][earlier].double()).abs() <= 4 * 4 * 2.0 ** -11).all())
    assert pkg.ops.device_status() == 0
