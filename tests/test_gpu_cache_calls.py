"""Calls that the documentation of the cache and its attentions allows, at the edges of what their arguments may say."""
import pytest
import torch

from test_gpu_cache_attention import _empty_cache, _filled

pytestmark = pytest.mark.gpu


def _args(c):
    return {n: c.get(n) for n in ("k_stats", "v_stats", "codebooks")}


@pytest.mark.parametrize("bits", [4, 16])
def test_a_bound_far_above_the_new_tokens(pkg, cuda_device, bits):
    """max_new only bounds the new tokens of a sequence where starts are given: results are those of the smallest bound, and no blocks are
    launched for rows that are not there."""
    gen = torch.Generator().manual_seed(1)
    c = _filled(pkg, gen, 20, 2, 64, bits, torch.float16, cuda_device)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    table = torch.arange(20, **i32).reshape(2, 10)
    q = torch.randn(200, 4, 64, generator=gen).half().to(cuda_device)

    def run(starts, bound, batch):
        return pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table[:batch], torch.tensor([630, 500][:batch], **i32), torch.tensor(starts, **i32), bound, **_args(c))
    one = run([0, 200], 200, 1)
    for bound in (201, 10 ** 6, 2 ** 30 - 129):
        assert torch.equal(run([0, 200], bound, 1), one), bound
    two = run([0, 150, 200], 150, 2)
    for bound in (200, 2 ** 30 - 129):
        # another number of row tiles, so keys may be split otherwise: two roundings of weights and outputs below 2
        assert float((run([0, 150, 200], bound, 2).double() - two.double()).abs().max()) <= 4 * 2 * 2.0 ** -11
    with pytest.raises(RuntimeError, match="too many"):
        run([0, 200], 2 ** 30 - 128, 1)
    assert pkg.ops.device_status() == 0


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("heads", [1, 20])                           # 4 and 80 rows a key head: both kernels
@pytest.mark.parametrize("starts,valid,zero", [
    # rows of a sequence that are as a call with it alone gives them (sequence, from, to), rows that are zero; the rest is not written
    ([0, 2, 4], [(0, 0, 2), (1, 2, 4)], []),
    ([0, 2, 10 ** 9], [(0, 0, 2)], [2, 3]),                          # the first 2 of a thousand million: they come before the context's 20 keys
    ([3, 2, 4], [(1, 2, 4)], []),                                    # backwards: no queries
    ([-5, 1, 2], [(1, 1, 2)], []),                                   # before the first row: no queries
    ([-2 ** 31, 2 ** 31 - 1, 2], [], []),
    ([2 ** 31 - 1, 4, 4], [], []),
    ([4, 9, 9], [], []),                                             # behind the last row
    ([1, 1, 4], [(1, 1, 4)], []),
    ([2, 4, 0], [(0, 2, 4)], [])])
def test_starts_that_are_not_in_order(pkg, cuda_device, bits, heads, starts, valid, zero):
    gen = torch.Generator().manual_seed(4)
    c = _filled(pkg, gen, 4, 1, 16, bits, torch.float16, cuda_device)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    table, lengths = torch.arange(4, **i32).reshape(2, 2), torch.tensor([20, 31], **i32)
    q = torch.randn(4, heads, 64, generator=gen).half().to(cuda_device)
    guarded = torch.full((4 + 64, heads, 64), 5.0, device=cuda_device).half()          # rows around out
    out = guarded[32:36]
    pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, lengths, torch.tensor(starts, **i32), 4, out=out, **_args(c))
    want = torch.full_like(guarded, 5.0)
    for b, lo, hi in valid:
        want[32 + lo:32 + hi] = pkg.ops.paged_attention(q[lo:hi], c["k_pages"], c["v_pages"], table[b:b + 1], lengths[b:b + 1], None, hi - lo, **_args(c))
    for row in zero:
        want[32 + row] = 0
    # keys may be split otherwise: two roundings of weights and outputs below 4; what is not written or zero is so exactly
    off = torch.zeros(4 + 64, 1, 1, device=cuda_device)
    for _, lo, hi in valid:
        off[32 + lo:32 + hi] = 4 * 4 * 2.0 ** -11
    assert bool(((guarded.float() - want.float()).abs() <= off).all())
    assert pkg.ops.device_status() == 0


def test_what_asks_for_gradients_is_refused(pkg, cuda_device):
    """The cache's own tensors and out, like queries, keys and values: there is no backward pass, and none is left out in silence."""
    dev, ops = cuda_device, pkg.ops
    i32 = dict(dtype=torch.int32, device=dev)
    table, lengths, slots = torch.zeros(2, 2, **i32), torch.ones(2, **i32), torch.arange(3, device=dev)
    q, k = torch.randn(2, 4, 64, device=dev).half(), torch.randn(3, 2, 64, device=dev).half()

    def calls(c, th, out=None):
        args = _args(c)
        return [lambda: ops.paged_attention(q, c["k_pages"], c["v_pages"], table, lengths, out=out, **args),
                lambda: ops.kv_cache_write(k, k, slots, thresholds=th, **c), lambda: ops.kv_cache_read(slots, **c)]
    for bits, names in ((16, ["k_pages", "v_pages"]), (4, ["k_stats", "v_stats", "codebooks"])):
        c, th = _empty_cache(4, 2, 16, bits, torch.float16, dev)
        for name in names:
            asks = {**c, name: c[name].clone().requires_grad_()}
            for f in calls(asks, th):
                with pytest.raises(RuntimeError, match="backward"):
                    f()
            with torch.no_grad():
                for f in calls(asks, th):
                    f()
    with pytest.raises(RuntimeError, match="backward"):
        calls(c, th.clone().requires_grad_())[1]()
    with pytest.raises(RuntimeError, match="backward"):
        calls(c, th, torch.empty_like(q).requires_grad_())[0]()
    with pytest.raises(RuntimeError, match="backward"):
        ops.cross_attention(q[None], k[None], k[None], out=torch.empty_like(q[None]).requires_grad_())
    for f in calls(c, th, torch.empty_like(q)):
        f()
    assert ops.device_status() == 0


@pytest.mark.parametrize("bits", [2, 4])
@pytest.mark.parametrize("tokens", [40, 1500])                       # both write kernels
@pytest.mark.parametrize("new", [1, 100])                            # both attentions
@pytest.mark.parametrize("last", ["another kernel", "codebooks", "thresholds"])
def test_codebooks_that_have_just_been_written(pkg, cuda_device, bits, tokens, new, last):
    """Fitted right before the first write, by the kernel before it or the one before that: eagerly and captured, with other levels each time,
    behind other work."""
    gen = torch.Generator().manual_seed(bits + tokens)
    pages = -(-tokens // 16)
    c, th = _empty_cache(pages, 2, 16, bits, torch.float16, cuda_device)
    base_cb, base_th = c["codebooks"].clone(), th.clone()
    k, v = (torch.randn(tokens, 2, 64, generator=gen).half().to(cuda_device) for _ in range(2))
    q = torch.randn(new, 4, 64, generator=gen).half().to(cuda_device)
    slots = torch.arange(tokens, device=cuda_device)
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    length = torch.tensor([tokens], dtype=torch.int32, device=cuda_device)
    factor, other = torch.ones((), device=cuda_device), torch.zeros(1 << 22, device=cuda_device)

    def fit_and_use():
        other.add_(1.0)
        if last == "thresholds":
            torch.mul(base_cb, factor, out=c["codebooks"])
            torch.mul(base_th, factor, out=th)
        else:
            torch.mul(base_th, factor, out=th)
            torch.mul(base_cb, factor, out=c["codebooks"])
        if last == "another kernel":
            other[:4].add_(1.0)
        pkg.ops.kv_cache_write(k, v, slots, thresholds=th, **c)
        read = pkg.ops.kv_cache_read(slots, **c)
        y = pkg.ops.paged_attention(q, c["k_pages"], c["v_pages"], table, length, None, new, **_args(c))
        return (*read, y)

    def one_by_one(f):
        c2, _ = _empty_cache(pages, 2, 16, bits, torch.float16, cuda_device)
        c2["codebooks"], th2 = base_cb * f, base_th * f
        torch.cuda.synchronize()
        pkg.ops.kv_cache_write(k, v, slots, thresholds=th2, **c2)
        read = pkg.ops.kv_cache_read(slots, **c2)
        return (*read, pkg.ops.paged_attention(q, c2["k_pages"], c2["v_pages"], table, length, None, new, **_args(c2)))
    factors = [1.0, 0.5, 1.5, 0.75] * 3
    want = {f: one_by_one(f) for f in set(factors)}
    assert not torch.equal(want[0.5][0], want[1.5][0])
    for f in factors:
        factor.fill_(f)
        assert all(torch.equal(a, b) for a, b in zip(fit_and_use(), want[f])), f
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = fit_and_use()
    for f in factors:
        factor.fill_(f)
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want[f])), f
    assert pkg.ops.device_status() == 0


@pytest.mark.parametrize("bits", [2, 3, 4])
def test_a_cache_with_codebooks_fitted_to_the_first_prompt(pkg, cuda_device, bits):
    """As a layer's are fitted: what is read back is the quantizer's reconstruction but for center and scale in fp16."""
    gen = torch.Generator().manual_seed(bits)
    k, v = ((torch.randn(300, 2, 64, generator=gen) + 0.3).half().to(cuda_device) for _ in range(2))
    fits = [pkg.codebook.calibrate_codebook(t.reshape(-1, 64), bits=bits) for t in (k, v)]
    codebooks, thresholds = (torch.stack(t) for t in zip(*fits))
    c, _ = _empty_cache(20, 2, 16, bits, torch.float16, cuda_device)
    c["codebooks"] = codebooks
    slots = torch.arange(300, device=cuda_device)
    pkg.ops.kv_cache_write(k, v, slots, thresholds=thresholds, **c)
    for i, (x, got) in enumerate(zip((k, v), pkg.ops.kv_cache_read(slots, out_dtype=torch.float32, **c))):
        want = pkg.ops.quantize_activation_dequant(x.reshape(300, 128), thresholds[i], codebooks[i], bits, 64).reshape(x.shape).double()
        st = c["kv"[i] + "_stats"][:19].permute(0, 2, 1, 3).reshape(304, 2, 2)[:300].double()
        off = 2.0 ** -11 * (st[..., :1].abs() + (want - st[..., :1]).abs()) * 1.01 + 2.0 ** -20 * want.abs() + 2.0 ** -24
        assert bool(((got.double() - want).abs() <= off).all())
