"""Calls that the documentation of the cache and its attentions allows, at the edges of what their arguments may say."""
import pytest
import torch

from test_gpu_cache_attention import _filled

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
