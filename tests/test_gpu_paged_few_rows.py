"""paged_attention of up to 8 rows a sequence: the weights meet the values as two bf16 summands, in the pages and in the block that
is not finished yet."""
import pytest
import torch
from kv_model import BF, D, Cache, attend, starts_of, stored

from mica_amd.kv_cache import paged_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[31], [2], [7, 30, 17], [63, 45], [32], [96, 64], [90] * 40])
@pytest.mark.parametrize("n", [1, 2, 5, 8])
def test_weights_of_two_summands(gpu, lens, n):
    """Values of +-1 that cancel and small queries, so that roundings of the weights show.  With A = sum p |v| and S keys:
    a weight's two summands leave 2^-8 of 2^-8 of it; its sum, its products' sum and their quotient are fp32 (2 (S + 8) 2^-24, the
    block's scales and the exponential's step among the 8); a score is an fp32 sum of 256 products, off by at most 256 x 2^-24 x
    sum |q k| / 16, and twice that reaches the weights; the result is rounded once, 2^-8 |ref|."""
    g = torch.Generator(device=gpu).manual_seed(sum(lens) + n)
    counts = [min(n, m) for m in lens]
    ks = [torch.randn(m, 2, D, generator=g, device=gpu).to(BF) for m in lens]
    vs = [torch.randint(0, 2, (m, 2, D), generator=g, device=gpu).mul(2).sub(1).to(BF) for m in lens]
    c = Cache(gpu, ks, vs)
    q = (torch.randn(sum(counts), 8, D, generator=g, device=gpu) / 64).to(BF)
    o = paged_attention(q, c.kv(), starts_of(counts, gpu), c.lens, c.table, longest=n).double()
    at = 0
    for b, m in enumerate(counts):
        x, k, v = q[at:at + m], stored(ks[b]), stored(vs[b])
        r, a = attend(x, k, v, lens[b] - m)
        reach = (x.float().abs().view(m, 2, 4, D).transpose(0, 1).reshape(2, -1, D) @ k.abs().permute(1, 2, 0)).max().item() / 16
        step = 2 ** -16 + 2 * (lens[b] + 8) * 2 ** -24 + 2 * 256 * 2 ** -24 * reach
        assert step < 2 ** -13.5, "sharp enough to tell one summand from two"
        assert ((o[at:at + m] - r).abs() <= 2 ** -8 * r.abs() + step * a).all()
        at += m
