"""packed_attention on both sides of the rule that divides a block's keys (the bound is derived beside kv_model.check)."""
import pytest
import torch
from kv_model import BF, D, attend, check, starts_of

from mica_amd.attention import packed_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts,HK", [
    ([2017], 4), ([2018], 4), ([2048], 4), ([2500], 4), ([2600], 4), ([900, 900], 4), ([1000, 500], 4), ([1500] + [50] * 10, 4),
    ([5000], 2), ([1000] * 6, 1), ([1500] + [50] * 50, 1)])
@pytest.mark.parametrize("hint", [False, True])
def test_against_float64(gpu, counts, HK, hint):
    g = torch.Generator(device=gpu).manual_seed(sum(counts))
    q, k, v = torch.randn(sum(counts), 6 * HK, D, generator=g, device=gpu).to(BF).split((4 * HK, HK, HK), dim=1)
    o = packed_attention(q, k, v, starts_of(counts, gpu), longest=max(counts) if hint else None)
    at = 0
    for n in counts:
        check(o[at:at + n], *attend(q[at:at + n], k[at:at + n], v[at:at + n], 0))
        at += n
