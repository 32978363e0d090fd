"""Queries all of whose keys score -inf have no softmax: NaN, as causal_gqa_attention gives; not the zeros of a query that
sees no key."""
import math

import pytest
import torch
from test_gpu_tree_window import check, heads, random_parents, tree_sees, window_sees

from mica_amd.attention import causal_gqa_attention, tree_attention, tree_masks, window_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,C", [(6, 0), (6, 40), (6, 1500), (14, 1500), (30, 1500), (60, 1500), (100, 40), (100, 3000)])
def test_tree(gpu, N, C):
    """Sequence 0: every key; 1: the cached keys alone, which then have no weight; 2: the cached keys and some nodes."""
    q, k, v, kc, vc = heads(gpu, N, 3, N, 4, C)
    q[..., 3] = 1.0
    par = [random_parents(N, 7, absent=True), random_parents(N, 8), random_parents(N, 9, absent=True)]
    par[0][N - 1] = -2
    sees = tree_sees(par, [0, 0, 0], C, gpu)
    low = torch.arange(N, device=gpu) % 3 == 0
    k[0, :, :, 3] = k[2, low, :, 3] = -math.inf
    kc[..., 3] = -math.inf
    o = tree_attention(q, k, v, tree_masks(par, gpu), (kc, vc) if C else None)
    some = sees[:, :, C:].any(2)
    some[0] = False
    some[2] = sees[2, :, C:][:, ~low].any(1)       # a key of another score
    present = torch.tensor(par, device=gpu) >= -1
    assert torch.isnan(o[present & ~some]).all() and (present & ~some)[0].any() and (present & ~some)[2].any()
    assert not o[~present].any()
    sees[2, :, C:][:, low] = False
    sees &= some[:, :, None]
    o[present & ~some] = 0.0
    check(o, q, torch.cat((torch.zeros_like(kc), torch.where(torch.isfinite(k), k, 0.0)), 1), torch.cat((vc, v), 1), sees)


@pytest.mark.parametrize("n,width", [(1, 50), (5, 900), (40, 30), (90, 40), (90, 1300)])
def test_window(gpu, n, width):
    q, _, _, k, v = heads(gpu, n, 2, n, 4, 1500)
    q[..., 3] = 1.0
    k[0, :, :, 3] = -math.inf
    lens = [1500, n // 2]
    o = window_attention(q, k, v, width, 3, kv_len=torch.tensor(lens, dtype=torch.int32, device=gpu))
    assert torch.isnan(o[0]).all() and not o[1, :n - n // 2].any()
    sees = window_sees(2, n, 1500, width, 3, lens, gpu)
    check(o[1:], q[1:], k[1:], v[1:], sees[1:])


def test_as_causal_attention(gpu):
    q, k, v = heads(gpu, 3, 1, 40, 4)
    q[..., 3] = 1.0
    k[..., 3] = -math.inf
    assert torch.isnan(causal_gqa_attention(q, k, v)).all() and torch.isnan(window_attention(q, k, v, 40)).all()
