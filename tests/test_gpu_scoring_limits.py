"""The scoring operators at the ends of their ranges."""
import math

import pytest
import torch
from test_gpu_tree_window import check, heads, window_sees

from mica_amd.attention import window_attention
from mica_amd.readout import token_logprobs

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_grid_holds(gpu):
    """2^26 workgroups of 64 threads are 2^32 work-items, one more than a grid may have."""
    T = 2 ** 26 + 5
    x = torch.zeros(T, 2, dtype=torch.bfloat16, device=gpu)
    x[:, 1] = (torch.arange(T, device=gpu) % 97).to(torch.bfloat16) / 16 - 3
    tokens = (torch.arange(T, device=gpu) % 2).int()
    out = token_logprobs(x, tokens, 1)
    lp = torch.log_softmax(x[:97].double(), 1).tile(T // 97 + 1, 1)[:T]
    want = torch.where(tokens == 0, lp[:, 0], lp[:, 1])
    # two terms: a few fp32 steps of values below 4
    assert ((out.logprobs.double() - want).abs() <= 2 ** -20).all()
    assert torch.equal(out.top_ids[:, 0], (x[:, 1] > 0).long())
    assert ((out.top_logprobs[:, 0].double() - lp.amax(1)).abs() <= 2 ** -20).all()
    assert ((out.entropy.double() + (lp.exp() * lp).sum(1)).abs() <= 2 ** -20).all()


def test_a_top_that_no_int_holds(gpu):
    x, tokens = torch.zeros(2, 50, device=gpu), torch.zeros(2, dtype=torch.long, device=gpu)
    for top in (2 ** 40, 2 ** 70, -2 ** 70):
        with pytest.raises(ValueError):
            token_logprobs(x, tokens, top)


@pytest.mark.parametrize("n,lens", [(300, [1, 40, 0]), (64, [1, 40, 0]), (200, [199, 130, 3])])
def test_window_blocks_before_the_first_key(gpu, n, lens):
    """Blocks of 32 queries of which none, or only the last ones, have a key: zeros before it, and nothing of the keys after a
    block's last position, whatever they hold."""
    q, _, _, k, v = heads(gpu, n, 3, n, 4, 400)
    kept = k.clone(), v.clone()
    for b, length in enumerate(lens):
        k[b, length:], v[b, length:] = math.nan, math.inf
    v[0, lens[0] - 1], k[0, lens[0] - 1], kept[1][0, lens[0] - 1] = math.inf, 1.0, math.inf      # seen by the last query alone
    kept[0][0, lens[0] - 1] = 1.0
    o = window_attention(q, k, v, 33, 2, kv_len=torch.tensor(lens, dtype=torch.int32, device=gpu))
    check(o, q, *kept, window_sees(3, n, 400, 33, 2, lens, gpu))
    assert torch.isinf(o[0, -1]).all() and torch.isfinite(o[0, :-1]).all()
    for b, length in enumerate(lens):
        assert not o[b, :n - length].any()
