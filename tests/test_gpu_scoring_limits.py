"""The scoring operators at the ends of their ranges."""
import math

import pytest
import torch
from test_gpu_tree_window import check, heads, window_sees

from mica_amd import _lib
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


@pytest.mark.parametrize("n", [5, 100])
def test_a_window_of_the_largest_int(gpu, n):
    """Through the C entry, which does not cut it to the keys: positions before the first key, and window and sinks beyond."""
    q, _, _, k, v = heads(gpu, 9 + n, 2, n, 4, 300)
    lens = [300, n // 2]
    t = torch.tensor(lens, dtype=torch.int32, device=gpu)
    L, big = _lib.load(), 2 ** 31 - 1
    for window, sinks in ((big, 0), (big, big), (2, big)):
        o = torch.empty_like(q, memory_format=torch.contiguous_format)
        need = L.mica_attention_window_workspace_bytes(2, n, 300, 4, window, sinks)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=gpu)
        st = lambda x: (x.data_ptr(), x.stride(0), x.stride(2), x.stride(1))  # noqa: E731
        assert L.mica_attention_window(*st(q), *st(k), *st(v), *st(o), 2, n, 300, 16, 4, 256, 1 / 16, window, sinks, t.data_ptr(),
                                       ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
        check(o, q, k, v, window_sees(2, n, 300, big, 0, lens, gpu))


@pytest.mark.parametrize("top", [1, 5, 31, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("parts", [2, 7, 31, 32, 33, 64])
def test_the_join_of_every_order_of_parts(gpu, parts, dtype, top):
    """Parts of one block each (16 KB) whose best keys rise, fall, lie in one part or one in each; the last part with all its
    keys, one, or none of its own but the row's end."""
    block = 16384 // dtype.itemsize
    for V in (parts * block, (parts - 1) * block + 8, (parts - 1) * block + 8 + 3):
        at = torch.arange(V, device=gpu)
        x = torch.randn(5, V, generator=torch.Generator(device=gpu).manual_seed(parts), device=gpu)
        x[0] += at // block * 8                                # rising by parts
        x[1] -= at // block * 8
        x[2, V // 2:V // 2 + 40] += 20                         # one part has them all (or two)
        x[3, ::block] += 20                                    # one in each
        x[4] = torch.where(at // block % 3 == 1, -math.inf, x[4])
        x = x.to(dtype)
        out = token_logprobs(x, at[:5], top)
        assert torch.equal(out.top_ids, torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top])
