"""Tree and window attention where a sequence's keys are divided over workgroups, against float64.

Every size here has a workspace, i.e. partial states that are written and joined: asserted for each, so that a change of the
division cannot take a case off that path unseen.  The bound is the one of the undivided forms (derived beside ``check``): the
join multiplies by fp32 weights and adds up to 64 parts or as many as there are runs in a sequence, each off by 2^-22 at most,
which is within the 2^-11 A that the scores' sums are given there and use four fifths of."""
import math

import pytest
import torch
from test_gpu_tree_window import check, heads, random_parents, tree_sees, window_sees

from mica_amd import _lib
from mica_amd.attention import tree_attention, tree_masks, window_attention

pytestmark = pytest.mark.gpu


def counts(lens, gpu):
    return None if lens is None else torch.tensor(lens, dtype=torch.int32, device=gpu)


def tree(q, k, v, kc, vc, par, lens, gpu):
    assert _lib.load().mica_attention_tree_workspace_bytes(*q.shape[:2], k.shape[2], kc.shape[1]) > 0, "this size is not divided"
    return tree_attention(q, k, v, tree_masks(par, gpu), (kc, vc), counts(lens, gpu))


def window(q, k, v, width, sinks, lens, gpu):
    need = _lib.load().mica_attention_window_workspace_bytes(*q.shape[:2], *k.shape[1:3], width, sinks)
    assert need > 0, "this size is not divided"
    return window_attention(q, k, v, width, sinks, kv_len=counts(lens, gpu))


@pytest.mark.parametrize("B,N,HK,C,lens", [
    (9, 30, 2, 2900, [2900, 0, 31, 2899, 1200, 33, 640, 5, 2050]), (9, 60, 2, 2900, [2900, 0, 31, 2899, 1200, 33, 640, 5, 2050]),
    (9, 60, 2, 2900, None), (1, 65, 4, 1000, None), (2, 100, 4, 3000, [3000, 17]), (3, 255, 4, 3001, [3001, 1500, 0]),
    (2, 500, 4, 3000, [2999, 64])])
def test_tree(gpu, B, N, HK, C, lens):
    q, k, v, kc, vc = heads(gpu, N + C, B, N, HK, C)
    par = [random_parents(N, 5 * b + N, absent=b % 2 == 1) for b in range(B)]
    o = tree(q, k, v, kc, vc, par, lens, gpu)
    check(o, q, torch.cat((kc, k), 1), torch.cat((vc, v), 1), tree_sees(par, lens or [C] * B, C, gpu))


@pytest.mark.parametrize("ragged", [True, False])
@pytest.mark.parametrize("N,B,HK,C", [(3, 140, 4, 2700), (30, 129, 4, 5300), (60, 65, 4, 5300)])
def test_tree_more_sequences_than_runs(gpu, N, B, HK, C, ragged):
    """The join goes by the runs' beginnings; with all keys of every sequence, the runs are found without lengths."""
    q, k, v, kc, vc = heads(gpu, N, B, N, HK, C)
    lens = None
    if ragged:
        lens = torch.randint(0, 70, (B,), generator=torch.Generator().manual_seed(N)).tolist()
        for b in (0, 1, 62, 63, 64, B - 1):
            lens[b] = C - b
    par = [random_parents(N, b) for b in range(B)]
    o = tree(q, k, v, kc, vc, par, lens, gpu)
    full = lens or [C] * B
    for lo in range(0, B, 16):      # (the reference a few sequences at a time)
        at = slice(lo, lo + 16)
        check(o[at], q[at], torch.cat((kc[at], k[at]), 1), torch.cat((vc[at], v[at]), 1), tree_sees(par[at], full[at], C, gpu))


@pytest.mark.parametrize("B,n,S,HK,width,sinks,lens", [
    (2, 200, 4000, 4, 2000, 40, [4000, 3333]), (1, 1024, 8192, 4, 4096, 4, None), (2, 200, 3000, 4, 1500, 33, [3000, 90]),
    (3, 70, 2500, 4, 1111, 64, [2500, 71, 0]), (2, 300, 2000, 2, 1800, 100, [2000, 1]), (1, 90, 4000, 4, 1000, 2500, None),
    (9, 30, 2900, 2, 1700, 4, [2900, 0, 31, 2899, 1200, 33, 640, 5, 2050]), (2, 60, 4000, 4, 4000, 0, [4000, 12]),
    (9, 60, 2900, 2, 1700, 40, [2900, 0, 31, 2899, 1200, 33, 640, 5, 2050]), (9, 60, 2900, 2, 1700, 0, None)])
def test_window(gpu, B, n, S, HK, width, sinks, lens):
    q, _, _, k, v = heads(gpu, S + n, B, n, HK, S)
    o = window(q, k, v, width, sinks, lens, gpu)
    check(o, q, k, v, window_sees(B, n, S, width, sinks, lens or [S] * B, gpu))


def test_window_more_sequences_than_runs(gpu):
    B, n, S = 140, 3, 4000
    q, _, _, k, v = heads(gpu, 5, B, n, 4, S)
    lens = torch.randint(0, 70, (B,), generator=torch.Generator().manual_seed(1)).tolist()
    for b in (0, 63, 64, 100, 139):
        lens[b] = S - b
    for given in (lens, None):
        o = window(q, k, v, 3000, 7, given, gpu)
        sees = window_sees(B, n, S, 3000, 7, given or [S] * B, gpu)
        for lo in range(0, B, 20):
            at = slice(lo, lo + 20)
            check(o[at], q[at], k[at], v[at], sees[at])


@pytest.mark.parametrize("N", [5, 12, 20, 40, 64, 100, 255])
def test_tree_values_not_finite(gpu, N):
    """inf and NaN in nodes, in padding, past the cached keys and in the last cached key (a part's last tile, that a mask
    ends in sequence 2 and none in sequence 0): to who sees them through the join, and into no other sequence of the run."""
    B, C = 4, 2000
    lens = [1984, 777, 1003, 1500]
    q, k, v, kc, vc = heads(gpu, 21, B, N, 4, C)
    par = [random_parents(N, 2), random_parents(N, 3, absent=True), random_parents(N, 4, absent=True), random_parents(N, 5)]
    for b in (1, 2):
        if -2 not in par[b]:
            par[b][N - 1] = -2
    v[0, N // 2, 1, 7], v[0, N - 1, 2, 200], v[0, N // 3, 3, 40] = math.inf, -math.inf, math.nan
    v[0, 0, 0, 3], v[0, N - 1, 0, 3] = math.inf, -math.inf
    vc[0, 1983, 0, 9], vc[0, 5, 1, 7], vc[2, 1002, 2, 11], vc[2, 400, 2, 11] = math.inf, -math.inf, math.inf, -math.inf
    vc[2, 1002, 3, 50], vc[2, 17, 0, 60] = math.nan, -math.inf
    kept = [t.clone() for t in (q, kc, k, vc)]       # what is written from here on nobody sees
    for b in (1, 2):
        for i, p in enumerate(par[b]):
            if p == -2:
                q[b, i], k[b, i], v[b, i] = math.nan, math.inf, math.nan
    for b in (1, 2):
        kc[b, lens[b]:], vc[b, lens[b]:] = math.nan, math.inf
    o = tree(q, k, v, kc, vc, par, lens, gpu)
    check(o, kept[0], torch.cat(kept[1:3], 1), torch.cat((kept[3], v), 1), tree_sees(par, lens, C, gpu))
    assert torch.isfinite(o[3]).all() and torch.isfinite(o[1]).all()
    for b in (1, 2):
        assert not o[b, [i for i, p in enumerate(par[b]) if p == -2]].any()


@pytest.mark.parametrize("n", [3, 15, 30, 60, 90, 200])
def test_window_values_not_finite(gpu, n):
    """In keys that a part of the queries sees (behind the window's beginning, at its end), in a sink, and past the keys."""
    B, S, width = 3, 4000, 2000
    lens = [4000, 3001, 2500]
    q, _, _, k, v = heads(gpu, 22, B, n, 4, S)
    for b, length in enumerate(lens[:2]):
        first = length - n                           # the first query's position; it sees from first - width + 1 on
        v[b, first - width + 1, 0, 5], v[b, first - width, 0, 6] = math.inf, math.inf       # the first query alone; none
        v[b, first - width + 1 + n // 2, 1, 9], v[b, length - 1 - n // 3, 1, 9] = math.nan, math.inf
        v[b, length - 1, 3, 100], v[b, first - 70, 3, 100] = -math.inf, math.inf
    v[0, 2, 2, 77] = -math.inf
    kept_k, kept_v = k.clone(), v.clone()            # what is written from here on nobody sees, but for the last query of 0
    k[1, 3001:], v[1, 3001:] = math.nan, math.inf
    k[0, 3999] = math.nan
    o = window(q, k, v, width, 5, lens, gpu)
    sees = window_sees(B, n, S, width, 5, lens, gpu)
    assert torch.isnan(o[0, -1]).all()               # its own key is NaN
    sees[0, -1] = False
    o[0, -1] = 0.0
    check(o, q, kept_k, kept_v, sees)
    assert torch.isfinite(o[2]).all()


@pytest.mark.parametrize("N", [5, 60, 100])
def test_replays_with_other_lengths(gpu, N):
    """A captured graph whose lengths move the runs and parts, with eager calls between."""
    q, k, v, kc, vc = heads(gpu, 23, 3, N, 4, 1500)
    par = [random_parents(N, b, absent=b == 1) for b in range(3)]
    masks, lens = tree_masks(par, gpu), counts([1500, 40, 900], gpu)
    call = lambda: (tree_attention(q, k, v, masks, (kc, vc), lens), window_attention(q, kc, vc, 1100, 9, kv_len=lens))  # noqa: E731
    tree(q, k, v, kc, vc, par, [1500, 40, 900], gpu)
    window(q, kc, vc, 1100, 9, [1500, 40, 900], gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=gpu))
        lens.copy_(torch.tensor([1500 - 401 * i, 33 * i, 900 - 7 * i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(call(), out))
        full = lens.tolist()
        check(out[0], q, torch.cat((kc, k), 1), torch.cat((vc, v), 1), tree_sees(par, full, 1500, gpu))
        check(out[1], q, kc, vc, window_sees(3, N, 1500, 1100, 9, full, gpu))


def test_the_same_bits_at_every_call(gpu):
    """The division goes by the lengths alone and the join adds in one order: no call differs from the one before."""
    for B, N, C in ((3, 5, 1500), (9, 30, 2900), (9, 60, 2900), (2, 255, 3000)):
        q, k, v, kc, vc = heads(gpu, N, B, N, 4, C)
        par, lens = [random_parents(N, b) for b in range(B)], [C - 211 * b for b in range(B)]
        first = tree(q, k, v, kc, vc, par, lens, gpu), window(q, kc, vc, C * 3 // 4, 4, lens, gpu)
        for _ in range(5):
            assert torch.equal(tree(q, k, v, kc, vc, par, lens, gpu), first[0])
            assert torch.equal(window(q, kc, vc, C * 3 // 4, 4, lens, gpu), first[1])
