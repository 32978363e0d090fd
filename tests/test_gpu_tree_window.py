"""attention.tree_attention and attention.window_attention against attention in float64 with an explicit mask.

Tolerance: each weight is rounded to bf16 (half a step, 2^-8) before the product with v, the result once more; the scores
are fp32 sums of 256 products (off by at most 256 x 2^-24 x sum |q k| / 16, about 2e-4 for unit normal heads) and twice that
reaches the weights.  With A = sum p |v|:  |o - ref| <= 2^-8 (A + |ref|) + 2^-11 A."""
import math

import pytest
import torch

from mica_amd import attention, int8_kernels
from mica_amd.attention import causal_gqa_attention, tree_attention, tree_masks, window_attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def ref(q, k, v, sees, scale=None):
    """q [B, n, HQ, 256], k / v [B, S, HK, 256], sees [B, n, S] -> (o, A) float64; zeros where nothing is seen.  Keys that
    a query does not see take no part, whatever they hold."""
    B, n, HQ, D = q.shape
    g = HQ // k.shape[2]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    if not k.shape[1]:
        return o, a
    for b in range(B):
        for h in range(HQ):
            z = q[b, :, h].double() @ k[b, :, h // g].double().t() * (1 / math.sqrt(D) if scale is None else scale)
            z = torch.where(sees[b], z, -math.inf)
            m = z.amax(1, keepdim=True)
            w = torch.exp(z - torch.where(torch.isfinite(m), m, 0.0))
            w = torch.where(sees[b], w, 0.0)
            t = w.sum(1, keepdim=True)
            w = torch.where(t > 0, w / t, 0.0)
            vv = v[b, :, h // g].double()
            if not torch.isfinite(vv).all():     # 0 x inf: by key
                odd = ~torch.isfinite(vv)
                fine = torch.where(odd, 0.0, vv)
                o[b, :, h], a[b, :, h] = w @ fine, w @ fine.abs()
                for key in odd.any(1).nonzero()[:, 0].tolist():
                    o[b, :, h] += torch.where((w[:, key:key + 1] > 0) & odd[key], w[:, key:key + 1] * vv[key], 0.0)
                continue
            o[b, :, h], a[b, :, h] = w @ vv, w @ vv.abs()
    return o, a


def check(got, q, k, v, sees, scale=None):
    o, a = ref(q, k, v, sees, scale)
    got = got.double()
    odd = ~torch.isfinite(o)
    assert torch.equal(odd, ~torch.isfinite(got)), "values that are not finite reach other rows than those that see them"
    assert torch.equal(torch.isnan(o), torch.isnan(got))
    d = torch.where(odd, 0.0, got - o).abs() - (2 ** -8 * (a + o.abs()) + 2 ** -11 * a)
    assert (torch.where(odd, 0.0, d) <= 0).all(), f"off by {d.max():.3g} more than the roundings allow"


def heads(gpu, seed, B, n, HK, *keys):
    g = torch.Generator(device=gpu).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=gpu).to(BF)  # noqa: E731
    out = list(rn(B, n, 6 * HK, 256).split((4 * HK, HK, HK), dim=2))
    return out + [rn(B, c, HK, 256) for c in keys for _ in range(2)]


def tree_sees(parents, lens, C, gpu):
    """[B, N, C + N] from parents [B, N] (-2: absent) and cached counts."""
    B, N = len(parents), len(parents[0])
    sees = torch.zeros(B, N, C + N, dtype=torch.bool)
    for b in range(B):
        for i, p in enumerate(parents[b]):
            if p == -2:
                continue
            sees[b, i, :lens[b]] = True
            j = i
            while j >= 0:
                sees[b, i, C + j] = True
                j = parents[b][j]
    return sees.to(gpu)


def random_parents(N, seed, absent=False):
    g = torch.Generator().manual_seed(seed)
    par = []
    for i in range(N):
        p = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
        if p >= 0 and par[p] == -2:
            p = -1
        par.append(-2 if absent and i and float(torch.rand(1, generator=g)) < 0.2 else p)
    return par


@pytest.mark.parametrize("B,N,HK,C,lens", [
    (1, 1, 4, 0, None), (1, 1, 4, 1, None), (1, 8, 4, 500, None), (2, 9, 4, 33, [33, 0]), (3, 16, 4, 64, [64, 1, 31]),
    (1, 17, 4, 1000, None), (2, 32, 4, 96, [95, 32]), (2, 33, 1, 130, [130, 7]), (1, 64, 4, 2050, None),
    (2, 65, 2, 40, [0, 40]), (1, 2, 600, 70, None), (70, 2, 1, 90, [90 - i for i in range(70)]), (1, 255, 4, 300, None), (1, 512, 1, 70, None), (5, 3, 4, 4000, [4000, 17, 0, 1999, 3968])])
def test_tree_against_float64(gpu, B, N, HK, C, lens):
    q, k, v, kc, vc = heads(gpu, N, B, N, HK, C)
    par = [random_parents(N, 7 * b + N, absent=b % 2 == 1) for b in range(B)]
    o = tree_attention(q, k, v, tree_masks(par, gpu), cache=(kc, vc) if C else None,
                       cache_len=None if lens is None else torch.tensor(lens, dtype=torch.int32, device=gpu))
    check(o, q, torch.cat((kc, k), 1), torch.cat((vc, v), 1), tree_sees(par, lens or [C] * B, C, gpu))


@pytest.mark.parametrize("N", [3, 12, 30, 60])
@pytest.mark.parametrize("B,C", [(130, 40), (70, 400), (9, 2900), (600, 50)])
def test_tree_sequences_of_every_length_side_by_side(gpu, B, C, N):
    """Workgroups begin and end anywhere in the row of all sequences' keys: at a sequence's first tile, in its last, within
    the new keys."""
    q, k, v, kc, vc = heads(gpu, B + N, B, N, 1, C)
    g = torch.Generator().manual_seed(B * N)
    lens = torch.randint(-C // 4, C + 1, (B,), generator=g).clamp(0).tolist()
    par = [random_parents(N, b, absent=b % 3 == 0) for b in range(B)]
    o = tree_attention(q, k, v, tree_masks(par, gpu), (kc, vc), torch.tensor(lens, dtype=torch.int32, device=gpu))
    check(o, q, torch.cat((kc, k), 1), torch.cat((vc, v), 1), tree_sees(par, lens, C, gpu))


@pytest.mark.parametrize("N", [3, 12])
def test_tree_a_few_long_sequences_among_many(gpu, N):
    """More sequences than runs of key tiles: most lie within a run, the long ones are divided over many."""
    B, C = 140, 2700
    q, k, v, kc, vc = heads(gpu, N, B, N, 4, C)
    g = torch.Generator().manual_seed(N)
    lens = torch.randint(0, 70, (B,), generator=g).tolist()
    for b in (0, 63, 64, 100, 101, 139):
        lens[b] = C - b
    par = [random_parents(N, b) for b in range(B)]
    o = tree_attention(q, k, v, tree_masks(par, gpu), (kc, vc), torch.tensor(lens, dtype=torch.int32, device=gpu))
    check(o, q, torch.cat((kc, k), 1), torch.cat((vc, v), 1), tree_sees(par, lens, C, gpu))


def test_tree_shared_cache_one_tree_and_scale(gpu):
    q, k, v, kc, vc = heads(gpu, 3, 4, 20, 4, 777)
    par = random_parents(20, 5)
    sees = tree_sees([par] * 4, [777] * 4, 777, gpu)
    masks = tree_masks(par, gpu)
    outs = [tree_attention(q, k, v, masks, cache=c, scale=0.1) for c in (
        (kc[:1], vc[:1]), (kc[0], vc[0]), (kc[:1].expand(4, -1, -1, -1), vc[:1].expand(4, -1, -1, -1)))]
    check(outs[0], q, torch.cat((kc[:1].expand(4, -1, -1, -1), k), 1), torch.cat((vc[:1].expand(4, -1, -1, -1), v), 1),
          sees, 0.1)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_tree_chain_is_causal_attention(gpu):
    """A chain after a prefix is the continuation that causal_gqa_attention runs."""
    q, k, v, kc, vc = heads(gpu, 4, 2, 40, 4, 320)
    o = tree_attention(q, k, v, tree_masks(list(range(-1, 39)), gpu), cache=(kc[:1], vc[:1]))
    c = causal_gqa_attention(q, k, v, prefix=(kc[0], vc[0]))
    assert (o.float() - c.float()).abs().max() <= 2 ** -6      # two results of one bf16 step at most 4 each apart


def test_tree_strided_cache_and_rows(gpu):
    """A cache whose heads lie apart ([B, HK, C, 256] memory), rows of wider tables, a mask that is no ancestry."""
    q, k, v, kc, vc = heads(gpu, 6, 2, 30, 4, 200)
    wide = torch.randn(2, 200, 8, 512, device=gpu).to(BF)
    kc2 = wide[:, :, 1:5, 128:384]
    vc2 = vc.transpose(1, 2).contiguous().transpose(1, 2)
    g = torch.Generator().manual_seed(1)
    bits = torch.rand(30, 30, generator=g) < 0.3
    bits[4] = False
    words = (bits.long() << torch.arange(30)).sum(1, keepdim=True)
    dirty = (words | ~((1 << 30) - 1)).to(gpu)         # bits past the last node do not count
    dirty[4] = ~((1 << 30) - 1)
    sees = torch.cat((torch.ones(2, 30, 200, dtype=torch.bool), bits[None].expand(2, -1, -1)), 2)
    sees[:, ~bits.any(1)] = False
    for m in (words.to(gpu), dirty):
        check(tree_attention(q, k, v, m, cache=(kc2, vc2)), q, torch.cat((kc2, k), 1), torch.cat((vc2, v), 1),
              sees.to(gpu))


@pytest.mark.parametrize("N", [5, 20, 40, 100])
def test_tree_values_not_finite_reach_only_who_sees_them(gpu, N):
    """inf and NaN in nodes, in padding, and past the sequences' cached keys."""
    q, k, v, kc, vc = heads(gpu, 8, 2, N, 4, 100)
    par = [random_parents(N, 2), random_parents(N, 3, absent=True)]
    if -2 not in par[1]:
        par[1][N - 1] = -2
    v[0, N // 2, 1, 7], v[0, N - 1, 2, 200], v[0, N // 3, 3, 40] = math.inf, -math.inf, math.nan
    v[0, 0, 0, 3], v[0, N - 1, 0, 3] = math.inf, -math.inf
    for i, p in enumerate(par[1]):
        if p == -2:
            q[1, i], k[1, i], v[1, i] = math.nan, math.inf, math.nan
    lens = [100, 43]
    kc[1, 43:], vc[1, 43:] = math.nan, math.inf
    o = tree_attention(q, k, v, tree_masks(par, gpu), cache=(kc, vc),
                       cache_len=torch.tensor(lens, dtype=torch.int32, device=gpu))
    kk, vv = torch.cat((kc, k), 1), torch.cat((vc, v), 1)
    q = torch.where(torch.isfinite(q), q, 0.0)
    kk = torch.where(torch.isfinite(kk), kk, 0.0)
    check(o, q, kk, vv, tree_sees(par, lens, 100, gpu))


def window_sees(B, n, S, window, sinks, lens, gpu):
    pos = torch.tensor(lens)[:, None] - n + torch.arange(n)[None]
    pos, key = pos[:, :, None], torch.arange(S)[None, None]
    return ((key <= pos) & ((key > pos - window) | (key < sinks))).to(gpu)


@pytest.mark.parametrize("B,n,S,window,sinks,lens", [
    (1, 1, 1, 1, 0, None), (2, 1, 300, 64, 4, [300, 5]), (3, 5, 1000, 100, 0, [1000, 4, 0]), (2, 12, 4000, 777, 33, [4000, 3001]),
    (1, 33, 33, 1, 0, None), (1, 100, 100, 1, 1, None), (2, 70, 70, 32, 4, None), (1, 257, 257, 31, 64, None),
    (1, 300, 500, 33, 5, None), (2, 300, 200, 50, 3, [200, 90]), (1, 1111, 1111, 200, 5, None), (2, 40, 90, 1000, 0, None),
    (1, 64, 640, 128, 640, None), (1, 5, 0, 4, 4, None), (1, 8, 9000, 8192, 4, None), (1, 40, 300, 2 ** 31 + 5, 2 ** 31 + 5, None)])
def test_window_against_float64(gpu, B, n, S, window, sinks, lens):
    q, _, _, k, v = heads(gpu, S + n, B, n, 2, S)
    t = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=gpu)
    o = window_attention(q, k, v, window, sinks, kv_len=t)
    check(o, q, k, v, window_sees(B, n, S, window, sinks, lens or [S] * B, gpu))


@pytest.mark.parametrize("n,window", [(1, 500), (3, 40), (14, 300), (30, 64), (60, 129)])
def test_window_sequences_of_every_length_side_by_side(gpu, n, window):
    B, S = 67, 700
    q, _, _, k, v = heads(gpu, n, B, n, 1, S)
    lens = torch.randint(-S // 4, S + 1, (B,), generator=torch.Generator().manual_seed(n)).clamp(0).tolist()
    o = window_attention(q, k, v, window, 4, kv_len=torch.tensor(lens, dtype=torch.int32, device=gpu))
    check(o, q, k, v, window_sees(B, n, S, window, 4, lens, gpu))


def test_window_wider_than_the_keys_is_causal_attention(gpu):
    q, k, v = heads(gpu, 11, 2, 333, 4)
    o, c = window_attention(q, k, v, 333), causal_gqa_attention(q, k, v)
    assert (o.float() - c.float()).abs().max() <= 2 ** -6


@pytest.mark.parametrize("n", [3, 15, 90])
def test_window_values_not_finite_reach_only_who_sees_them(gpu, n):
    q, _, _, k, v = heads(gpu, 12, 2, n, 4, 200)
    lens = [200, 150]
    v[0, 190, 0, 5], v[0, 150, 1, 9], v[0, 2, 2, 100] = math.inf, math.nan, -math.inf
    k[0, 199] = math.nan
    k[1, 150:], v[1, 150:] = math.nan, math.inf
    o = window_attention(q, k, v, 40, 5, kv_len=torch.tensor(lens, dtype=torch.int32, device=gpu))
    sees = window_sees(2, n, 200, 40, 5, lens, gpu)
    assert torch.isnan(o[0, -1]).all()                 # its own key is NaN
    kk = torch.where(torch.isfinite(k), k, 0.0)
    check(o[:, :-1], q[:, :-1], kk, v, sees[:, :-1])


def test_scores_beyond_every_margin(gpu):
    """Scores of hundreds: the softmax's reference moves, weights underflow."""
    q, k, v, kc, vc = heads(gpu, 13, 1, 24, 4, 400)
    q, kc = (q.float() * 20).to(BF), (kc.float() * 2).to(BF)
    par = random_parents(24, 9)
    o = tree_attention(q, k, v, tree_masks(par, gpu), cache=(kc, vc)).double()
    r, a = ref(q, torch.cat((kc, k), 1), torch.cat((vc, v), 1), tree_sees([par], [400], 400, gpu))
    # scores are 40 times the unit ones: their fp32 error too, 40 x 2e-4, and twice that in the weights
    assert ((o - r).abs() <= 2 ** -8 * (a + r.abs()) + 0.016 * a).all()


def test_long_cache_offsets_past_32_bits(gpu):
    """A cache of 4.6 GB a tensor: the last rows lie past 2^32 bytes."""
    C = 600_000
    kc = torch.zeros(1, C, 15, 256, dtype=BF, device=gpu)[:, :, :4]
    vc = torch.zeros(1, C, 15, 256, dtype=BF, device=gpu)[:, :, :4]
    q, k, v, kt, vt = heads(gpu, 14, 1, 6, 4, 64)
    kc[:, C - 64:], vc[:, C - 64:] = (kt.float() * 8).to(BF), vt
    par = random_parents(6, 1)
    o = tree_attention(q, k, v, tree_masks(par, gpu), cache=(kc, vc))
    # in float64, the zero keys together: C - 64 scores of 0
    sees = tree_sees([par], [64], 64, gpu)
    kk, vv = torch.cat((kc[:, C - 64:], k), 1).double(), torch.cat((vt, v), 1).double()
    for h in range(16):
        z = q[0, :, h].double() @ kk[0, :, h // 4].t() / 16
        w = torch.where(sees[0], torch.exp(z), 0.0)
        t = w.sum(1, keepdim=True) + (C - 64)
        r, a = w @ vv[0, :, h // 4] / t, w @ vv[0, :, h // 4].abs() / t
        # the sum of 600000 equal weights in fp32, a lane's 16 of a tile at a time: at most 2^-24 a step
        assert ((o[0, :, h].double() - r).abs() <= 2 ** -8 * (a + r.abs()) + 2 ** -9 * a).all()
    w = window_attention(q[:, -1:], kc, vc, 64, 4)
    z = kk[0, :64].transpose(0, 1) @ q[0, -1].double().view(4, 4, 256).transpose(1, 2) / 16       # [HK, 64, 4]
    e = torch.exp(z)
    t = e.sum(1) + 4
    r = torch.einsum("gkj,kgd->gjd", e, vv[0, :64]) / t[..., None]
    a = torch.einsum("gkj,kgd->gjd", e, vv[0, :64].abs()) / t[..., None]
    assert ((w[0, 0].double().view(4, 4, 256) - r).abs() <= 2 ** -8 * (a + r.abs()) + 2 ** -9 * a).all()


def test_streams_and_graphs(gpu):
    """A side stream, and a captured graph replayed with the program's own calls between, on new inputs each time."""
    q, k, v, kc, vc = heads(gpu, 15, 2, 24, 4, 900)
    masks = tree_masks([random_parents(24, 1), random_parents(24, 2)], gpu)
    lens = torch.tensor([900, 400], dtype=torch.int32, device=gpu)
    call = lambda: (tree_attention(q, k, v, masks, cache=(kc, vc), cache_len=lens),  # noqa: E731
                    window_attention(q, kc, vc, 300, 4, kv_len=lens))
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        q.copy_(torch.randn(q.shape, device=gpu))
        lens.copy_(torch.tensor([900 - 13 * i, 17 * i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(call(), out))


def test_no_rows_no_sequences(gpu):
    q, k, v, kc, vc = heads(gpu, 16, 2, 4, 4, 10)
    masks = tree_masks([-1, 0, 1, 2], gpu)
    n0 = int8_kernels.STATS["launch"]
    assert tree_attention(q[:0], k[:0], v[:0], masks, cache=(kc[:0], vc[:0])).shape == (0, 4, 16, 256)
    assert tree_attention(q[:, :0], k[:, :0], v[:, :0], masks[:0, :0], cache=(kc, vc)).shape == (2, 0, 16, 256)
    assert window_attention(q[:, :0], kc, vc, 5).shape == (2, 0, 16, 256)
    assert int8_kernels.STATS["launch"] == n0 + 3


def test_refusals(gpu):
    q, k, v, kc, vc = heads(gpu, 17, 2, 4, 4, 10)
    m = tree_masks([-1, 0, 1, 2], gpu)
    lens = torch.tensor([3, 4], dtype=torch.int32, device=gpu)
    bad = [
        lambda: tree_attention(q.float(), k, v, m), lambda: tree_attention(q, k[:, :3], v[:, :3], m),
        lambda: tree_attention(q[:, :, :8], k, v, m), lambda: tree_attention(q, k, v, m.int()),
        lambda: tree_attention(q, k, v, m[:3]), lambda: tree_attention(q, k, v, m.cpu()),
        lambda: tree_attention(q, k, v, m, cache=(kc, vc[:, :9])), lambda: tree_attention(q, k, v, m, cache=(kc[:, :, :2], vc[:, :, :2])),
        lambda: tree_attention(q, k, v, m, cache=(kc, vc), cache_len=lens.long()),
        lambda: tree_attention(q, k, v, m, cache=(kc, vc), cache_len=lens[:1]), lambda: tree_attention(q, k, v, m, scale=-1.0),
        lambda: tree_attention(q, k, v, m, scale=math.nan), lambda: tree_attention(q, k.cpu(), v, m),
        lambda: tree_attention(q, k, v, m, cache=(kc[..., :128], vc[..., :128])),
        lambda: tree_attention(q.contiguous().view(-1)[1:1 + 2 * 4 * 8 * 256].view(2, 4, 8, 256), k[:, :, :2], v[:, :, :2], m),   # misaligned
        lambda: tree_attention(q, k[:, :1].expand(-1, 4, -1, -1), v, m),                                     # rows overlap
        lambda: window_attention(q, kc, vc, 0), lambda: window_attention(q, kc, vc, 4, -1),
        lambda: window_attention(q, kc, vc[:, :9], 4), lambda: window_attention(q, kc[:1], vc[:1], 4),
        lambda: window_attention(q, kc, vc, 4, kv_len=lens.cpu()), lambda: window_attention(q, kc.half(), vc.half(), 4)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    assert attention.MAX_TREE_NODES == 512
