"""kv_cache.paged_attention against attention in float64 over what the cache stands for (the bound is derived beside
kv_model.check)."""
import math

import pytest
import torch
from kv_model import BF, D, PAGE, Cache, attend, check, starts_of, stored

from mica_amd import int8_kernels
from mica_amd.kv_cache import paged_attention

pytestmark = pytest.mark.gpu


def sequences(gpu, seed, lens, HK, shared=0):
    """bf16 keys and values of each sequence; the first `shared` blocks are the same."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    rn = lambda n: torch.randn(n, HK, D, generator=g, device=gpu).to(BF)  # noqa: E731
    ks, vs = [rn(n) for n in lens], [rn(n) for n in lens]
    for x in ks[1:]:
        x[:shared * PAGE] = ks[0][:shared * PAGE]
    for x in vs[1:]:
        x[:shared * PAGE] = vs[0][:shared * PAGE]
    return ks, vs


def queries(gpu, seed, T, HK):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.randn(T, 6 * HK, D, generator=g, device=gpu).to(BF)[:, :4 * HK]


def check_all(o, q, ks, vs, counts, before=0, scale=1 / 16):
    lo = before
    for b, n in enumerate(counts):
        at = slice(lo, lo + n)
        check(o[at], *attend(q[at], stored(ks[b]), stored(vs[b]), ks[b].shape[0] - n, scale))
        lo += n
    return lo


CASES = [
    ([1], [1], 4, 0), ([31], [1], 4, 0), ([32], [1], 4, 0), ([33, 64, 1000], [1, 1, 1], 4, 0), ([5, 0, 40, 9], [1, 0, 2, 0], 2, 0),
    ([500], [500], 2, 0), ([70, 300, 33], [8, 3, 33], 4, 0), ([100, 90], [12, 16], 4, 0), ([2000, 17, 64], [30, 17, 1], 4, 0),
    ([1200, 700], [240, 65], 2, 0), ([4, 70], [9, 80], 2, 0), ([40] * 150, [1] * 150, 1, 0), ([3000] + [33] * 70, [2] * 71, 1, 0),
    ([700, 641, 690], [60, 1, 50], 4, 20), ([6000], [3], 4, 0), ([9000, 8999, 10], [1, 1, 1], 4, 0), ([5000, 300], [64, 64], 2, 0),
    ([4100], [300], 1, 0), ([2500] * 9, [20] * 9, 2, 70)]


@pytest.mark.parametrize("lens,counts,HK,shared", CASES)
@pytest.mark.parametrize("hint", [False, True])
def test_against_float64(gpu, lens, counts, HK, shared, hint):
    ks, vs = sequences(gpu, sum(lens), lens, HK, shared)
    B = len(lens)
    c = Cache(gpu, ks, vs, slots=torch.randperm(B, generator=torch.Generator().manual_seed(2)).tolist() if B > 1 else None, shared=shared)
    q = queries(gpu, 1, sum(counts), HK)
    o = paged_attention(q, c.kv(), starts_of(counts, gpu), c.lens, c.table, c.slots, longest=max(counts) if hint else None)
    check_all(o, q, ks, vs, counts)


@pytest.mark.parametrize("n", [1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65])
@pytest.mark.parametrize("keys", [90, 1500])
def test_rows_of_every_block_size(gpu, n, keys):
    """Sequences of all lengths up to `keys` side by side, n rows of each (more than some have)."""
    g = torch.Generator().manual_seed(n + keys)
    lens = torch.randint(0, keys + 1, (12,), generator=g).tolist() + [keys, 0, 32, 64]
    counts = torch.randint(0, n + 1, (12,), generator=g).tolist() + [n] * 4
    ks, vs = sequences(gpu, n, lens, 2)
    c = Cache(gpu, ks, vs)
    q = queries(gpu, 2, sum(counts), 2)
    for longest in (n, None):
        o = paged_attention(q, c.kv(), starts_of(counts, gpu), c.lens, c.table, longest=longest)
        check_all(o, q, ks, vs, counts)


def test_the_hint_may_be_wrong(gpu):
    lens, counts = [900, 100, 300], [130, 3, 20]
    ks, vs = sequences(gpu, 1, lens, 4)
    c = Cache(gpu, ks, vs)
    q = queries(gpu, 3, sum(counts), 4)
    for longest in (1, 5, 12, 40, 10 ** 10):
        check_all(paged_attention(q, c.kv(), starts_of(counts, gpu), c.lens, c.table, longest=longest), q, ks, vs, counts)


@pytest.mark.parametrize("n", [1, 40, 100])
def test_rows_of_no_sequence_and_strides(gpu, n):
    lens, counts, before, behind = [300, 99], [n, 7], 45, 70
    T = before + sum(counts) + behind
    ks, vs = sequences(gpu, 2, lens, 2)
    c = Cache(gpu, ks, vs)
    q = queries(gpu, 4, T, 2).clone()
    q[:before], q[T - behind:] = math.nan, math.inf
    starts = starts_of(counts, gpu, before)
    args = (c.kv(), starts, c.lens, c.table)
    o = paged_attention(q, *args, longest=n, scale=0.1)
    assert check_all(o, q, ks, vs, counts, before, 0.1) == T - behind
    assert not o[:before].any() and not o[T - behind:].any()
    wide = torch.full((8, T, 512), 7.0, dtype=BF, device=gpu)
    got = paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), *args, longest=n, scale=0.1,
                          out=wide[:, :, 128:384].transpose(0, 1))
    assert torch.equal(got[before:T - behind], o[before:T - behind])
    got[before:T - behind] = 7.0
    assert (wide == 7.0).all()


@pytest.mark.parametrize("n", [1, 3, 12, 30, 60, 100])
@pytest.mark.parametrize("keys", [140, 2010])
def test_values_not_finite_reach_only_who_sees_them(gpu, n, keys):
    """In the rest by row, in a finished block by block; sequence 1 is free of them.  keys % 32 rows are in the rest."""
    n = min(n, keys)
    ks, vs = sequences(gpu, 5, [keys, keys - 7, keys], 2)
    left = keys % PAGE
    vs[0][keys - 1, 0, 5], vs[0][keys - left // 2, 1, 9], vs[0][keys - left, 0, 100] = math.inf, math.nan, -math.inf
    ks[0][keys - 2, 1, 3] = math.nan
    block = (keys - n) // PAGE                         # the block of the first row: later rows see it, and all of this block
    vs[2][block * PAGE + 31 if block * PAGE + 31 < keys - left else 3, 0, 0] = math.inf
    ks[2][70, 1, 0] = -math.inf
    c = Cache(gpu, ks, vs)
    q = queries(gpu, 5, 3 * n, 2)
    for longest in (n, None):
        o = paged_attention(q, c.kv(), starts_of([n] * 3, gpu), c.lens, c.table, longest=longest)
        check_all(o, q, ks, vs, [n] * 3)
        assert torch.isfinite(o[n:2 * n]).all()


def test_what_is_missing_is_nan(gpu):
    """A block without a page, a rest without a slot; a sequence beside them is right."""
    lens = [100, 100, 100]
    ks, vs = sequences(gpu, 6, lens, 2)
    for n in (1, 20, 70):
        c = Cache(gpu, ks, vs)
        c.table[0, 1] = -1
        slots = torch.tensor([0, 1, 9], dtype=torch.int32, device=gpu)
        q = queries(gpu, 6, 3 * n, 2)
        o = paged_attention(q, c.kv(), starts_of([n] * 3, gpu), c.lens, c.table, slots)
        pos = 100 - n + torch.arange(n, device=gpu)
        assert torch.equal(torch.isnan(o[:n]).all(-1).all(-1), pos >= 32) and torch.equal(torch.isnan(o[2 * n:]).any(-1).any(-1), pos >= 96)
        check(o[n:2 * n], *attend(q[n:2 * n], stored(ks[1]), stored(vs[1]), 100 - n))
        # lengths past the table and below 0 are cut: nothing outside is touched, and the right sequence stays so
        wild = torch.tensor([2 ** 31 - 1, 100, -9], dtype=torch.int32, device=gpu)
        o2 = paged_attention(q, c.kv(), starts_of([n] * 3, gpu), wild, c.table, longest=n)
        check(o2[n:2 * n], *attend(q[n:2 * n], stored(ks[1]), stored(vs[1]), 100 - n))
        assert not o2[2 * n:].any()


def test_scores_beyond_every_margin(gpu):
    """Scores of hundreds: the softmax's reference moves, weights underflow."""
    lens, counts = [1500, 300], [24, 1]
    ks, vs = sequences(gpu, 7, lens, 4)
    c = Cache(gpu, ks, vs)
    q = (queries(gpu, 7, 25, 4).float() * 30).to(BF)
    o = paged_attention(q, c.kv(), starts_of(counts, gpu), c.lens, c.table).double()
    for at, b in ((slice(0, 24), 0), (slice(24, 25), 1)):
        r, a = attend(q[at], stored(ks[b]), stored(vs[b]), lens[b] - counts[b])
        # scores are 30 times the unit ones: their fp32 error too, 30 x 2e-4, and twice that in the weights; weights below 2^-126
        # of the largest are not fp32's: at most 1500 of them x |v| of 6, below 2^-112 (where the largest meets an int8 of 0)
        assert ((o[at] - r).abs() <= 2 ** -8 * (a + r.abs()) + 0.012 * a + 2.0 ** -112).all()


def test_blocks_of_very_different_scales(gpu):
    ks, vs = sequences(gpu, 8, [640], 2)
    for j in range(20):
        vs[0][j * PAGE:(j + 1) * PAGE] *= 2.0 ** (3 * j - 40)
        ks[0][j * PAGE:(j + 1) * PAGE] *= 2.0 ** (-(j % 5))
    ks[0][64:96], vs[0][96:128] = 0.0, 0.0
    c = Cache(gpu, ks, vs)
    for n in (1, 20, 300):
        q = queries(gpu, 8, n, 2)
        check(paged_attention(q, c.kv(), starts_of([n], gpu), c.lens, c.table), *attend(q, stored(ks[0]), stored(vs[0]), 640 - n))


def test_offsets_past_32_bits(gpu):
    """A pool of 4.6 GB whose last pages are in use."""
    ks, vs = sequences(gpu, 9, [70], 4)
    c = Cache(gpu, ks, vs)
    P = 70_000
    data, scales = torch.zeros(P, 2, 4, 8, 32, 32, dtype=torch.int8, device=gpu), torch.zeros(P, 2, 4, device=gpu)
    for j in range(2):
        data[P - 1 - j], scales[P - 1 - j] = c.data[c.table[0, j]], c.scales[c.table[0, j]]
    table = torch.tensor([[P - 1, P - 2]], dtype=torch.int32, device=gpu)
    for n in (1, 70):
        q = queries(gpu, 9, n, 4)
        o = paged_attention(q, c.kv()._replace(data=data, scales=scales), starts_of([n], gpu), c.lens, table)
        check(o, *attend(q, stored(ks[0]), stored(vs[0]), 70 - n))


@pytest.mark.parametrize("n", [1, 30, 90])
def test_streams_and_graphs(gpu, n):
    """A captured call replayed with other queries and lengths, the program's own calls between."""
    lens = [1500, 700, 900]
    ks, vs = sequences(gpu, 10, lens, 4)
    c = Cache(gpu, ks, vs)
    q, starts = queries(gpu, 10, 3 * n, 4).clone(), starts_of([n] * 3, gpu)
    call = lambda: paged_attention(q, c.kv(), starts, c.lens, c.table, longest=n)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=gpu))
        now = [x - PAGE * ((211 * i) % x // PAGE) for x in lens]          # whole blocks less: the rest is another's then
        c.lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(call(), out)
        for b, m in enumerate(now):
            k, v = (torch.cat((stored(x[b])[:m // PAGE * PAGE], x[b][lens[b] // PAGE * PAGE:].float())) for x in (ks, vs))
            check(out[b * n:(b + 1) * n], *attend(q[b * n:(b + 1) * n], k, v, m - n))


def test_the_same_bits_at_every_call(gpu):
    for lens, counts in (([5000, 70], [1, 1]), ([3000, 2000], [20, 33]), ([900] * 5, [100] * 5)):
        ks, vs = sequences(gpu, 11, lens, 4)
        c = Cache(gpu, ks, vs)
        q, starts = queries(gpu, 11, sum(counts), 4), starts_of(counts, gpu)
        first = paged_attention(q, c.kv(), starts, c.lens, c.table, longest=max(counts))
        for _ in range(4):
            assert torch.equal(paged_attention(q, c.kv(), starts, c.lens, c.table, longest=max(counts)), first)


def test_no_rows(gpu):
    ks, vs = sequences(gpu, 12, [40, 3], 2)
    c = Cache(gpu, ks, vs)
    q = queries(gpu, 12, 6, 2)
    n0 = int8_kernels.STATS["launch"]
    assert paged_attention(q[:0], c.kv(), starts_of([0, 0], gpu), c.lens, c.table).shape == (0, 8, D)
    assert not paged_attention(q, c.kv(), starts_of([0, 0], gpu), c.lens, c.table).any()
    assert not paged_attention(q, c.kv(), starts_of([], gpu), c.lens[:0], c.table[:0]).any()
    assert int8_kernels.STATS["launch"] == n0 + 3


def test_refusals(gpu):
    ks, vs = sequences(gpu, 13, [40, 3], 2)
    c = Cache(gpu, ks, vs)
    q, s = queries(gpu, 13, 6, 2), starts_of([3, 3], gpu)
    f = lambda qq=q, st=s, ln=c.lens, tb=c.table, kv=c.kv(), **kw: paged_attention(qq, kv, st, ln, tb, **kw)  # noqa: E731
    bad = [lambda: f(qq=q.float()), lambda: f(qq=q[:, :4]), lambda: f(qq=q[..., :128]), lambda: f(qq=q[None]), lambda: f(st=s.long()),
           lambda: f(st=s.cpu()), lambda: f(ln=c.lens[:1]), lambda: f(ln=None), lambda: f(tb=c.table.long()), lambda: f(tb=c.table[:1]),
           lambda: f(kv=c.kv()._replace(scales=c.scales.half())), lambda: f(kv=c.kv()._replace(data=c.data[:, :1])),
           lambda: f(slots=c.lens.float()), lambda: f(longest=-1), lambda: f(scale=-1.0), lambda: f(scale=math.nan),
           lambda: f(out=torch.empty(5, 8, D, dtype=BF, device=gpu)), lambda: f(out=torch.empty(6, 8, D, device=gpu)),
           lambda: f(qq=q.cpu()), lambda: f(qq=q.contiguous().view(-1)[1:1 + 5 * 2048].view(5, 8, D))]
    for i, g in enumerate(bad):
        with pytest.raises(ValueError):
            g()
            pytest.fail(f"call {i} was taken")
