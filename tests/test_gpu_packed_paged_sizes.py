"""The packed and paged operators at the sizes where their work is divided another way: more sequences than a wave has lanes,
more than there are runs, blocks in chunks, and rows of no sequence alone."""
import pytest
import torch
from kv_model import Cache, attend, check, starts_of, stored

from mica_amd import _lib
from mica_amd.attention import packed_attention
from mica_amd.kv_cache import PagedKV, append_kv, paged_attention, read_kv

pytestmark = pytest.mark.gpu
BF, D = torch.bfloat16, 256


def heads(gpu, seed, T, HK):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.randn(T, 6 * HK, D, generator=g, device=gpu).to(BF).split((4 * HK, HK, HK), dim=1)


@pytest.mark.parametrize("counts,HK,divided", [
    ([1000], 4, True), ([769], 1, True), ([768, 3, 2], 2, True), ([1], 4, False), ([730], 4, False), ([5] * 65, 1, False), ([40, 1, 0] * 60, 1, False),
    ([4000, 10, 900], 1, True), ([7, 0] * 700, 1, False)])
def test_packed(gpu, counts, HK, divided):
    T = sum(counts)
    q, k, v = heads(gpu, len(counts), T, HK)
    nbytes = _lib.load().mica_attention_packed_workspace_bytes(len(counts), T, HK, max(counts))
    assert (nbytes > 0) == divided
    o = packed_attention(q, k, v, starts_of(counts, gpu), longest=max(counts))
    at = 0
    for n in counts:
        if n:
            check(o[at:at + n], *attend(q[at:at + n], k[at:at + n], v[at:at + n], 0))
        at += n


def test_packed_chunks_whatever_the_hint(gpu):
    """Chunks of a length that the hint gave, for blocks that are longer or shorter than it says; rows of none between them."""
    q, k, v = heads(gpu, 3, 1400, 2)
    for counts, before in (([1400], 0), ([900, 100], 37), ([33, 1200], 0), ([5], 100)):
        for hint in (1, 768, 900, 1400, 5000):
            o = packed_attention(q, k, v, starts_of(counts, gpu, before), longest=hint)
            at = before
            assert not o[:before].any()
            for n in counts:
                check(o[at:at + n], *attend(q[at:at + n], k[at:at + n], v[at:at + n], 0))
                at += n
            assert not o[at:].any()


@pytest.mark.parametrize("lens,counts,HK", [
    ([70] * 130, [1] * 130, 1), ([40 + 3 * i for i in range(200)], [1, 0, 2, 1] * 50, 2), ([90] * 300, [9] * 300, 1), ([33] * 1100, [1] * 1100, 1),
    ([500] * 70, [40] * 70, 1), ([64, 3000] * 40, [64, 70] * 40, 1), ([65] * 300, [65] * 300, 1), ([5000], [3], 8), ([31, 32, 33] * 30, [31, 32, 33] * 30, 2)])
def test_paged(gpu, lens, counts, HK):
    g = torch.Generator(device=gpu).manual_seed(len(lens))
    ks, vs = [[torch.randn(n, HK, D, generator=g, device=gpu).to(BF) for n in lens] for _ in range(2)]
    c = Cache(gpu, ks, vs)
    q = heads(gpu, 1, sum(counts), HK)[0]
    assert _lib.load().mica_attention_paged_workspace_bytes(len(lens), sum(counts), HK, c.table.shape[1], max(counts)) > 0
    o = paged_attention(q, c.kv(), starts_of(counts, gpu), c.lens, c.table, longest=max(counts))
    at = 0
    for b, n in enumerate(counts):
        if n:
            check(o[at:at + n], *attend(q[at:at + n], stored(ks[b]), stored(vs[b]), lens[b] - n))
        at += n
    kb, vb = read_kv(c.kv(), sum(counts), starts_of(counts, gpu), c.lens, c.table, longest=max(counts))
    at = 0
    for b, n in enumerate(counts):
        assert torch.equal(kb[at:at + n], stored(ks[b])[lens[b] - n:].to(BF)) and torch.equal(vb[at:at + n], stored(vs[b])[lens[b] - n:].to(BF))
        at += n


def test_many_sequences_appended(gpu):
    """300 sequences, some without rows, to lengths before and behind the ends of blocks; read back as the tokens say."""
    HK, lens, add = 1, [(7 * i) % 70 for i in range(300)], [(i * i) % 37 for i in range(300)]
    g = torch.Generator(device=gpu).manual_seed(8)
    ks, vs = [[torch.randn(a + b, HK, D, generator=g, device=gpu).to(BF) for a, b in zip(lens, add)] for _ in range(2)]
    cache = PagedKV.empty(1300, 300, HK, gpu)
    table = torch.randperm(1300, generator=torch.Generator().manual_seed(3))[:1200].to(torch.int32).view(300, 4).to(gpu)
    n0 = torch.zeros(300, dtype=torch.int32, device=gpu)
    n1, n2 = n0 + torch.tensor(lens, dtype=torch.int32, device=gpu), torch.tensor([a + b for a, b in zip(lens, add)], dtype=torch.int32, device=gpu)
    cat = lambda xs: torch.cat(list(xs))  # noqa: E731
    append_kv(cache, cat(k[:n] for k, n in zip(ks, lens)), cat(v[:n] for v, n in zip(vs, lens)), starts_of(lens, gpu), n0, table)
    append_kv(cache, cat(k[n:] for k, n in zip(ks, lens)), cat(v[n:] for v, n in zip(vs, lens)), starts_of(add, gpu), n1, table)
    n = n2.tolist()
    for hint in (None, max(n)):
        kb, vb = read_kv(cache, sum(n), starts_of(n, gpu), n2, table, longest=hint)
        for b, (x, y) in enumerate(zip(kb.split(n), vb.split(n))):
            assert torch.equal(x, stored(ks[b]).to(BF)) and torch.equal(y, stored(vs[b]).to(BF))


def test_rows_of_no_sequence_alone(gpu):
    """No sequence at all, and none with rows, for many rows: zeros, or what was there."""
    q, k, v = heads(gpu, 5, 1500, 2)
    c = Cache(gpu, [k[:200], k[:3]], [v[:200], v[:3]])
    for B in (0, 2):
        s, n, t = starts_of([0] * B, gpu), c.lens[:B], c.table[:B]
        for hint in (None, 1, 20, 1500):
            assert not packed_attention(q, k, v, s, longest=hint).any()
            assert not paged_attention(q, c.kv(), s, n, t, longest=hint).any()
            out = torch.full((1500, 8, D), 7.0, dtype=BF, device=gpu)
            packed_attention(q, k, v, s, longest=hint, out=out)
            paged_attention(q, c.kv(), s, n, t, longest=hint, out=out)
            assert (out == 7).all()
        assert not any(x.any() for x in read_kv(c.kv(), 1500, s, n, t))


def test_starts_and_lengths_that_are_none(gpu):
    """What no caller means: starts that fall, lie outside or repeat, lengths and pages outside the cache.  Nothing outside the
    output is written, and the call ends."""
    q, k, v = heads(gpu, 6, 600, 2)
    c = Cache(gpu, [k[:200]] * 3, [v[:200]] * 3)
    kept = [x.clone() for x in c.kv()]
    big = 2 ** 31 - 1
    for s in ([0, 600, 0, 600], [600, 300, 0, 0], [-5, 700, big, -big], [big, big, big, big], [0, 1, 0, 1], [-big, -7, 3, 900]):
        for lens in (c.lens, torch.tensor([-3, big, 10 ** 6], dtype=torch.int32, device=gpu)):
            st = torch.tensor(s, dtype=torch.int32, device=gpu)
            for hint in (None, 1, 9, 600):
                mem = torch.full((800, 8, D), 5.0, dtype=BF, device=gpu)
                paged_attention(q, c.kv(), st, lens, c.table, longest=hint, out=mem[100:700])
                assert (mem[:100] == 5).all() and (mem[700:] == 5).all()
                read_kv(c.kv(), 600, st, lens, c.table, longest=hint)
    torch.cuda.synchronize()
    assert all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())) for a, b in zip(kept, c.kv()))


@pytest.mark.parametrize("n", [1, 3, 12, 30, 60, 300, 1000])
def test_results_in_the_queries_place(gpu, n):
    """out= q itself, strided as the fused rows leave it: the same bits as beside it, k and v left alone."""
    counts = [n, max(1, n // 3)]
    q, k, v = heads(gpu, n, sum(counts), 2)
    g = torch.Generator(device=gpu).manual_seed(n)
    c = Cache(gpu, *[[torch.randn(n + 150, 2, D, generator=g, device=gpu).to(BF) for _ in counts] for _ in range(2)])
    s, kept = starts_of(counts, gpu), (k.clone(), v.clone())
    want = packed_attention(q, k, v, s, longest=n), paged_attention(q, c.kv(), s, c.lens, c.table, longest=n)
    for f, w in ((lambda x: packed_attention(x, k, v, s, longest=n, out=x), want[0]), (lambda x: paged_attention(x, c.kv(), s, c.lens, c.table, longest=n, out=x), want[1])):
        was = q.clone()
        assert f(q) is q and torch.equal(q, w)
        q.copy_(was)
    assert torch.equal(k, kept[0]) and torch.equal(v, kept[1])
