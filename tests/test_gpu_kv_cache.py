"""kv_cache.append_kv and read_kv against the definition in kv_model, bit for bit; norm and rotation against float64."""
import math

import pytest
import torch
from kv_model import BF, D, PAGE, Cache, key_page, quantized, starts_of, stored, value_page

from mica_amd import int8_kernels
from mica_amd.kv_cache import PagedKV, append_kv, read_kv

pytestmark = pytest.mark.gpu


def new_rows(gpu, seed, T, HK, scale=1.0):
    """k, v views of fused rows."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = (torch.randn(T, 6 * HK, D, generator=g, device=gpu) * scale).to(BF)
    return x[:, 4 * HK:5 * HK], x[:, 5 * HK:]


def fresh(gpu, B, HK, blocks, slots=None):
    """A cache of garbage, a table of pages in a random order."""
    cache = PagedKV.empty(B * blocks + 3, slots or B, HK, gpu)
    cache.data.fill_(-77)
    cache.scales.fill_(-3.0)
    cache.recent.fill_(-5.0)
    order = torch.randperm(B * blocks + 3, generator=torch.Generator().manual_seed(B))[:B * blocks]
    return cache, order.view(B, blocks).to(torch.int32).to(gpu)


def expect(cache, table, keys, values, slots=None):
    """The cache holds these sequences' bf16 rows, and everything else is as fresh() left it."""
    data, scales, recent = (t.clone() for t in (cache.data, cache.scales, cache.recent))
    for b, (k, v) in enumerate(zip(keys, values)):
        full, left = divmod(k.shape[0], PAGE)
        slot = b if slots is None else slots[b]
        for side, (x, lay) in enumerate(((k, key_page), (v, value_page))):
            for j in range(full):
                q, s = quantized(x[j * PAGE:(j + 1) * PAGE].transpose(0, 1))
                page = int(table[b, j])
                assert torch.equal(data[page, side], lay(q)) and torch.equal(scales[page, side].nan_to_num(-1), s.nan_to_num(-1))
            assert torch.equal(recent[slot, side, :, :left].view(torch.int16), x[full * PAGE:].transpose(0, 1).view(torch.int16))
        used = table[b, :full].long()
        data[used], scales[used] = -77, -3.0
    assert (data == -77).all() and (scales == -3.0).all()


@pytest.mark.parametrize("counts,HK", [
    ([1], 4), ([31], 1), ([32], 4), ([33, 0, 64, 5], 2), ([0, 0, 7], 4), ([1000, 1, 95, 96, 97], 4), ([3] * 130, 1), ([700] + [2] * 70, 2)])
def test_prompts_into_an_empty_cache(gpu, counts, HK):
    T, B = sum(counts), len(counts)
    k, v = new_rows(gpu, T, T, HK)
    cache, table = fresh(gpu, B, HK, max(counts) // PAGE + 1)
    zero = torch.zeros(B, dtype=torch.int32, device=gpu)
    got = append_kv(cache, k, v, starts_of(counts, gpu), zero, table)
    assert got is cache
    expect(cache, table, k.split(counts), v.split(counts))


@pytest.mark.parametrize("treated", [False, True])
def test_the_same_bits_whichever_calls_brought_them(gpu, treated):
    """One at a time, in odd pieces, all at once; with slots, with the search for units and without."""
    B, HK, total = 3, 2, [150, 97, 64]
    k, v = new_rows(gpu, 1, sum(total), HK)
    ks, vs = k.split(total), v.split(total)
    ang = torch.arange(200, device=gpu)[:, None] * 10000.0 ** (-torch.arange(32, device=gpu) / 32)
    more = dict(rope=(ang.cos().to(BF), ang.sin().to(BF)), norm=(torch.randn(D, device=gpu).to(BF), 1.0, 1e-6)) if treated else {}
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device=gpu)
    caches = []
    for step in (1000, 1, 37, 64, 5):
        cache, table = fresh(gpu, B, HK, 5, slots=6)
        held = [0] * B
        while held != total:
            counts = [min(step + b, n - h) for b, (n, h) in enumerate(zip(total, held))]
            kk = torch.cat([x[h:h + c] for x, h, c in zip(ks, held, counts)])
            vv = torch.cat([x[h:h + c] for x, h, c in zip(vs, held, counts)])
            append_kv(cache, kk, vv, starts_of(counts, gpu), torch.tensor(held, dtype=torch.int32, device=gpu), table, slots,
                      longest=(None, max(counts), 1)[step % 3], **more)
            held = [h + c for h, c in zip(held, counts)]
        caches.append(cache)
        if not treated:
            expect(cache, table, ks, vs, [4, 0, 2])
    lefts = [n % PAGE for n in total]
    for c in caches[1:]:
        assert torch.equal(c.data, caches[0].data) and torch.equal(c.scales, caches[0].scales)
        for s, left in zip((4, 0, 2), lefts):
            assert torch.equal(c.recent[s, :, :, :left], caches[0].recent[s, :, :, :left])


@pytest.mark.parametrize("rot", [0, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("wide", [False, True])
def test_norm_and_rotation(gpu, rot, wide):
    """Against float64.  The norm's factor is a sum of 256 squares in fp32 (256 x 2^-24 relative at most, half of it after the
    root), a quotient and a root; the products and the rotation add a few 2^-24 of the pair's magnitude: 2^-15 (|x| + |y|) holds
    all of it.  Then bf16's half step, 2^-8 of the value."""
    HK, n = 2, 31
    k, v = new_rows(gpu, rot, n, HK, 3.0)
    w = torch.randn(D, device=gpu).to(BF)
    tab = torch.float32 if wide else BF
    pos = torch.randint(0, 5000, (n,), device=gpu, dtype=torch.int32)
    pos[3], pos[7] = -1, 4000                                  # outside the tables: not rotated
    half = max(rot // 2, 1)
    ang = torch.arange(4000, device=gpu, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(half, device=gpu).double() / half)
    cos, sin = ang.cos().to(tab), ang.sin().to(tab)
    for norm in (None, (w, 1.0, 1e-6), (w, 0.0, 0.5)):
        for given in ((True, False) if rot else (False,)):
            cache, table = fresh(gpu, 1, HK, 1)
            at = 1000
            append_kv(PagedKV(*cache), k, v, starts_of([n], gpu), torch.tensor([at // 32 * 32], dtype=torch.int32, device=gpu),
                      torch.zeros(1, 64, dtype=torch.int32, device=gpu), norm=norm,
                      rope=((cos, sin, pos) if given else (cos, sin)) if rot else None)
            x = k.double()
            if norm is not None:
                x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + norm[2]) * (norm[1] + w.double())
            size = x.abs().clone()
            if rot:
                p = pos.long() if given else torch.arange(n, device=gpu) + at // 32 * 32
                inside = (p >= 0) & (p < 4000)
                c, s = (torch.where(inside[:, None], t[p.clamp(0, 3999)].double(), e)[:, None] for t, e in ((cos, 1.0), (sin, 0.0)))
                a, b = x[..., :half].clone(), x[..., half:rot].clone()
                x[..., :half], x[..., half:rot] = a * c - b * s, b * c + a * s
                size[..., :half] = size[..., half:rot] = a.abs() + b.abs()
            got = cache.recent[0, 0, :, :n].transpose(0, 1).double()
            assert ((got - x).abs() <= 2 ** -8 * x.abs() + 2 ** -15 * size).all()
            assert torch.equal(cache.recent[0, 1, :, :n].transpose(0, 1), v)      # values are not treated


def test_finished_blocks_hold_the_treated_bf16_rows(gpu):
    """The int8 of a page are those of the rows that waited."""
    HK, n = 4, 96
    k, v = new_rows(gpu, 5, n, HK)
    ang = torch.arange(200, device=gpu)[:, None] * 1e4 ** (-torch.arange(32, device=gpu) / 32)
    more = dict(rope=(ang.cos().to(BF), ang.sin().to(BF)), norm=(torch.randn(D, device=gpu).to(BF), 1.0, 1e-6))
    table = torch.arange(4, dtype=torch.int32, device=gpu)[None]
    got = []
    for lo in range(0, n, PAGE):        # each block's first 31 rows, and its last alone in a slot of its own
        one, _ = fresh(gpu, 1, HK, 4)
        append_kv(one, k[lo:lo + 31], v[lo:lo + 31], starts_of([31], gpu), torch.tensor([lo], dtype=torch.int32, device=gpu), table, **more)
        pos = torch.tensor([lo + 31], dtype=torch.int32, device=gpu)
        two, _ = fresh(gpu, 1, HK, 4)
        append_kv(two, k[lo + 31:lo + 32], v[lo + 31:lo + 32], starts_of([1], gpu), torch.zeros(1, dtype=torch.int32, device=gpu),
                  table, rope=(*more["rope"], pos), norm=more["norm"])
        got.append(torch.cat((one.recent[0, 0, :, :31], two.recent[0, 0, :, :1]), 1).transpose(0, 1))
    cache, _ = fresh(gpu, 1, HK, 4)
    append_kv(cache, k, v, starts_of([n], gpu), torch.zeros(1, dtype=torch.int32, device=gpu), table, **more)
    q, s = quantized(torch.cat(got).view(3, PAGE, HK, D).transpose(1, 2))
    for j in range(3):
        assert torch.equal(cache.data[j, 0], key_page(q[j])) and torch.equal(cache.scales[j, 0], s[j])


def test_extreme_values(gpu):
    """Zeros, subnormals, the largest, one value alone; NaN and infinity make the scale of their block, head and side NaN."""
    HK = 2
    k, v = (x.clone() for x in new_rows(gpu, 6, 256, HK))
    k[:32], v[:32] = 0.0, 1e-39
    k[32:64], v[32:64] = 3e38, -1e-9
    k[64:96] = 0.0
    k[77, 1, 100] = -2.5
    v[100, 0, 3], v[130, 1, 255], k[170, 0, 0], k[171, 0, 1] = math.inf, math.nan, -math.inf, math.nan
    v[200, 0] = (torch.randn(D, device=gpu) * 2 ** torch.randint(-60, 60, (D,), device=gpu).float()).to(BF)
    cache, table = fresh(gpu, 1, HK, 9)
    append_kv(cache, k, v, starts_of([256], gpu), torch.zeros(1, dtype=torch.int32, device=gpu), table)
    expect(cache, table, [k], [v])
    bad = torch.isnan(cache.scales[table[0, :8].long()])
    assert bad.nonzero().tolist() == [[3, 1, 0], [4, 1, 1], [5, 0, 0]]


def test_what_has_no_place_is_not_stored(gpu):
    """Pages outside the pool, blocks past the table, slots outside: nothing else is written."""
    HK, counts = 2, [100, 100, 70, 40]
    k, v = new_rows(gpu, 7, sum(counts), HK)
    cache, table = fresh(gpu, 4, HK, 3)
    table = table.clone()
    table[0, 1], table[0, 2], table[1, 0] = -1, cache.data.shape[0], 2 ** 31 - 1
    slots = torch.tensor([2, 0, 4, -1], dtype=torch.int32, device=gpu)
    narrow = table[:, :2]                                         # rows 3 apart: block 2 has no place
    append_kv(cache, k, v, starts_of(counts, gpu), torch.zeros(4, dtype=torch.int32, device=gpu), narrow, slots)
    data, recent = cache.data.clone(), cache.recent.clone()
    ks, vs = k.split(counts), v.split(counts)
    for page, b, j in ((int(table[0, 0]), 0, 0), (int(table[1, 1]), 1, 1)):
        for side, (x, lay) in enumerate(((ks[b], key_page), (vs[b], value_page))):
            assert torch.equal(data[page, side], lay(quantized(x[j * PAGE:(j + 1) * PAGE].transpose(0, 1))[0]))
        data[page] = -77
    assert (data == -77).all()
    for b, slot in ((0, 2), (1, 0)):
        assert torch.equal(recent[slot, 0, :, :4], ks[b][96:].transpose(0, 1))
        recent[slot, :, :, :4] = -5.0
    assert (recent == -5.0).all()


@pytest.mark.parametrize("lens,counts,HK", [
    ([1], [1], 4), ([320], [320], 4), ([33, 64, 100, 31], [33, 1, 77, 0], 2), ([5, 0, 64], [9, 3, 70], 1), ([40] * 100, [9] * 100, 1),
    ([2000, 7], [1990, 7], 4)])
def test_read(gpu, lens, counts, HK):
    """Bit for bit scale x int8 rounded once; zeros before a sequence's beginning and in rows of no sequence."""
    B = len(lens)
    keys, values = zip(*(new_rows(gpu, 10 * b + n, n, HK) for b, n in enumerate(lens)))
    order = torch.randperm(B, generator=torch.Generator().manual_seed(1)).tolist()
    c = Cache(gpu, keys, values, slots=order if B > 2 else None)
    T = sum(counts)
    for before, behind in ((0, 0), (40, 33)):
        k, v = read_kv(c.kv(), before + T + behind, starts_of(counts, gpu, before), c.lens, c.table, c.slots)
        assert k.shape == (before + T + behind, HK, D) and v.shape == k.shape
        lo = before
        for b, n in enumerate(counts):
            for got, x in ((k, keys[b]), (v, values[b])):
                want = torch.cat((torch.zeros(max(0, n - lens[b]), HK, D, device=gpu), stored(x)[max(0, lens[b] - n):])).to(BF)
                assert torch.equal(got[lo:lo + n], want)
            lo += n
        for x in (k, v):
            assert not x[:before].any() and not x[lo:].any()


def test_read_what_is_missing(gpu):
    """A block without a page, a rest without a slot, lengths past the table: NaN, and nothing is touched."""
    k0, v0 = new_rows(gpu, 3, 70, 2)
    c = Cache(gpu, [k0, k0], [v0, v0], extra=0)
    c.table[0, 1] = 10 ** 6
    slots = torch.tensor([0, 77], dtype=torch.int32, device=gpu)
    k, v = read_kv(c.kv(), 140, starts_of([70, 70], gpu), c.lens, c.table, slots)
    for x, y in ((k, k0), (v, v0)):
        want = stored(y).to(BF)
        assert torch.equal(x[:32], want[:32]) and torch.isnan(x[32:64]).all() and torch.equal(x[64:70], want[64:])
        assert torch.equal(x[70:134], want[:64]) and torch.isnan(x[134:]).all()
    k, _ = read_kv(c.kv(), 8, starts_of([4, 4], gpu), torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device=gpu), c.table)
    assert torch.equal(k[4:], torch.zeros_like(k[4:]))           # (no tokens; the first is cut to 2 pages and a rest)


def test_offsets_past_32_bits(gpu):
    """A pool of 4.6 GB: the pages in use lie at its end."""
    P = 70_000
    cache = PagedKV.empty(P, 1, 4, gpu)
    k, v = new_rows(gpu, 4, 70, 4)
    table = torch.tensor([[P - 1, P - 2]], dtype=torch.int32, device=gpu)
    append_kv(cache, k, v, starts_of([70], gpu), torch.zeros(1, dtype=torch.int32, device=gpu), table)
    for j in range(2):
        q, s = quantized(k[j * PAGE:(j + 1) * PAGE].transpose(0, 1))
        assert torch.equal(cache.data[P - 1 - j, 0], key_page(q)) and torch.equal(cache.scales[P - 1 - j, 0], s)
    kk, vv = read_kv(cache, 70, starts_of([70], gpu), torch.tensor([70], dtype=torch.int32, device=gpu), table)
    assert torch.equal(kk, stored(k).to(BF)) and torch.equal(vv, stored(v).to(BF))


def test_streams_and_graphs(gpu):
    """A captured step replayed with other rows and lengths, the program's own calls between."""
    B, HK = 5, 4
    k, v = new_rows(gpu, 8, B, HK)
    k, v = k.clone(), v.clone()
    cache, table = fresh(gpu, B, HK, 3)
    twin = PagedKV(*(t.clone() for t in cache))
    lens = torch.zeros(B, dtype=torch.int32, device=gpu)
    starts = starts_of([1] * B, gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        append_kv(cache, k, v, starts, lens, table, longest=1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append_kv(cache, k, v, starts, lens, table, longest=1)
        lens += 1
        got = read_kv(cache, B, starts, lens, table)
    rows = []
    lens.zero_()
    for i in range(70):
        k.copy_(torch.randn(k.shape, device=gpu))
        v.copy_(torch.randn(v.shape, device=gpu))
        rows.append((k.clone(), v.clone()))
        append_kv(twin, k, v, starts, lens, table)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], read_kv(twin, B, starts, lens, table)[0])
    assert all(torch.equal(a, b) for a, b in zip(cache[:2], twin[:2])) and lens.tolist() == [70] * B
    keys, values = ([torch.stack([x[side][b] for x in rows]) for b in range(B)] for side in (0, 1))
    expect(cache, table, keys, values)


def test_no_rows(gpu):
    cache, table = fresh(gpu, 2, 2, 1)
    k, v = new_rows(gpu, 9, 4, 2)
    lens = torch.tensor([3, 31], dtype=torch.int32, device=gpu)
    n0 = int8_kernels.STATS["launch"]
    append_kv(cache, k[:0], v[:0], starts_of([0, 0], gpu), lens, table)
    append_kv(cache, k, v, starts_of([], gpu), lens[:0], table[:0])
    assert read_kv(cache, 0, starts_of([0, 0], gpu), lens, table)[0].shape == (0, 2, D)
    assert not read_kv(cache, 5, starts_of([], gpu), lens[:0], table[:0])[1].any()
    assert int8_kernels.STATS["launch"] == n0 + 4
    assert (cache.data == -77).all() and (cache.recent == -5.0).all()


def test_refusals(gpu):
    cache, table = fresh(gpu, 2, 2, 2)
    k, v = new_rows(gpu, 10, 9, 2)
    s, n = starts_of([4, 5], gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    cos = torch.ones(50, 32, dtype=BF, device=gpu)
    w = torch.ones(D, dtype=BF, device=gpu)
    a = lambda kk=k, vv=v, st=s, ln=n, tb=table, c=cache, **kw: append_kv(c, kk, vv, st, ln, tb, **kw)  # noqa: E731
    r = lambda rows=9, st=s, ln=n, tb=table, c=cache, **kw: read_kv(c, rows, st, ln, tb, **kw)  # noqa: E731
    other = PagedKV.empty(4, 2, 4, gpu)
    bad = [
        lambda: a(kk=k.float()), lambda: a(vv=v[:8]), lambda: a(kk=k[:, :1], vv=v[:, :1]), lambda: a(st=s.long()), lambda: a(st=s.cpu()),
        lambda: a(ln=n.long()), lambda: a(ln=n[:1]), lambda: a(ln=None), lambda: a(tb=table.long()), lambda: a(tb=table[:1]),
        lambda: a(tb=table.t()), lambda: a(tb=table[:1].expand(2, -1)), lambda: a(c=other), lambda: a(c=cache._replace(data=cache.data.float())),
        lambda: a(c=cache._replace(scales=cache.scales.double())), lambda: a(c=cache._replace(recent=cache.recent[:, :, :, :16])),
        lambda: a(c=cache._replace(data=cache.data.transpose(4, 5))), lambda: a(slots=n.long()), lambda: a(slots=n[:1]),
        lambda: a(longest=-2), lambda: a(norm=(w.float(), 1.0, 1e-6)), lambda: a(norm=(w[:128], 1.0, 1e-6)),
        lambda: a(rope=(cos, cos[:9])), lambda: a(rope=(cos.half(), cos.half())), lambda: a(rope=(cos, cos.float())),
        lambda: a(rope=(cos[:, :24].contiguous(),) * 2), lambda: a(rope=(cos.t(),) * 2), lambda: a(rope=(cos, cos, n)),
        lambda: a(rope=(cos, cos, torch.zeros(9, device=gpu))), lambda: a(kk=k.cpu()),
        lambda: a(kk=k.contiguous().view(-1)[1:1 + 8 * 512].view(8, 2, D), vv=v[:8]), lambda: r(rows=-1), lambda: r(st=s[None]),
        lambda: r(ln=n.cpu()), lambda: r(c=cache._replace(data=cache.data.cpu()))]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    assert (cache.data == -77).all()
