"""attention.packed_attention against attention in float64 (the bound is derived beside kv_model.check)."""
import math

import pytest
import torch
from kv_model import BF, attend, check, starts_of

from mica_amd import int8_kernels
from mica_amd.attention import causal_gqa_attention, packed_attention

pytestmark = pytest.mark.gpu


def rows(gpu, seed, T, HK):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.randn(T, 6 * HK, 256, generator=g, device=gpu).to(BF).split((4 * HK, HK, HK), dim=1)


def check_all(o, q, k, v, counts, before=0, scale=1 / 16):
    lo = before
    for n in counts:
        at = slice(lo, lo + n)
        check(o[at], *attend(q[at], k[at], v[at], 0, scale))
        lo += n
    return lo


CASES = [([1], 1), ([1, 1, 1], 4), ([0, 5, 0, 0, 33, 0], 2), ([31, 32, 33, 64, 65, 1], 4), ([257], 4), ([700, 2, 90], 1),
         ([1000, 0, 37, 999], 2), (list(range(1, 70)), 1), ([3] * 200, 2), ([1, 2050], 4), ([40] * 65 + [500], 1)]


@pytest.mark.parametrize("counts,HK", CASES)
@pytest.mark.parametrize("hint", [False, True])
def test_against_float64(gpu, counts, HK, hint):
    q, k, v = rows(gpu, sum(counts), sum(counts), HK)
    o = packed_attention(q, k, v, starts_of(counts, gpu), longest=max(counts) if hint else None)
    check_all(o, q, k, v, counts)


def test_the_hint_may_be_wrong(gpu):
    counts = [700, 3, 90]
    q, k, v = rows(gpu, 1, sum(counts), 4)
    for longest in (1, 40, 10 ** 9):
        check_all(packed_attention(q, k, v, starts_of(counts, gpu), longest=longest), q, k, v, counts)


def test_rows_of_no_sequence(gpu):
    """Zeros in a new output, as they were in a given one; what they hold reaches nothing."""
    counts, before, behind = [70, 0, 33], 41, 100
    T = before + sum(counts) + behind
    q, k, v = (x.clone() for x in rows(gpu, 2, T, 2))
    for x in (q, k, v):
        x[:before], x[T - behind:] = math.nan, math.inf
    starts = starts_of(counts, gpu, before)
    o = packed_attention(q, k, v, starts)
    assert check_all(o, q, k, v, counts, before) == T - behind
    assert not o[:before].any() and not o[T - behind:].any()
    wide = torch.full((T, 8, 512), 7.0, dtype=BF, device=gpu)
    got = packed_attention(q, k, v, starts, out=wide[:, :, 128:384])
    assert got.data_ptr() == wide[:, :, 128:].data_ptr()
    assert torch.equal(got[before:T - behind], o[before:T - behind])
    got[before:T - behind] = 7.0
    assert (wide == 7.0).all()
    for s in ([0], [5], [0, 0], [T, T], [9, 9, 9]):        # nobody has rows
        assert not packed_attention(q, k, v, torch.tensor(s, dtype=torch.int32, device=gpu)).any()


def test_strided_rows_and_scale(gpu):
    counts = [50, 129]
    T = sum(counts)
    q, _, _ = rows(gpu, 3, T, 2)
    heads_apart = torch.randn(2, T, 256, device=gpu).to(BF).transpose(0, 1)      # [HK, T, 256] memory
    wide = torch.randn(T, 5, 320, device=gpu).to(BF)[:, 1:3, 64:]
    o = packed_attention(q, heads_apart, wide, starts_of(counts, gpu), scale=0.1)
    check_all(o, q, heads_apart, wide, counts, scale=0.1)


def test_one_sequence_is_causal_attention(gpu):
    q, k, v = rows(gpu, 4, 333, 4)
    o, c = packed_attention(q, k, v, starts_of([333], gpu)), causal_gqa_attention(q[None], k[None], v[None])[0]
    assert (o.float() - c.float()).abs().max() <= 2 ** -6      # two results of one bf16 step at most 4 each apart


@pytest.mark.parametrize("counts", [[40, 90], [600, 5, 300]])
def test_values_not_finite_reach_only_who_sees_them(gpu, counts):
    q, k, v = rows(gpu, 5, sum(counts), 2)
    n = counts[0]
    v[n - 3, 0, 5], v[n - 20, 1, 9], v[n, 0, 100], v[n + 3, 0, 100] = math.inf, math.nan, -math.inf, math.inf
    v[0, 1, 7] = -math.inf
    k[n - 1] = math.nan
    o = packed_attention(q, k, v, starts_of(counts, gpu))
    check_all(o, q, k, v, counts)
    assert torch.isnan(o[n - 1]).all()


def test_scores_beyond_every_margin(gpu):
    """Scores of hundreds, and rows whose scores are all -inf."""
    q, k, v = rows(gpu, 6, 150, 2)
    q = (q.float() * 30).to(BF)
    o = packed_attention(q, k, v, starts_of([150], gpu)).double()
    r, a = attend(q, k, v, 0)
    # scores are 30 times the unit ones: their fp32 error too, 30 x 2e-4, and twice that in the weights
    assert ((o - r).abs() <= 2 ** -8 * (a + r.abs()) + 0.012 * a).all()
    q, k = torch.ones_like(q), k.clone()
    k[:] = -math.inf
    assert torch.isnan(packed_attention(q, k, v, starts_of([150], gpu))).all()


def test_offsets_past_32_bits(gpu):
    """Rows 16 KB apart: the last sequence lies past 2^32 bytes."""
    T = 300_000
    x = torch.zeros(T, 8192, dtype=BF, device=gpu)
    rowsv = x.view(T, 32, 256)
    q, k, v = rowsv[:, :4], rowsv[:, 4:5], rowsv[:, 5:6]
    g = torch.Generator(device=gpu).manual_seed(7)
    rowsv[-100:, :6] = torch.randn(100, 6, 256, generator=g, device=gpu).to(BF)
    o = packed_attention(q, k, v, starts_of([10, T - 110, 100], gpu)[[0, 1, 1, 2, 3]].contiguous(), longest=T)
    check(o[-100:], *attend(q[-100:], k[-100:], v[-100:], 0))
    assert not o[:-100].any()


def test_starts_that_are_none(gpu):
    """Values outside 0 .. T and falling ones touch no other memory: nothing is faulted, and the sequences that are right stay so."""
    q, k, v = rows(gpu, 8, 100, 2)
    want = packed_attention(q, k, v, starts_of([60, 40], gpu))
    got = packed_attention(q, k, v, torch.tensor([-5, 60, 2 ** 30], dtype=torch.int32, device=gpu))
    assert torch.equal(got, want)
    got = packed_attention(q, k, v, torch.tensor([0, 60, 20, 7], dtype=torch.int32, device=gpu), out=torch.zeros_like(want))
    assert torch.equal(got[:60], want[:60]) and not got[60:].any()


def test_streams_and_graphs(gpu):
    """A side stream, and a captured graph replayed with other starts and the program's own calls between."""
    q, k, v = rows(gpu, 9, 900, 4)
    starts = starts_of([500, 0, 37, 300], gpu)
    call = lambda: packed_attention(q, k, v, starts, longest=900)  # noqa: E731
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
        counts = [[500, 0, 37, 300], [1, 899, 0, 0], [225] * 4, [0, 0, 0, 0]][i]
        q.copy_(torch.randn(q.shape, device=gpu))
        starts.copy_(starts_of(counts, gpu))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(call(), out)
        check_all(out, q, k, v, counts)


def test_the_same_bits_at_every_call(gpu):
    for counts in ([2000, 3, 700], [40] * 65):
        q, k, v = rows(gpu, 10, sum(counts), 4)
        starts = starts_of(counts, gpu)
        first = packed_attention(q, k, v, starts, longest=max(counts))
        for _ in range(4):
            assert torch.equal(packed_attention(q, k, v, starts, longest=max(counts)), first)


def test_no_rows(gpu):
    q, k, v = rows(gpu, 11, 4, 2)
    n0 = int8_kernels.STATS["launch"]
    assert packed_attention(q[:0], k[:0], v[:0], starts_of([0, 0], gpu)).shape == (0, 8, 256)
    assert int8_kernels.STATS["launch"] == n0 + 1


def test_refusals(gpu):
    q, k, v = rows(gpu, 12, 20, 2)
    s = starts_of([12, 8], gpu)
    bad = [
        lambda: packed_attention(q.float(), k, v, s), lambda: packed_attention(q, k[:9], v[:9], s),
        lambda: packed_attention(q[:, :4], k, v, s), lambda: packed_attention(q, k, v[:, :1], s),
        lambda: packed_attention(q[None], k, v, s), lambda: packed_attention(q[..., :128], k[..., :128], v[..., :128], s),
        lambda: packed_attention(q, k, v, s.long()), lambda: packed_attention(q, k, v, s.cpu()),
        lambda: packed_attention(q, k, v, s[:0]), lambda: packed_attention(q, k, v, s[None]),
        lambda: packed_attention(q, k, v, s, longest=-1), lambda: packed_attention(q, k, v, s, scale=0.0),
        lambda: packed_attention(q, k, v, s, scale=math.inf), lambda: packed_attention(q, k, v, s, out=q[:9]),
        lambda: packed_attention(q, k, v, s, out=torch.empty(20, 8, 256, device=gpu)), lambda: packed_attention(q, k.cpu(), v, s),
        lambda: packed_attention(q, k, v, s, out=torch.empty(1, 8, 256, device=gpu, dtype=BF).expand(20, -1, -1)),
        lambda: packed_attention(q, k[:1].expand(20, -1, -1), v, s),                                           # rows overlap
        lambda: packed_attention(q.contiguous().view(-1)[1:1 + 19 * 8 * 256].view(19, 8, 256), k[:19], v[:19], s)]   # misaligned
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
