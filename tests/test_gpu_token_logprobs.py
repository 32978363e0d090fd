"""readout.token_logprobs against log-softmax in float64.

Tolerance: a thread adds up to n = V / 256 terms one after the other in fp32, 2^-24 each at most, then 256 threads in a
tree, and an exponential is off by about 2^-22: d = (n + 64) 2^-24 + 2^-22 of S and, relative to sum e^y |y|, of the
entropy's sum.  So |lp - ref| <= d + 2^-22 |lp| + 2^-22 M-differences, |H - ref| <= d (1 + 2 H) + 2^-22 H."""
import math

import pytest
import torch

from mica_amd import int8_kernels
from mica_amd.readout import MAX_TOP, token_logprobs

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def ref(x, tokens, top):
    x = x.double()
    lp = x - x.amax(1, keepdim=True)          # first: near 1e38 the logarithm would be lost beside the maximum
    lp = lp - torch.log(torch.exp(lp).sum(1, keepdim=True))
    p = torch.exp(lp)
    ent = -torch.where(p > 0, p * lp, 0.0 * p).sum(1)
    order = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    t = tokens.long().view(x.shape[0], -1)
    ok = (t >= 0) & (t < x.shape[1])
    got = torch.where(ok, lp.gather(1, t.clamp(0, x.shape[1] - 1)), math.nan).view(tokens.shape)
    return got, ent, order, lp.gather(1, order)


def near(a, b, tol):
    a, odd = a.double(), ~torch.isfinite(b)
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a[odd & ~torch.isnan(b)], b[odd & ~torch.isnan(b)])
    d = (a - b).abs() - tol
    assert (d[~odd] <= 0).all(), f"off by {d[~odd].max():.3g} more than allowed"


def check(out, x, tokens, top):
    got, ent, ids, best = ref(x, tokens, top)
    d = (x.shape[1] / 256 + 64) * 2 ** -24 + 2 ** -22
    assert out.logprobs.shape == tokens.shape and out.logprobs.dtype == torch.float32 and out.top_ids.dtype == torch.int64
    near(out.logprobs, got, d + 2 ** -21 * got.abs())
    near(out.entropy, ent, d * (1 + 2 * ent.abs()) + 2 ** -21 * ent.abs())
    assert torch.equal(out.top_ids, ids), "top alternatives"
    near(out.top_logprobs, best, d + 2 ** -21 * best.abs())


def rows(gpu, T, V, dtype, seed=0, spread=2.5):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return (torch.randn(T, V, generator=g, device=gpu) * spread).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,top,C", [
    (1, 1, 1, 1), (1, 7, 7, 1), (3, 33, 32, 2), (2, 300, 20, 1), (5, 2047, 1, 3), (1, 8193, 32, 1), (2, 32003, 7, 40),
    (1, 151936, 5, 1), (3, 151936, 20, 1), (1100, 16411, 20, 1), (1030, 501, 0, 2), (2, 200001, 32, 0)])
def test_against_float64(gpu, dtype, T, V, top, C):
    x = rows(gpu, T, V, dtype, V + T)
    tokens = torch.randint(0, V, (T,) if C == 1 else (T, C), device=gpu)
    check(token_logprobs(x, tokens, top), x, tokens, top)
    i32 = tokens.int()
    assert all(torch.equal(a, b) for a, b in zip(token_logprobs(x, tokens, top), token_logprobs(x, i32, top)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off", range(9))
def test_every_alignment_of_a_row(gpu, dtype, off):
    wide = rows(gpu, 3, 20011, dtype, off)
    for width in (1, 3, 5, 17, 8200, 20000):
        x = wide[:, off:off + width]
        tokens = torch.tensor([0, width - 1, width // 2], device=gpu)
        check(token_logprobs(x, tokens, min(width, 9)), x, tokens, min(width, 9))


@pytest.mark.parametrize("T", [2, 1030])
@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_index(gpu, dtype, T):
    V = 30011
    x = torch.zeros(T, V, dtype=dtype, device=gpu)            # all equal
    x[1] = torch.randint(0, 3, (V,), device=gpu).to(dtype)    # three values
    if T > 2:
        x[2] = -torch.arange(V, device=gpu) // 700           # long runs, falling
        x[3] = torch.arange(V, device=gpu) // 700            # and rising (fp16 and bf16 round: longer runs)
        x[4, ::2] = -0.0                                       # -0 equals 0
        x[5, :] = -math.inf
        x[5, V - 25:] = 1.0                                   # only the end of the row counts
        x[6, V - 3:] = 5.0
        x[7, :] = torch.finfo(dtype).min                      # the type's lowest value is a value
        x[8, 5:] = -math.inf                                  # fewer possible tokens than alternatives
    tokens = torch.randint(0, V, (T,), device=gpu)
    check(token_logprobs(x, tokens, 20), x, tokens, 20)


@pytest.mark.parametrize("top", [1, 20, 32])
@pytest.mark.parametrize("T", [4, 1026])
def test_orders_that_bring_many_candidates(gpu, T, top):
    """Rising rows (every element is the largest so far), and rows whose blocks bring from a few to thousands of them."""
    V = 50021
    x = rows(gpu, T, V, torch.float32, 9)
    up = torch.arange(V, device=gpu, dtype=torch.float32)
    x[0] = up / 4096
    x[1] = up // 8 / 4096 - up % 8                 # eight rising runs
    x[2] += up / 2000                               # a slope under the noise: some of each block
    x[3] = torch.where(up % 37 == 0, up / 4096, x[3] - 9)
    tokens = torch.randint(0, V, (T,), device=gpu)
    check(token_logprobs(x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 250, 1015, 1016, 1017, 1500, 2031, 2032, 2033, 2050])
def test_short_rows(gpu, dtype, V):
    """Rows of up to a few vectors a lane: ordinary ones, ties, -inf, rising and falling ones, at every alignment."""
    T = 2060
    x = rows(gpu, T, V + 1, dtype, V)[:, 1:]            # (rows V + 1 apart: each begins elsewhere)
    up = torch.arange(V, device=gpu)
    x[0], x[1], x[2], x[3] = 0.0, -math.inf, up // 9, -up // 9
    x[4, 3:] = -math.inf
    x[5], x[6] = torch.finfo(dtype).min, up % 2
    x[7, ::5] = -math.inf
    for top in (0, 1, 20, 32):
        tokens = torch.randint(0, V, (T, 3), device=gpu)
        out = token_logprobs(x, tokens, top)
        assert torch.isnan(out.logprobs[1]).all() and out.top_ids[1].tolist() == list(range(top))
        keep = [i for i in range(T) if i != 1]
        check(type(out)(*(o[keep] for o in out)), x[keep], tokens[keep], top)


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 2100), (torch.bfloat16, 4064), (torch.float16, 4065), (torch.float32, 2032)])
def test_many_short_rows(gpu, dtype, V):
    T = 4099
    x = rows(gpu, T, V, dtype, V)
    up = torch.arange(V, device=gpu)
    x[0], x[1], x[2], x[3] = 0.0, up % 2, up // 17, -up // 17
    x[4, : V // 2] = -math.inf
    x[5, V // 2:] = -math.inf
    tokens = torch.randint(0, V, (T,), device=gpu)
    for top in (0, 32):
        check(token_logprobs(x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("T", [3, 1026])
def test_a_nan_in_every_thread(gpu, T):
    V = 30000
    x = rows(gpu, T, V, torch.bfloat16, 4)
    x[0, ::7] = math.nan
    x[1, ::301] = math.nan                          # from then on a thread looks at all its elements
    x[2, 5::8192] = math.nan
    out = token_logprobs(x, torch.zeros(T, dtype=torch.int64, device=gpu), 32)
    for row, step in ((0, 7), (1, 301)):
        assert out.top_ids[row].tolist() == [i * step for i in range(32)] and torch.isnan(out.entropy[row])
    best = torch.sort(torch.nan_to_num(x[2].float(), nan=-math.inf), descending=True, stable=True).indices
    assert out.top_ids[2].tolist() == [5, 8197, 16389, 24581] + best[:28].tolist()


@pytest.mark.parametrize("T", [6, 1030])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_and_nan_logits(gpu, dtype, T):
    V = 20003
    x = rows(gpu, T, V, dtype, 5)
    x[0, ::2] = -math.inf
    x[1] = -math.inf
    x[2, 12345] = math.inf
    x[3, 777], x[3, 19999] = math.nan, -math.nan
    x[4, 1:] = -math.inf
    x[5] = math.nan
    tokens = torch.randint(0, V, (T,), device=gpu)
    out = token_logprobs(x, tokens, 8)
    r = list(ref(x, tokens, 8))
    d = (V / 256 + 64) * 2 ** -24 + 2 ** -22
    for row in (1, 2, 3, 5):      # no distribution
        assert all(torch.isnan(v[row]).all() for v in (out.logprobs, out.entropy, out.top_logprobs))
    keep = [i for i in range(T) if i not in (1, 2, 3, 5)]
    near(out.logprobs[keep], r[0][keep], d + 2 ** -21 * r[0][keep].abs())
    near(out.entropy[keep], r[1][keep], d * (1 + 2 * r[1][keep]) + 2 ** -21 * r[1][keep])
    near(out.top_logprobs[keep], r[3][keep], d + 2 ** -21 * r[3][keep].abs())
    assert torch.equal(out.top_ids[keep], r[2][keep])
    assert out.top_ids[1].tolist() == out.top_ids[5].tolist() == list(range(8))
    assert out.top_ids[2, 0] == 12345 and torch.equal(out.top_ids[2], r[2][2])
    assert out.top_ids[3, :2].tolist() == [777, 19999]     # NaN counts as the largest
    assert float(out.entropy[4]) == 0.0 and float(out.top_logprobs[4, 0]) == 0.0


def test_ids_that_are_no_tokens(gpu):
    x = rows(gpu, 3, 1000, torch.bfloat16)
    tokens = torch.tensor([[0, -1, 999], [1000, 5, 2 ** 40], [-2 ** 40, 999, 1]], device=gpu)
    check(token_logprobs(x, tokens, 3), x, tokens, 3)


def test_large_and_small_logits(gpu):
    for spread in (1e-3, 200.0, 3e4):
        x = rows(gpu, 4, 9000, torch.float32, 9, spread)
        x += 1e4 if spread < 1 else 0.0
        tokens = torch.randint(0, 9000, (4,), device=gpu)
        check(token_logprobs(x, tokens, 6), x, tokens, 6)


def test_streams_and_graphs(gpu):
    x, tokens = rows(gpu, 5, 50000, torch.bfloat16), torch.randint(0, 50000, (5, 2), device=gpu)
    want = token_logprobs(x, tokens, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_logprobs(x, tokens, 9)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(x, tokens, 9)
    for i in range(3):
        x.copy_(torch.randn(x.shape, device=gpu))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(token_logprobs(x, tokens, 9), out))


def test_nothing_to_do_and_refusals(gpu):
    x, tokens = rows(gpu, 4, 100, torch.bfloat16), torch.zeros(4, dtype=torch.long, device=gpu)
    n0 = int8_kernels.STATS["launch"]
    out = token_logprobs(x[:0], tokens[:0], 3)
    assert out.logprobs.shape == (0,) and out.top_ids.shape == (0, 3) and int8_kernels.STATS["launch"] == n0 + 1
    bad = [lambda: token_logprobs(x.cpu(), tokens), lambda: token_logprobs(x.double(), tokens), lambda: token_logprobs(x[0], tokens),
           lambda: token_logprobs(x.t(), tokens), lambda: token_logprobs(x, tokens[:3]), lambda: token_logprobs(x, tokens.cpu()),
           lambda: token_logprobs(x, tokens.float()), lambda: token_logprobs(x, tokens, -1), lambda: token_logprobs(x, tokens, MAX_TOP + 1),
           lambda: token_logprobs(x[:, :5], tokens, 6), lambda: token_logprobs(x[:, :0], tokens, 0),
           lambda: token_logprobs(x[:1].expand(4, -1), tokens)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
