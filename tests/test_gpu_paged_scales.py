"""Pages that another quantizer has written: a value is scale x int8 for any scale, 0 and negative ones among them, and a scale
that is not finite makes its block NaN, for the rows that see it."""
import math

import pytest
import torch
from kv_model import BF, D, PAGE, Cache, attend, check, quantized, starts_of, stored

from mica_amd.kv_cache import paged_attention, read_kv

pytestmark = pytest.mark.gpu


def rescaled(gpu, lens, HK, scales, seed=3):
    """A cache whose blocks' scales are replaced, and what it stands for, a list of float32 [n, HK, 256] for each side.  scales:
    {(sequence, block, side, head): factor of the scale that the block has}."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    rows = [[torch.randn(n, HK, D, generator=g, device=gpu).to(BF) for n in lens] for _ in range(2)]
    c = Cache(gpu, *rows)
    is_ = [[stored(x) for x in side] for side in rows]
    for (b, j, side, h), f in scales.items():
        at = slice(j * PAGE, (j + 1) * PAGE)
        q, s = quantized(rows[side][b][at, h])
        s = s * f
        c.scales[c.table[b, j], side, h] = s
        is_[side][b][at, h] = q.float() * s if torch.isfinite(s) else math.nan
    return c, is_


@pytest.mark.parametrize("n", [1, 2, 4, 8, 16, 32, 40, 64, 100])
@pytest.mark.parametrize("f", [0.0, -1.0, -3.0, 1e-30, math.inf, -math.inf, math.nan])
def test_any_scale(gpu, n, f):
    """The newest rows lie in the blocks in question, so that some see a block, some a part of it and some nothing of it; in
    sequence 1 it is the last block, with no rest behind it."""
    lens, HK = [n + 140, max(n // 32 + 2, 3) * 32, 100], 2
    blocks = {(0, (lens[0] - n) // PAGE, 0, 0): f, (0, (lens[0] - n // 2) // PAGE, 1, 1): f, (1, lens[1] // PAGE - 1, 0, 1): f,
              (1, lens[1] // PAGE - 1, 1, 0): f, (0, 0, 0, 1): f}
    blocks = {key: x for key, x in blocks.items() if (key[1] + 1) * PAGE <= lens[key[0]] and (key[1] or math.isfinite(x))}
    c, (k, v) = rescaled(gpu, lens, HK, blocks)
    counts = [min(n, m) for m in lens]
    q = torch.randn(sum(counts), 4 * HK, D, generator=torch.Generator(device=gpu).manual_seed(n), device=gpu).to(BF)
    starts = starts_of(counts, gpu)
    for longest in (n, None, 1, 50):
        o = paged_attention(q, c.kv(), starts, c.lens, c.table, longest=longest)
        at = 0
        for b, m in enumerate(counts):
            check(o[at:at + m], *attend(q[at:at + m], k[b], v[b], lens[b] - m))
            at += m
    got = read_kv(c.kv(), sum(lens), starts_of(lens, gpu), c.lens, c.table)
    for x, want in zip(got, (k, v)):
        assert torch.equal(torch.nan_to_num(x, nan=99.0), torch.nan_to_num(torch.cat(want).to(BF), nan=99.0))


@pytest.mark.parametrize("n", [1, 16, 64])
def test_a_product_of_scales_below_fp32(gpu, n):
    """A block scale (1e-8 / 127 of zeros is the smallest that an append writes) times a tiny softmax scale is 0: the weights
    are even, and what a row does not see has none."""
    lens = [96, 70]
    g = torch.Generator(device=gpu).manual_seed(4)
    k, v = [[torch.randn(m, 2, D, generator=g, device=gpu).to(BF) for m in lens] for _ in range(2)]
    for x in k:
        x.zero_()
    c = Cache(gpu, k, v)
    q = torch.randn(2 * n, 8, D, generator=g, device=gpu).to(BF)
    o = paged_attention(q, c.kv(), starts_of([n, n], gpu), c.lens, c.table, longest=n, scale=1e-38)
    for b in range(2):
        at = slice(b * n, (b + 1) * n)
        check(o[at], *attend(q[at], stored(k[b]), stored(v[b]), lens[b] - n, 1e-38))
