"""The paged cache in plain torch: what its memory holds after rows have come, from the definition, and attention in float64
over what it stands for."""
import math

import torch

BF, PAGE, D = torch.bfloat16, 32, 256
FOURS = [0, 4, 2, 6, 1, 5, 3, 7]


def quantized(x):
    """Blocks of bf16 rows [..., 32, 256] -> (int8 of the same shape, fp32 scales [...])."""
    x = x.float()
    top = x.abs().amax((-1, -2))
    s = torch.clamp(top, min=1e-8) / torch.tensor(127.0, device=x.device)
    q = torch.round(x / s[..., None, None]).clamp(-127, 127)
    fine = torch.isfinite(x).all(-1).all(-1)
    return torch.where(fine[..., None, None], q, 0.0).to(torch.int8), torch.where(fine, s, math.nan)


def key_page(q):
    """[HK, 32, 256] int8 -> a page's keys [HK, 8, 32, 32]."""
    return q.view(-1, PAGE, 8, 32).transpose(1, 2)


def value_page(q):
    """[HK, 32, 256] int8 -> a page's values [HK, 8, 32, 32]."""
    return q.transpose(1, 2).reshape(-1, D, 8, 4)[:, :, FOURS].reshape(-1, 8, 32, PAGE)


def stored(rows):
    """bf16 rows [n, HK, 256] of a whole sequence -> what the cache stands for, float32 [n, HK, 256]."""
    n, full = rows.shape[0], rows.shape[0] // PAGE * PAGE
    out = rows.float().clone()
    if full:
        blocks = rows[:full].view(-1, PAGE, rows.shape[1], D).transpose(1, 2)
        q, s = quantized(blocks)
        out[:full] = (q.float() * s[..., None, None]).transpose(1, 2).reshape(full, rows.shape[1], D)
    return out


class Cache:
    """A cache filled from whole sequences' bf16 rows, with pages in a random order and slots given."""

    def __init__(self, gpu, keys, values, seed=0, spare=3, extra=2, slots=None, shared=0):
        """keys / values: a list of [n, HK, 256] bf16 rows; shared: the first blocks of all sequences, in the same pages."""
        g = torch.Generator().manual_seed(seed)
        HK, B = keys[0].shape[1], len(keys)
        full = [k.shape[0] // PAGE for k in keys]
        total = shared + sum(max(0, f - shared) for f in full)
        order = torch.randperm(total + spare, generator=g).tolist()
        self.lens = torch.tensor([k.shape[0] for k in keys], dtype=torch.int32, device=gpu)
        self.table = torch.full((B, max(full) + extra), -7, dtype=torch.int32)
        self.slots = None if slots is None else torch.tensor(slots, dtype=torch.int32, device=gpu)
        n_slots = B if slots is None else max(slots) + 2
        # what is no token's is garbage that must not be read into anything
        self.data = torch.randint(-127, 128, (total + spare, 2, HK, 8, 32, 32), generator=g, dtype=torch.int32).to(torch.int8).to(gpu)
        self.scales = torch.full((total + spare, 2, HK), math.nan, device=gpu)
        self.recent = torch.full((n_slots, 2, HK, PAGE, D), math.inf, dtype=BF, device=gpu)
        at = shared
        for b, (k, v) in enumerate(zip(keys, values)):
            for j in range(full[b]):
                if j < shared:
                    page = order[j]
                else:
                    page, at = order[at], at + 1
                self.table[b, j] = page
                for side, (x, lay) in enumerate(((k, key_page), (v, value_page))):
                    q, s = quantized(x[j * PAGE:(j + 1) * PAGE].transpose(0, 1))
                    self.data[page, side], self.scales[page, side] = lay(q), s
            left, slot = k.shape[0] % PAGE, b if slots is None else slots[b]
            for side, x in enumerate((k, v)):
                self.recent[slot, side, :, :left] = x[full[b] * PAGE:].transpose(0, 1)
        self.table = self.table.to(gpu)

    def kv(self):
        from mica_amd.kv_cache import PagedKV
        return PagedKV(self.data, self.scales, self.recent)


def starts_of(counts, gpu, before=0):
    return torch.tensor([before, *counts], dtype=torch.int32).cumsum(0, dtype=torch.int32).to(gpu)


def attend(q, k, v, first, scale=1 / 16):
    """(o, A) in float64 of one sequence: q [n, HQ, 256] at positions first, first + 1, ...; k / v [S, HK, 256] as the cache
    stands for them; A = sum p |v|.  Zeros for positions below 0; what a row does not see takes no part, whatever it holds."""
    n, HQ, _ = q.shape
    S, HK, _ = k.shape
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    if not S or not n:
        return o, a
    at = first + torch.arange(n, device=q.device)
    sees = torch.arange(S, device=q.device)[None] <= at[:, None]
    for h in range(HQ):
        z = q[:, h].double() @ k[:, h * HK // HQ].double().t() * scale
        bad = (sees & torch.isnan(z)).any(1)
        z = torch.where(sees, z, -math.inf)
        m = z.nan_to_num(nan=0.0, neginf=-math.inf).amax(1, keepdim=True)
        w = torch.where(sees, torch.exp(z - torch.where(torch.isfinite(m), m, 0.0)), 0.0)
        t = w.sum(1, keepdim=True)
        w = torch.where(at[:, None] < 0, 0.0, w / t)
        vv = v[:, h * HK // HQ].double()
        odd = ~torch.isfinite(vv)
        fine = torch.where(odd, 0.0, vv)
        o[:, h], a[:, h] = w @ fine, w @ fine.abs()
        for key in odd.any(1).nonzero()[:, 0].tolist():
            o[:, h] += torch.where((w[:, key:key + 1] > 0) & odd[key], w[:, key:key + 1] * vv[key], 0.0)
        o[bad, h] = math.nan
    return o, a


def check(got, o, a):
    """Each weight is rounded to bf16 (half a step, 2^-8) before the product with v, the result once more; the scores are fp32
    sums of 256 products (off by at most 256 x 2^-24 x sum |q k| / 16, about 2e-4 for unit normal heads) and twice that reaches
    the weights.  With A = sum p |v|:  |o - ref| <= 2^-8 (A + |ref|) + 2^-11 A.  A scale of the cache multiplies scores and
    weights in fp32 (2^-24 each), within that."""
    got = got.double()
    odd = ~torch.isfinite(o)
    assert torch.equal(odd, ~torch.isfinite(got)), "values that are not finite reach other rows than those that see them"
    assert torch.equal(torch.isnan(o), torch.isnan(got))
    d = torch.where(odd, 0.0, got - o).abs() - (2 ** -8 * (a + o.abs()) + 2 ** -11 * a)
    assert (torch.where(odd, 0.0, d) <= 0).all(), f"off by {d.max():.3g} more than the roundings allow"
