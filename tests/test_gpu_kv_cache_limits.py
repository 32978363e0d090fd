"""append_kv at the limits of what it takes."""
import pytest
import torch
from kv_model import BF, starts_of
from test_gpu_kv_cache import expect, fresh, new_rows

from mica_amd.kv_cache import append_kv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tab", [BF, torch.float32])
def test_empty_tables_are_refused(gpu, tab):
    """Also those that lie within others, through the native path and beside it."""
    cache, table = fresh(gpu, 1, 2, 1)
    k, v = new_rows(gpu, 1, 5, 2)
    zero = torch.zeros(1, dtype=torch.int32, device=gpu)
    whole = torch.ones(40, 32, dtype=tab, device=gpu)
    for t in (torch.empty(0, 32, dtype=tab, device=gpu), whole[8:8]):
        for more in ((), (torch.zeros(5, dtype=torch.int32, device=gpu),)):
            with pytest.raises(ValueError):
                append_kv(cache, k, v, starts_of([5], gpu), zero, table, rope=(t, t, *more))
    assert (cache.recent == -5.0).all()
    append_kv(cache, k, v, starts_of([5], gpu), zero, table, rope=(whole[:1], 0 * whole[:1]))      # one position: row 0's
    assert torch.equal(cache.recent[0, 0, :, 1:5].transpose(0, 1), k[1:])


@pytest.mark.parametrize("treated", [False, True])
@pytest.mark.parametrize("step", [1000, 45, 77])
def test_the_same_bits_for_every_hint(gpu, treated, step):
    """One long sequence beside many short ones, in pieces that begin inside a block: without a hint a call of several rows looks
    for its units among the sequences, with one it has a fixed number of workgroups for each."""
    HK, total = 2, [700, 40, 33, 65, 31, 32, 1, 5, 97, 64, 20, 300]
    B = len(total)
    k, v = new_rows(gpu, 1, sum(total), HK)
    ks, vs = k.split(total), v.split(total)
    ang = torch.arange(800, device=gpu)[:, None] * 10000.0 ** (-torch.arange(32, device=gpu) / 32)
    more = dict(rope=(ang.cos().to(BF), ang.sin().to(BF)), norm=(torch.randn(256, device=gpu).to(BF), 1.0, 1e-6)) if treated else {}
    caches, searched = [], {}
    for hint in (max, None, 1):
        cache, table = fresh(gpu, B, HK, 22)
        held, searched[hint] = [0] * B, 0
        while held != total:
            counts = [min(step + 3 * b, n - h) for b, (n, h) in enumerate(zip(total, held))]
            T, longest = sum(counts), max(counts) if hint is max else hint
            kk = torch.cat([x[h:h + c] for x, h, c in zip(ks, held, counts)])
            vv = torch.cat([x[h:h + c] for x, h, c in zip(vs, held, counts)])
            each = -(-min(longest or T, T) // 32)                # workgroups a sequence, or a search for the call's units
            searched[hint] += each * B > 2 * min((T + 31 * B) // 32, T)
            append_kv(cache, kk, vv, starts_of(counts, gpu), torch.tensor(held, dtype=torch.int32, device=gpu), table, longest=longest,
                      **more)
            held = [h + c for h, c in zip(held, counts)]
        caches.append(cache)
        if not treated:
            expect(cache, table, ks, vs)
    assert searched[None] > 0 and searched[1] == 0
    for c in caches[1:]:
        assert torch.equal(c.data, caches[0].data) and torch.equal(c.scales, caches[0].scales) and torch.equal(c.recent, caches[0].recent)
