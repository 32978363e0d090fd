"""append_kv at the limits of what it takes."""
import pytest
import torch
from kv_model import BF, starts_of
from test_gpu_kv_cache import fresh, new_rows

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
