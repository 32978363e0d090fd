"""What the packed and paged operators refuse before any device call (CPU)."""
import pytest
import torch

from mica_amd import _lib
from mica_amd.attention import packed_attention
from mica_amd.kv_cache import PagedKV, append_kv, paged_attention, read_kv

A16 = 1 << 20      # a 16-byte aligned fake address, never dereferenced: every call below is rejected first
SHAPE, DTYPE, ALIGN, STRIDE, RANGE, ARG = 1, 2, 3, 4, 5, 6
INF, NAN = float("inf"), float("nan")


def packed(**kw):
    a = dict(q=A16, shq=256, ldq=1024, k=A16, shk=256, ldk=256, v=A16, shv=256, ldv=256, o=A16, sho=256, ldo=1024, starts=A16,
             B=2, T=50, HQ=4, HK=1, d=256, scale=0.0625, fill=1, longest=0, ws=A16, nbytes=1 << 40, stream=None)
    a.update(kw)
    return _lib.load().mica_attention_packed(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(d=128), SHAPE), (dict(HQ=8), SHAPE), (dict(HK=0, HQ=0), SHAPE), (dict(B=-1), SHAPE), (dict(T=-1), SHAPE),
    (dict(scale=0.0), ARG), (dict(scale=NAN), ARG), (dict(scale=INF), ARG), (dict(q=None), ARG), (dict(k=None), ARG),
    (dict(v=None), ARG), (dict(o=None), ARG), (dict(starts=None), ARG), (dict(ldk=128), STRIDE), (dict(ldv=260), STRIDE),
    (dict(shq=4), STRIDE), (dict(ldo=-8), STRIDE), (dict(ldk=1 << 26), RANGE), (dict(q=A16 + 8), ALIGN), (dict(o=A16 + 2), ALIGN),
    (dict(starts=A16 + 2), ALIGN), (dict(T=1 << 30), RANGE), (dict(B=1 << 25, T=1 << 30), RANGE), (dict(T=0, q=None), 0),
    (dict(B=0, fill=0, q=None), 0)])
def test_packed_refuses(kw, code):
    assert packed(**kw) == code


CACHE = dict(data=A16, scales=A16, recent=A16, pages=9, n_slots=2, HK=1, d=256, table=A16, ldt=4, width=4, lens=A16, slots=None)
BAD_CACHE = [
    (dict(d=64), SHAPE), (dict(HK=0), SHAPE), (dict(pages=-1), SHAPE), (dict(n_slots=-1), SHAPE), (dict(width=-1), SHAPE),
    (dict(width=1 << 25, ldt=1 << 25), SHAPE), (dict(lens=None), ARG), (dict(recent=None), ARG), (dict(data=None), ARG),
    (dict(scales=None), ARG), (dict(table=None), ARG), (dict(ldt=3), STRIDE), (dict(data=A16 + 8), ALIGN),
    (dict(recent=A16 + 8), ALIGN), (dict(scales=A16 + 2), ALIGN), (dict(table=A16 + 1), ALIGN), (dict(lens=A16 + 2), ALIGN),
    (dict(slots=A16 + 2), ALIGN)]


def append(**kw):
    a = dict(k=A16, shk=256, ldk=256, v=A16, shv=256, ldv=256, starts=A16, B=2, T=50, **CACHE, w=None, off=1.0, eps=1e-6, rot=0,
             cos=None, sin=None, dt=0, n_pos=0, pos=None, longest=0, stream=None)
    a.update(kw)
    return _lib.load().mica_kv_append(*a.values())


@pytest.mark.parametrize("kw,code", BAD_CACHE + [
    (dict(B=-1), SHAPE), (dict(T=-1), SHAPE), (dict(rot=48), SHAPE), (dict(rot=512), SHAPE), (dict(dt=1), DTYPE), (dict(k=None), ARG),
    (dict(v=None), ARG), (dict(starts=None), ARG), (dict(rot=64), ARG), (dict(rot=64, cos=A16, sin=A16, n_pos=-1), ARG),
    (dict(ldk=100), STRIDE), (dict(shv=-8), STRIDE), (dict(k=A16 + 2), ALIGN), (dict(w=A16 + 8), ALIGN),
    (dict(rot=64, cos=A16 + 4, sin=A16), ALIGN), (dict(pos=A16 + 1), ALIGN), (dict(T=1 << 30), RANGE),
    (dict(B=1 << 24, T=1 << 24, longest=1), RANGE), (dict(T=0, k=None), 0), (dict(B=0, k=None), 0)])
def test_append_refuses(kw, code):
    assert append(**kw) == code


def read(**kw):
    a = dict(k=A16, v=A16, starts=A16, B=2, T=50, **CACHE, longest=0, stream=None)
    a.update(kw)
    return _lib.load().mica_kv_read(*a.values())


@pytest.mark.parametrize("kw,code", BAD_CACHE + [
    (dict(B=-1), SHAPE), (dict(T=-1), SHAPE), (dict(k=None), ARG), (dict(starts=None), ARG), (dict(v=A16 + 8), ALIGN),
    (dict(T=1 << 30), RANGE), (dict(T=0, k=None), 0)])
def test_read_refuses(kw, code):
    assert read(**kw) == code


def paged(**kw):
    a = dict(q=A16, shq=256, ldq=1024, o=A16, sho=256, ldo=1024, starts=A16, B=2, T=50, HQ=4, **CACHE, scale=0.0625, fill=1,
             longest=0, ws=A16, nbytes=1 << 40, stream=None)
    a.update(kw)
    return _lib.load().mica_attention_paged(*a.values())


@pytest.mark.parametrize("kw,code", BAD_CACHE + [
    (dict(B=-1), SHAPE), (dict(HQ=8), SHAPE), (dict(scale=-1.0), ARG), (dict(scale=NAN), ARG), (dict(q=None), ARG), (dict(o=None), ARG),
    (dict(ldq=4), STRIDE), (dict(sho=12), STRIDE), (dict(q=A16 + 8), ALIGN), (dict(T=1 << 30), RANGE), (dict(T=0, q=None), 0)])
def test_paged_refuses(kw, code):
    assert paged(**kw) == code


def test_workspace_sizes():
    L = _lib.load()
    assert L.mica_attention_packed_workspace_bytes(-1, 4, 4, 0) == -1 and L.mica_attention_packed_workspace_bytes(1, 4, 0, 0) == -1
    assert L.mica_attention_paged_workspace_bytes(1, -4, 4, 9, 0) == -1 and L.mica_attention_paged_workspace_bytes(1, 4, 4, -9, 0) == -1
    for B, T, HK, w, n in ((1, 1, 4, 10, 1), (64, 64, 4, 257, 1), (2 ** 20, 2 ** 30, 4, 2 ** 24, 0), (3, 5000, 1, 2 ** 24, 2 ** 31 - 1),
                           (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 16, 2 ** 24, 1)):
        assert L.mica_attention_packed_workspace_bytes(B, T, HK, n) >= 0
        assert L.mica_attention_paged_workspace_bytes(B, T, HK, w, n) >= 0


def test_cpu_tensors_are_refused():
    q, k, v = torch.zeros(4, 6, 256, dtype=torch.bfloat16).split((4, 1, 1), dim=1)
    s, n, t = torch.tensor([0, 4], dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    cache = PagedKV.empty(2, 1, 1, "cpu")
    for f in (lambda: packed_attention(q, k, v, s), lambda: append_kv(cache, k, v, s, n, t), lambda: read_kv(cache, 4, s, n, t),
              lambda: paged_attention(q, cache, s, n, t)):
        with pytest.raises(ValueError, match="GPU only"):
            f()


def test_value_order_is_bit_reversed():
    assert [int(f"{i:03b}"[::-1], 2) for i in range(8)] == [0, 4, 2, 6, 1, 5, 3, 7]
