"""What the scoring operators refuse before any device call, and the tree masks (CPU)."""
import pytest
import torch

from mica_amd import _lib
from mica_amd.attention import tree_attention, tree_masks, window_attention
from mica_amd.readout import token_logprobs

A16 = 1 << 20      # a 16-byte aligned fake address, never dereferenced: every call below is rejected first
SHAPE, DTYPE, ALIGN, STRIDE, RANGE, ARG = 1, 2, 3, 4, 5, 6


def lp(**kw):
    a = dict(logits=A16, dtype=0, ldx=1000, T=4, V=1000, tokens=A16, t64=1, C=1, top=5, lp=A16, ent=A16, ids=A16, tlp=A16,
             ws=A16, nbytes=1 << 30, stream=None)
    a.update(kw)
    return _lib.load().mica_token_logprobs(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), DTYPE), (dict(T=-1), SHAPE), (dict(V=0), SHAPE), (dict(top=33), SHAPE), (dict(V=4, ldx=4), SHAPE),
    (dict(C=-1), SHAPE), (dict(logits=None), ARG), (dict(ent=None), ARG), (dict(tokens=None), ARG), (dict(lp=None), ARG),
    (dict(ids=None), ARG), (dict(tlp=None), ARG), (dict(ldx=999), STRIDE), (dict(logits=A16 + 1), ALIGN),
    (dict(dtype=2, logits=A16 + 2), ALIGN), (dict(tokens=A16 + 4), ALIGN), (dict(ids=A16 + 4), ALIGN),
    (dict(V=100000, ldx=100000, nbytes=16), ARG), (dict(V=100000, ldx=100000, ws=None), ARG),
    (dict(V=100000, ldx=100000, ws=A16 + 8), ARG), (dict(V=(1 << 30) + 1, ldx=1 << 31, T=2000), RANGE),
    (dict(T=0, logits=None), 0)])
def test_token_logprobs_refuses(kw, code):
    assert lp(**kw) == code


def tree(**kw):
    a = dict(q=A16, sbq=0, shq=256, ldq=1024, k=A16, sbk=0, shk=256, ldk=256, v=A16, sbv=0, shv=256, ldv=256, kc=A16, sbkc=0,
             shkc=256, ldkc=256, vc=A16, sbvc=0, shvc=256, ldvc=256, cap=100, len=None, tree=A16, sbt=0, o=A16, sbo=0,
             sho=256, ldo=1024, B=1, N=8, HQ=4, HK=1, d=256, scale=0.0625, ws=A16, nbytes=1 << 30, stream=None)
    a.update(kw)
    return _lib.load().mica_attention_tree(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(d=128), SHAPE), (dict(HQ=8), SHAPE), (dict(N=513), SHAPE), (dict(N=-1), SHAPE), (dict(B=-1), SHAPE),
    (dict(cap=-1), SHAPE), (dict(HK=0, HQ=0), SHAPE), (dict(scale=0.0), ARG), (dict(scale=float("nan")), ARG),
    (dict(scale=float("inf")), ARG), (dict(q=None), ARG), (dict(tree=None), ARG), (dict(kc=None), ARG), (dict(vc=None), ARG),
    (dict(o=None), ARG), (dict(ldk=128), STRIDE), (dict(ldkc=0), STRIDE), (dict(ldvc=260), STRIDE), (dict(sbq=-8), STRIDE),
    (dict(shkc=4), STRIDE), (dict(sbt=-1), STRIDE), (dict(ldkc=1 << 26), RANGE), (dict(q=A16 + 8), ALIGN),
    (dict(vc=A16 + 2), ALIGN), (dict(tree=A16 + 4), ALIGN), (dict(cap=100000, nbytes=1000), ARG),
    (dict(cap=100000, ws=None), ARG), (dict(B=1 << 25), RANGE), (dict(N=0, q=None), 0), (dict(B=0, q=None), 0)])
def test_tree_refuses(kw, code):
    assert tree(**kw) == code


def window(**kw):
    a = dict(q=A16, sbq=0, shq=256, ldq=1024, k=A16, sbk=0, shk=256, ldk=256, v=A16, sbv=0, shv=256, ldv=256, o=A16, sbo=0,
             sho=256, ldo=1024, B=1, Sq=8, Sk=100, HQ=4, HK=1, d=256, scale=0.0625, window=50, sinks=4, len=None, ws=A16,
             nbytes=1 << 30, stream=None)
    a.update(kw)
    return _lib.load().mica_attention_window(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(d=64), SHAPE), (dict(HQ=5), SHAPE), (dict(Sk=-1), SHAPE), (dict(window=0), SHAPE), (dict(sinks=-1), SHAPE),
    (dict(scale=-1.0), ARG), (dict(k=None), ARG), (dict(o=None), ARG), (dict(ldk=8), STRIDE), (dict(ldv=1 << 26), RANGE),
    (dict(sbo=12), STRIDE), (dict(k=A16 + 4), ALIGN), (dict(Sk=100000, window=90000, nbytes=0), ARG), (dict(Sq=0), 0)])
def test_window_refuses(kw, code):
    assert window(**kw) == code


def test_workspace_sizes_refuse():
    L = _lib.load()
    assert L.mica_token_logprobs_workspace_bytes(4, 1000, 0, 33) == -1 and L.mica_token_logprobs_workspace_bytes(4, 5, 0, 6) == -1
    assert L.mica_token_logprobs_workspace_bytes(0, 5, 0, 1) == 0 and L.mica_token_logprobs_workspace_bytes(4, 5, 4, 1) == -1
    assert L.mica_attention_tree_workspace_bytes(1, 513, 4, 10) == -1 and L.mica_attention_tree_workspace_bytes(1, 8, 0, 10) == -1
    assert L.mica_attention_window_workspace_bytes(1, 8, 10, 4, 0, 0) == -1


@pytest.mark.parametrize("N,Sk,win,sinks", [(1, 10 ** 9, 2 ** 31 - 1, 2 ** 31 - 1), (2 ** 20, 2 ** 31 - 1, 2 ** 31 - 1, 0), (1, 2 ** 31 - 1, 1, 4)])
def test_sizes_at_the_end_of_int(N, Sk, win, sinks):
    """Workspace sizes neither overflow nor turn negative."""
    assert _lib.load().mica_attention_window_workspace_bytes(1, N, Sk, 1, win, sinks) >= 0
    assert _lib.load().mica_attention_tree_workspace_bytes(64, 512, 4, 2 ** 31 - 1) >= 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 6, 256, dtype=torch.bfloat16)
    q, k, v = x.split((4, 1, 1), dim=2)
    for f in (lambda: tree_attention(q, k, v, tree_masks([-1, 0, 1, 2])), lambda: window_attention(q, k, v, 4),
              lambda: token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long))):
        with pytest.raises(ValueError, match="GPU only"):
            f()


def test_tree_masks():
    m = tree_masks([-1, 0, 0, 1, -1, -2])
    assert m.tolist() == [[1], [3], [5], [11], [16], [0]] and m.dtype == torch.int64
    chain = tree_masks(torch.arange(-1, 129))
    for i in (0, 63, 64, 127, 129):
        bits = sum((w & (2 ** 64 - 1)) << 64 * j for j, w in enumerate(chain[i].tolist()))
        assert bits == 2 ** (i + 1) - 1
    assert tree_masks([[-1, 0], [-1, -1]]).tolist() == [[[1], [3]], [[1], [2]]]
    assert tree_masks(torch.zeros(0, dtype=torch.long)).shape == (0, 0)
    for bad in ([0], [-1, 1], [-1, 2, 0], [-3], [-1, -2, 1], [[[-1]]], [0.5], list(range(-1, 512))):
        with pytest.raises(ValueError):
            tree_masks(bad)
