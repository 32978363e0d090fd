"""A paged key/value cache in 8 bits on the gfx950 HIP kernels (head dim 256), for one attention layer and many sequences.

  append_kv        new rows into the cache, their keys normed and rotated on the way
  paged_attention  each sequence's newest rows over its cached tokens: single tokens, drafts, questions
  read_kv          rows of the cache back in bf16, for the operators that take a bf16 cache

A sequence's tokens lie in blocks of 32 (``PAGE``).  A finished block is one of the cache's pages, int8 with one scale for each
head and side; the block that a sequence has not filled yet stays in bf16 in the sequence's slot.  Every value is rounded to 8
bits once, and what the cache holds depends on the tokens, not on the calls that brought them.  Pages may be shared, e.g. a
state's by the questions about it.  The reference keeps its prefixes' keys and values in bf16, one tensor each
(v0.5/serving/lib/prefill_engine.py:218-226).

The rows of a call are packed, sequence b's being starts[b] .. starts[b + 1] - 1.  GPU only; no fallback.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .attention import GROUP, HEAD_DIM, _counts, _hint, _out, _rows, _scale, _starts
from .int8_kernels import _gpu_ok, _launched, _native, _on, _stream

PAGE = 32        # tokens of a block


class PagedKV(NamedTuple):
    """The cache's memory: data int8 [pages, 2, HK, 8, 32, 32], scales fp32 [pages, 2, HK], recent bf16 [slots, 2, HK, 32, 256],
    all contiguous; axis 1 is keys, values.

    Keys of a page lie as [8 groups of 32 dims][32 tokens][32 dims], values as [256 dims][32 tokens], the tokens in fours in
    the order 0 4 2 6 1 5 3 7; a value is scale x int8, NaN where the scale is not finite (an append writes positive ones).  A
    sequence of n tokens needs n // 32 pages and a slot."""

    data: torch.Tensor
    scales: torch.Tensor
    recent: torch.Tensor

    @classmethod
    def empty(cls, pages: int, slots: int, kv_heads: int = 4, device="cuda") -> "PagedKV":
        """A cache of `pages` finished blocks and `slots` sequences (16 KB a page and head, 32 KB a slot and head)."""
        return cls(torch.empty(pages, 2, kv_heads, 8, 32, 32, dtype=torch.int8, device=device),
                   torch.empty(pages, 2, kv_heads, dtype=torch.float32, device=device),
                   torch.empty(slots, 2, kv_heads, PAGE, HEAD_DIM, dtype=torch.bfloat16, device=device))


def _cache(cache, B, lens, table, slots, dev=None):
    """Checks a cache and its index tensors; (device, heads, the C functions' arguments for them)."""
    data, scales, recent = cache
    if not data.is_cuda:
        raise ValueError("mica_amd kv_cache runs on the GPU only (got a CPU tensor)")
    dev = data.device if dev is None else dev
    P, HK = data.shape[0], data.shape[2] if data.dim() == 6 else 0
    if (data.dtype != torch.int8 or data.shape != (P, 2, HK, 8, 32, 32) or scales.dtype != torch.float32
            or scales.shape != (P, 2, HK) or recent.dtype != torch.bfloat16 or recent.dim() != 5
            or recent.shape[1:] != (2, HK, PAGE, HEAD_DIM) or HK < 1):
        raise ValueError("a cache holds data int8 [pages, 2, heads, 8, 32, 32], scales fp32 [pages, 2, heads] and recent bf16 "
                         "[slots, 2, heads, 32, 256]")
    for t in cache:
        if t.device != dev or not t.is_contiguous():
            raise ValueError("a cache's tensors must be contiguous and on the rows' device")
    if (table.dtype != torch.int32 or table.device != dev or table.dim() != 2 or table.shape[0] != B
            or (table.shape[1] > 1 and table.stride(1) != 1) or (B > 1 and table.shape[1] and table.stride(0) < table.shape[1])):
        raise ValueError("table must be an int32 [B, blocks] tensor with unit column stride on the cache's device")
    if lens is None:
        raise ValueError("lens must be a contiguous int32 [B] tensor on the cache's device")
    n = _counts(lens, B, dev, "lens")
    s = _counts(slots, B, dev, "slots")
    if not _gpu_ok(dev):
        raise RuntimeError(f"mica_amd kernels need a gfx950 GPU (device {dev})")
    width = table.shape[1]
    return dev, HK, (data.data_ptr(), scales.data_ptr(), recent.data_ptr(), P, recent.shape[0], HK, HEAD_DIM, table.data_ptr(),
                     table.stride(0) if B > 1 and width else width, width, n, s)


def append_kv(cache: PagedKV, k, v, starts, lens, table, slots=None, longest: int | None = None, rope=None, norm=None) -> PagedKV:
    """New rows into the cache (mica_kv_append): row i of sequence b becomes its token lens[b] + i.  Returns the cache; the
    caller adds the rows to lens afterwards.

    k / v [T, HK, 256]: bf16 views with unit feature stride and other strides of whole 16 bytes (e.g. of the fused QKV rows), not
    changed.  starts: int32 [B + 1], not falling; lens: int32 [B], the tokens before the call; table: int32 [B, blocks], the
    page of each block (needed for those that the call finishes); slots: int32 [B], where each sequence's unfinished block lies
    (None: b).  All on the device.  Two sequences of a call must not share a slot, nor a page that it writes.  longest: the
    longest sequence's rows where the host knows it (a hint).

    norm: (weight bf16 [256], offset, eps): each key head becomes (x / sqrt(mean(x^2) + eps)) (offset + weight).  rope: (cos,
    sin) or (cos, sin, pos): then its first 2 cos.shape[1] dims (16, 32, 64, 128 or 256) are rotated at the row's position,
    lens[b] + i or pos[t] (int32 [T]); tables bf16 or fp32 [n_pos, dims / 2], n_pos >= 1; a row whose position lies outside
    them is not rotated.  Both in fp32 and rounded to bf16 once (``fused_kernels.head_norm_rope`` rounds each step as the model's bf16
    operations do; rows that it has treated go in without these)."""
    w, offset, eps = (None, 0.0, 0.0) if norm is None else norm
    cos, sin, pos = (None, None, None) if rope is None else rope if len(rope) == 3 else (*rope, None)
    r = _lib.FAST.append_kv(*cache, k, v, starts, lens, table, slots, longest, cos, sin, pos, w, offset, eps)
    if r is not None:
        _native(r, "mica_kv_append")
        return cache
    sk, sv = _rows(k, "k"), _rows(v, "v", k.device)
    if k.shape != v.shape:
        raise ValueError("k and v must have one shape")
    B, longest = _starts(starts, k.device), _hint(longest)
    dev, HK, args = _cache(cache, B, lens, table, slots, k.device)
    T = k.shape[0]
    if k.shape[1] != HK:
        raise ValueError("k and v must have the cache's heads")
    rot_dim, code = 0, _lib.BF16
    if norm is not None:
        if w.dtype != torch.bfloat16 or w.device != dev or w.numel() != HEAD_DIM or not w.is_contiguous():
            raise ValueError("the norm weight must be a contiguous bf16 [256] tensor on the rows' device")
    if rope is not None:
        for t in (cos, sin):
            if (t.dtype not in (torch.bfloat16, torch.float32) or t.device != dev or t.dim() != 2 or not t.is_contiguous()
                    or t.shape != cos.shape or t.dtype != cos.dtype):
                raise ValueError("rope tables must be two contiguous bf16 or fp32 [n_pos, dims / 2] tensors on the rows' device")
        rot_dim, code = 2 * cos.shape[1], _lib.BF16 if cos.dtype == torch.bfloat16 else _lib.FP32
        if rot_dim not in (16, 32, 64, 128, 256):
            raise ValueError("rope tables must be for 16, 32, 64, 128 or 256 dims")
        if pos is not None and (pos.dtype != torch.int32 or pos.device != dev or pos.numel() != T or not pos.is_contiguous()):
            raise ValueError("rope positions must be a contiguous int32 [T] tensor on the rows' device")
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    L = _lib.load()
    rc = _lib.check(_on(dev, lambda: L.mica_kv_append(
        k.data_ptr(), *sk, v.data_ptr(), *sv, starts.data_ptr(), B, T, *args, ptr(w), float(offset), float(eps), rot_dim,
        ptr(cos), ptr(sin), code, 0 if cos is None else cos.shape[0], ptr(pos), longest, _stream(dev))), "mica_kv_append")
    if rc:
        raise ValueError(f"append_kv: unsupported input ({_lib.status_name(rc)})")
    _launched()
    return cache


def read_kv(cache: PagedKV, rows: int, starts, lens, table, slots=None, longest: int | None = None):
    """Rows of the cache back in bf16 (mica_kv_read): (k, v), [rows, HK, 256] each, the rows of sequence b (starts[b] ..
    starts[b + 1] - 1) being its last tokens; zeros for those before its first and for rows of no sequence.  rows: how many there
    are in all (starts[B], which the host is not to wait for); the other arguments as in append_kv, lens the tokens now."""
    r = _lib.FAST.read_kv(*cache, rows, starts, lens, table, slots, longest)
    if r is not None:
        return _native(r, "mica_kv_read")
    B, rows, longest = _starts(starts, cache[0].device), int(rows), _hint(longest)
    if not 0 <= rows < 2 ** 31:
        raise ValueError("rows must be a count of rows")
    dev, HK, args = _cache(cache, B, lens, table, slots)
    k, v = (torch.empty((rows, HK, HEAD_DIM), dtype=torch.bfloat16, device=dev) for _ in range(2))
    L = _lib.load()
    rc = _lib.check(_on(dev, lambda: L.mica_kv_read(k.data_ptr(), v.data_ptr(), starts.data_ptr(), B, rows, *args,
                                                    longest, _stream(dev))), "mica_kv_read")
    if rc:
        raise ValueError(f"read_kv: unsupported input ({_lib.status_name(rc)})")
    _launched()
    return k, v


def paged_attention(q, cache: PagedKV, starts, lens, table, slots=None, longest: int | None = None, scale: float | None = None,
                    out=None):
    """Attention of each sequence's newest rows over the cache (mica_attention_paged), which holds their keys and values already:
    row i of the n of sequence b is at position lens[b] - n + i and sees the tokens up to its own.

    q [T, HQ, 256]: a bf16 view with unit feature stride, positions applied, HQ = 4 HK.  lens: the tokens now; starts, table, slots
    as in append_kv.  longest: the longest sequence's rows, a hint (None: as if all had as many).  The result and out= as in
    ``attention.packed_attention``; a row before its sequence's first token has zeros."""
    scale = _scale(scale)
    r = _lib.FAST.paged_attention(q, *cache, starts, lens, table, slots, longest, scale, out)
    if r is not None:
        return _native(r, "mica_attention_paged")
    sq = _rows(q, "q")
    B, longest = _starts(starts, q.device), _hint(longest)
    dev, HK, args = _cache(cache, B, lens, table, slots, q.device)
    T, HQ, _ = q.shape
    if HQ != GROUP * HK:
        raise ValueError("q must have 4 heads for each of the cache's")
    L = _lib.load()
    o, so, fill = _out(out, q)
    nbytes = int(L.mica_attention_paged_workspace_bytes(B, T, HK, table.shape[1], longest))
    if nbytes < 0:
        raise ValueError("attention: invalid sizes")
    ws = torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=dev)
    rc = _lib.check(_on(dev, lambda: L.mica_attention_paged(
        q.data_ptr(), *sq, o.data_ptr(), *so, starts.data_ptr(), B, T, HQ, *args, scale, fill, longest, ws.data_ptr(), nbytes,
        _stream(dev))), "mica_attention_paged")
    if rc:
        raise ValueError(f"attention: unsupported input ({_lib.status_name(rc)})")
    _launched()
    return o
