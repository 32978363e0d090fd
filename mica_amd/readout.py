"""Last-position label readout on the gfx950 kernel: only the allowed answer rows of the output
embedding are ever multiplied, and only at each request's last token.

Reference: the readout closure built in HFJudge.__init__ (akivet/Mica
v0.5/serving/lib/release_runtime.py:298-306) applied to ``body.norm`` of the last hidden row
(prefill_engine.py:280-304), then the slice + softmax of judge_many (release_runtime.py:509-517).

``token_logprobs`` reads whole rows of logits instead: the log probabilities of given tokens, the entropy and the best
alternatives.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .int8_kernels import DT, _gpu_ok, _launched, _native, _on, _stream


class LabelReadout:
    """Readout over label rows of the output embedding.

    ``gather=True`` copies the rows once as fp32, as the reference does (release_runtime.py:301);
    ``gather=False`` keeps the bf16 table and indexes it by id inside the kernel.
    """

    def __init__(self, lm_head_weight: torch.Tensor, ids, gather: bool = True):
        ids = torch.as_tensor(ids, dtype=torch.long, device=lm_head_weight.device)
        self.n_labels = int(ids.numel())
        if gather:
            self.weight = lm_head_weight.detach().index_select(0, ids).float().contiguous()
            self.ids = None
        else:
            if lm_head_weight.dtype != torch.bfloat16:
                raise ValueError("an un-gathered table must be bf16")
            self.weight = lm_head_weight.detach().contiguous()
            self.ids = ids.to(torch.int32).contiguous()

    def __call__(self, h, rows, norm_weight=None, eps=1e-6, offset=1.0, lo=None, cnt=None, probs_width=None):
        """h: [T, K] bf16 hidden states (packed requests); rows: int [B] index of each request's last
        token; norm_weight: the final RMSNorm weight or None (h already normed).
        lo / cnt: int [B] start and length of each request's softmax slice (None: all labels).
        Returns (logits fp32 [B, L], probs fp32 [B, width])."""
        if not h.is_cuda:
            raise ValueError("mica_amd readout runs on the GPU only (got a CPU tensor)")
        if h.dtype != torch.bfloat16 or h.dim() != 2 or h.stride(1) != 1:
            raise ValueError("h must be a 2-D bf16 tensor with unit feature stride")
        dev = h.device
        if not _gpu_ok(dev):
            raise RuntimeError(f"mica_amd kernels need a gfx950 GPU (device {dev})")
        K = h.shape[1]
        rows = torch.as_tensor(rows, device=dev).to(torch.int32).contiguous()
        B = rows.numel()
        L = self.n_labels
        logits = torch.empty((B, L), dtype=torch.float32, device=dev)
        if lo is not None:
            if probs_width is None:
                # the width is read from host values only: a device tensor would need a synchronising
                # read, which stalls the stream and cannot be captured in a HIP graph
                if isinstance(cnt, torch.Tensor) and cnt.is_cuda:
                    raise ValueError("give probs_width when cnt is a device tensor")
                host = torch.as_tensor(cnt, dtype=torch.int64)
                probs_width = int(host.max()) if host.numel() else 0
            lo = torch.as_tensor(lo, device=dev).to(torch.int32).contiguous()
            cnt = torch.as_tensor(cnt, device=dev).to(torch.int32).contiguous()
            width = probs_width if B else 0
        else:
            width = L
        probs = torch.zeros((B, max(width, 1)), dtype=torch.float32, device=dev)
        nw = None if norm_weight is None else norm_weight.contiguous()
        lib = _lib.load()
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        wdt = _lib.FP32 if self.weight.dtype == torch.float32 else _lib.BF16
        rc = _lib.check(_on(dev, lambda: lib.mica_gather_logits(
            h.data_ptr(), h.stride(0), h.shape[0], rows.data_ptr(), B, ptr(nw),
            DT[nw.dtype] if nw is not None else 0, float(offset), float(eps), self.weight.data_ptr(), wdt,
            self.weight.stride(0), self.weight.shape[0], ptr(self.ids), L, K, logits.data_ptr(), ptr(lo), ptr(cnt),
            probs.data_ptr(), probs.shape[1], _stream(dev))), "mica_gather_logits")
        if rc > 0:
            raise ValueError(f"readout does not support this input ({_lib.status_name(rc)})")
        _launched()
        return logits, probs


def gather_logits(h, last_idx, norm_w, eps, label_W, n_opts, offset=1.0):
    """The readout as one function: the final RMSNorm of h at each request's last token (rows
    last_idx of the packed [T, K] bf16 h), fp32 dots with the label rows label_W ([L, K] fp32 or bf16:
    No, Yes, then the option labels, as gathered by release_runtime.py:298-302), and the softmax of
    each request's slice (release_runtime.py:509-517): n_opts[b] == 0 reads the No / Yes pair, n > 0
    the first n option labels.  n_opts is one int for every request or one per request.  Returns the
    probabilities, fp32 [B, max slice] (zero past each request's slice); one kernel launch pair."""
    if label_W.dtype not in (torch.float32, torch.bfloat16) or label_W.dim() != 2:
        raise ValueError("label_W must be a 2-D fp32 or bf16 tensor")
    ro = LabelReadout.__new__(LabelReadout)
    ro.weight, ro.ids, ro.n_labels = label_W.contiguous(), None, int(label_W.shape[0])
    B = int(torch.as_tensor(last_idx).numel())
    ns = [int(n_opts)] * B if isinstance(n_opts, int) else [int(n) for n in n_opts]
    if len(ns) != B or any(n < 0 or n > ro.n_labels - 2 for n in ns):
        raise ValueError("n_opts must give 0 (No / Yes) or 1 .. L - 2 options for every request")
    lo = torch.tensor([0 if n == 0 else 2 for n in ns], dtype=torch.int32)
    cnt = [2 if n == 0 else n for n in ns]
    _, probs = ro(h, last_idx, norm_w, eps, offset, lo=lo, cnt=torch.tensor(cnt, dtype=torch.int32),
                  probs_width=max(cnt) if cnt else 0)
    return probs


MAX_TOP = 32     # alternatives of token_logprobs


class TokenLogprobs(NamedTuple):
    """token_logprobs' results: fp32 of the tokens' shape, fp32 [T], int64 [T, top], fp32 [T, top]."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def token_logprobs(logits, tokens, top: int = 0) -> TokenLogprobs:
    """Log probabilities of given tokens under rows of logits, each row's entropy (nats) and its `top` most probable
    tokens, in one pass over the logits (mica_token_logprobs).

    logits: [T, V] bf16 / fp16 / fp32 with unit column stride (a view of wider rows will do), e.g. a full-vocabulary
    head's output.  tokens: int32 or int64, one token for each row [T] or several [T, C]; an id outside 0 .. V - 1 gives
    NaN.  top: 0 .. 32 alternatives, equal logits by the lower id.  A logit of -inf has probability 0; a row with a NaN or
    +inf logit, or with -inf only, gives NaN."""
    r = _lib.FAST.token_logprobs(logits, tokens, top)
    if r is not None:
        return TokenLogprobs._make(_native(r, "mica_token_logprobs"))
    if not logits.is_cuda:
        raise ValueError("mica_amd readout runs on the GPU only (got a CPU tensor)")
    if logits.dim() != 2 or logits.dtype not in DT or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be a 2-D bf16, fp16 or fp32 tensor with unit column stride")
    dev = logits.device
    T, V = logits.shape
    if (tokens.device != dev or tokens.dtype not in (torch.int32, torch.int64) or tokens.dim() not in (1, 2)
            or tokens.shape[0] != T):
        raise ValueError("tokens must be an int32 or int64 [T] or [T, C] tensor on the logits' device")
    top = int(top)
    if V < 1 or not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top must be 0 .. {MAX_TOP} and at most the vocabulary")
    if not _gpu_ok(dev):
        raise RuntimeError(f"mica_amd kernels need a gfx950 GPU (device {dev})")
    tokens = tokens.contiguous()
    C = 1 if tokens.dim() == 1 else tokens.shape[1]
    out = TokenLogprobs(torch.empty(tokens.shape, dtype=torch.float32, device=dev),
                        torch.empty(T, dtype=torch.float32, device=dev),
                        torch.empty((T, top), dtype=torch.int64, device=dev),
                        torch.empty((T, top), dtype=torch.float32, device=dev))
    lib = _lib.load()
    nbytes = int(lib.mica_token_logprobs_workspace_bytes(T, V, DT[logits.dtype], top))
    ws = torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=dev)
    rc = _lib.check(_on(dev, lambda: lib.mica_token_logprobs(
        logits.data_ptr(), DT[logits.dtype], logits.stride(0) if T > 1 else V, T, V, tokens.data_ptr(),
        int(tokens.dtype == torch.int64), C, top, *(t.data_ptr() for t in out), ws.data_ptr(), nbytes, _stream(dev))),
        "mica_token_logprobs")
    if rc > 0:
        raise ValueError(f"token_logprobs does not support this input ({_lib.status_name(rc)})")
    _launched()
    return out
