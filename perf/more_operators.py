"""Cases of four operators that a server of many states and questions needs beside the padded prefill path:

  packed   attention.packed_attention    causal attention over prompts of different lengths, packed one behind the other
  append   kv_cache.append_kv            keys and values into a paged 8-bit cache, normed and rotated on the way
  paged    kv_cache.paged_attention      the newest rows of each sequence over that cache: a single token, drafts, questions
  read     kv_cache.read_kv              rows of the cache back in bf16

The cache keeps blocks of 32 tokens in int8 with one scale for each block, head and side (keys, values); the block that a
sequence has not filled yet stays in bf16.  ``run`` computes the operators in plain torch, in float32, or with ``own`` set
through the package.  The head layout is that of the 4B configuration (16 query and 4 key/value heads of 256), its rotation
over the first 64 dims; other sizes are generic.
"""
import math

import torch

own = False

DEV = "cuda"
HD, PAGE, GROUP = 256, 32, 4
ROT, EPS = 64, 1e-6
TOP = 16384          # most rows of a packed case


def listed():
    return [
        # one short request: where only latency counts
        dict(name="packed_one", kind="packed", heads=4, count=1, longest=77, ragged=False),
        # a batch of requests as they come, odd lengths from a few tokens to a state's
        dict(name="packed_batch", kind="packed", heads=4, count=13, longest=2047, ragged=True),
        # long states and what fits beside them: the largest
        dict(name="packed_long", kind="packed", heads=4, count=2, longest=10922, ragged=True),
        # one new token of each of 64 requests
        dict(name="append_step", kind="append", heads=4, count=64, longest=1, ragged=False, before=4099, fresh=False),
        # the prompts of a packed batch into an empty cache
        dict(name="append_prompts", kind="append", heads=4, count=15, longest=2047, ragged=True, before=0, fresh=True),
        # the next token of one request
        dict(name="paged_one", kind="paged", heads=4, count=1, rows=1, mixed=False, keys=500, ragged=False, shared=0),
        # the next token of each of 64 requests with caches of different lengths
        dict(name="paged_step", kind="paged", heads=4, count=64, rows=1, mixed=False, keys=8192, ragged=True, shared=0),
        # a few drafted tokens of each of 32 requests
        dict(name="paged_drafts", kind="paged", heads=4, count=32, rows=16, mixed=True, keys=4096, ragged=True, shared=0),
        # eight questions of different lengths about one state, whose pages they share
        dict(name="paged_questions", kind="paged", heads=4, count=8, rows=240, mixed=True, keys=7152, ragged=False, shared=6912),
        # a long prompt's next piece
        dict(name="paged_piece", kind="paged", heads=4, count=1, rows=2048, mixed=False, keys=18001, ragged=False, shared=0),
        # a short header back in bf16
        dict(name="read_header", kind="read", heads=4, count=1, rows=320, keys=320, ragged=False),
        # the states of a batch
        dict(name="read_states", kind="read", heads=4, count=9, rows=8001, keys=8001, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind, heads = rng.choice(("packed", "append", "paged", "paged", "read")), rng.choice((1, 2, 4, 4, 4))
    ragged = rng.random() < 0.6
    if kind == "packed":
        count = _log(rng, 1, 200)
        return dict(kind=kind, heads=heads, count=count, longest=_log(rng, 1, min(10922, TOP // count)), ragged=ragged)
    if kind == "append":
        fresh = rng.random() < 0.5
        count = _log(rng, 1, 200)
        longest = _log(rng, 1, min(8192, 16376 // count)) if fresh else rng.choice((1, rng.randint(1, 16)))
        return dict(kind=kind, heads=heads, count=count, longest=longest, ragged=ragged,
                    before=32 * rng.randint(0, 40) if fresh else _log(rng, 1, 9000), fresh=fresh)
    if kind == "read":
        count = _log(rng, 1, 64)
        keys = _log(rng, 1, min(16384, 40000 // count))
        return dict(kind=kind, heads=heads, count=count, rows=rng.choice((keys, rng.randint(1, keys))), keys=keys, ragged=ragged)
    count, rows = _log(rng, 1, 64), rng.choice((1, _log(rng, 1, 64), _log(rng, 1, 2048)))
    keys = _log(rng, rows, 32768)
    while count * keys > 64 * 8192 or count * rows * keys > 2048 * 18001:
        count, keys = max(1, count - 1), max(rows, keys * 3 // 4)
    shared = rng.choice((0, 0, max(0, keys - rows) // PAGE * PAGE))
    return dict(kind=kind, heads=heads, count=count, rows=rows, mixed=rng.random() < 0.6, keys=keys,
                ragged=ragged and not shared, shared=shared)


# ------------------------------------------------------------------------------------------------ inputs
def _falling(count, longest, ragged):
    """`count` lengths, equal or falling from the longest to a `count`-th of it, the long and the short ones mixed."""
    lens = [max(1, longest - (longest * b // count if ragged else 0)) for b in range(count)]
    return lens[::2] + lens[1::2][::-1]


def _counts(case):
    """(rows of each sequence in the call, tokens of each in the cache: before an append, otherwise at the call)."""
    if case["kind"] in ("packed", "append"):
        new = _falling(case["count"], case["longest"], case["ragged"])
        if case["kind"] == "packed":
            return new, [0] * len(new)
        old = []
        for b, n in enumerate(new):
            p = case["before"] if case["fresh"] else case["before"] + 5 * b
            if not case["fresh"] and p % PAGE + n > PAGE:     # a block is finished with its last new token, or not at all
                p += PAGE - (p + n) % PAGE
            old.append(p)
        return new, old
    keys = _falling(case["count"], case["keys"], case["ragged"])
    rows = _falling(case["count"], case["rows"], case.get("mixed", case["ragged"]))
    return [min(r, n) for r, n in zip(rows, keys)], keys


def _starts(counts):
    return torch.tensor([0] + counts, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    HK = case["heads"]
    HQ = GROUP * HK
    new, held = _counts(case)
    T, B = sum(new), len(new)
    st = dict(case=case, starts=_starts(new), longest=max(new), rows=T)
    if case["kind"] != "read":
        # the rows' heads as a fused projection leaves them
        st["q"], st["k"], st["v"] = rn(T, HQ + 2 * HK, HD).split((HQ, HK, HK), dim=1)
    if case["kind"] == "packed":
        st["seq"] = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(new, device=DEV))
        return st
    # the cache: finished blocks in pages of any order, shared ones first; a row of the table for each sequence
    after = [h + n for h, n in zip(held, new)] if case["kind"] == "append" else held
    first, full = case.get("shared", 0) // PAGE, [n // PAGE for n in after]
    width = max(max(full), 1)
    total = first + sum(max(0, f - first) for f in full)
    order = torch.randperm(total + 3, generator=g, device=DEV).cpu()
    table, at = torch.full((B, width), -1, dtype=torch.int32), first
    for b, f in enumerate(full):
        table[b, :min(first, f)] = order[:min(first, f)]
        table[b, first:max(first, f)] = order[at:at + max(0, f - first)]
        at += max(0, f - first)
    P = total + 3
    # values as a quantizer of unit normals leaves them
    st["data"] = (torch.randn(P, 2, HK, 8, 32, 32, generator=g, device=DEV) * 31).round_().clamp_(-127, 127).to(torch.int8)
    st["scales"] = (0.7 + 0.6 * torch.rand(P, 2, HK, generator=g, device=DEV)) / 31
    st["recent"] = rn(B, 2, HK, PAGE, HD)
    st["table"] = table.to(DEV)
    st["lens"] = torch.tensor(held, dtype=torch.int32, device=DEV)
    if case["kind"] == "append":
        ang = torch.arange(max(after), device=DEV, dtype=torch.float64)[:, None]
        ang = ang * 1e7 ** (-torch.arange(0, ROT, 2, device=DEV, dtype=torch.float64) / ROT)
        st["cos"], st["sin"] = ang.cos().to(torch.bfloat16), ang.sin().to(torch.bfloat16)
        st["weight"] = (torch.randn(HD, generator=g, device=DEV) * 0.1).to(torch.bfloat16)
        # what is read back: every row of the blocks that the append touches
        back = [h % PAGE + n for h, n in zip(held, new)]
        st["back"], st["back_rows"], st["back_longest"] = _starts(back), sum(back), max(back)
        st["after"] = torch.tensor(after, dtype=torch.int32, device=DEV)
    return st


# --------------------------------------------------------------------------------------------- plain forms
def _owner(starts, rows):
    """The sequence and the index within it of each of `rows` packed rows."""
    at = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), at.to(torch.int32), right=True)
    return seq, at - starts[seq]


def _packed(st):
    q, k, v, seq = st["q"].float(), st["k"].float(), st["v"].float(), st["seq"]
    T, HQ, HK = q.shape[0], q.shape[1], k.shape[1]
    at = torch.arange(T, device=DEV)
    hidden = (seq[:, None] != seq[None]) | (at[None] > at[:, None])
    z = torch.matmul(q.view(T, HK, GROUP, HD).permute(1, 2, 0, 3).reshape(HK, GROUP * T, HD), k.permute(1, 2, 0).contiguous())
    z = z.view(HK, GROUP, T, T)
    z /= math.sqrt(HD)
    z.masked_fill_(hidden, -math.inf)
    z -= z.amax(-1, keepdim=True)
    z.exp_()
    z /= z.sum(-1, keepdim=True)
    o = torch.matmul(z.view(HK, GROUP * T, T), v.transpose(0, 1).contiguous())
    return o.view(HQ, T, HD).transpose(0, 1).to(torch.bfloat16)


def _values(st):
    """The finished blocks of every sequence, [B, blocks, 2, heads, 32, 256] in float32 (a page of the table's -1: the last)."""
    pages = st["table"].long()
    x = st["data"][pages].float() * st["scales"][pages][..., None, None, None]
    B, M, _, HK = x.shape[:4]
    k = x[:, :, 0].transpose(3, 4).reshape(B, M, HK, PAGE, HD)                   # [8, 32 tokens, 32 dims]
    v = x[:, :, 1].reshape(B, M, HK, HD, 2, 2, 2, 4)                             # [256 dims, fours of tokens in bit-reversed order]
    v = v.permute(0, 1, 2, 6, 5, 4, 7, 3).reshape(B, M, HK, PAGE, HD)
    return torch.stack((k, v), 2)


def _cached(st):
    """Keys and values of every sequence, two [B, 32 (blocks + 1), heads, 256], from position 0 on."""
    x = _values(st)
    B, M, _, HK = x.shape[:4]
    x = torch.cat((x, x[:, :1]), 1)
    x[torch.arange(B, device=DEV), (st["lens"] // PAGE).long()] = st["recent"].float()
    x = x.permute(2, 0, 1, 4, 3, 5).reshape(2, B, (M + 1) * PAGE, HK, HD)
    return x[0], x[1]


def _paged(st):
    k, v = _cached(st)
    B, S, HK = k.shape[:3]
    n, T, HQ = st["longest"], st["rows"], st["q"].shape[1]
    seq, i = _owner(st["starts"], T)
    q = torch.zeros(B, n, HQ, HD, device=DEV)
    q[seq, i] = st["q"].float()
    count = st["starts"][1:] - st["starts"][:-1]
    at = (st["lens"] - count)[:, None] + torch.arange(n, device=DEV)[None]
    sees = torch.arange(S, device=DEV)[None, None] <= at[:, :, None]
    q = q.view(B, n, HK, GROUP, HD).permute(0, 2, 3, 1, 4).reshape(B, HK, GROUP * n, HD)
    z = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(B, HK, GROUP, n, S)
    z /= math.sqrt(HD)
    z.masked_fill_(~sees[:, None, None], -math.inf)
    z -= z.amax(-1, keepdim=True)
    z.exp_()
    z /= z.sum(-1, keepdim=True)
    o = torch.matmul(z.view(B, HK, GROUP * n, S), v.transpose(1, 2).contiguous())
    return o.view(B, HQ, n, HD).transpose(1, 2)[seq, i].to(torch.bfloat16)


def _read(st):
    k, v = _cached(st)
    seq, i = _owner(st["starts"], st["rows"])
    at = (st["lens"] - (st["starts"][1:] - st["starts"][:-1]))[seq] + i
    return k[seq, at].to(torch.bfloat16), v[seq, at].to(torch.bfloat16)


def _append(st):
    """The rows of the touched blocks as the cache then holds them."""
    T, HK = st["k"].shape[:2]
    seq, i = _owner(st["starts"], T)
    pos = st["lens"][seq] + i
    k = st["k"].float()
    k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * (1.0 + st["weight"].float())
    c, s = st["cos"][pos].float()[:, None], st["sin"][pos].float()[:, None]
    a, b = k[..., :ROT // 2], k[..., ROT // 2:ROT]
    k = torch.cat((a * c - b * s, b * c + a * s, k[..., ROT:]), -1).to(torch.bfloat16)
    seq2, j = _owner(st["back"], st["back_rows"])
    rest = (st["lens"] % PAGE)[seq2]                                # rows that were there already
    src = (st["starts"][seq2] + j - rest).clamp(min=0)
    x = torch.stack((k, st["v"]))[:, src]
    held = st["recent"].permute(1, 0, 3, 2, 4)[:, seq2, j.clamp(max=PAGE - 1)]
    x = torch.where((j < rest)[None, :, None, None], held, x).float()
    # a scale for each block, head and side of those that are full now
    width = (st["back_longest"] + PAGE - 1) // PAGE
    block = seq2 * width + j // PAGE
    top = torch.zeros(2, st["table"].shape[0] * width, HK, device=DEV)
    top.scatter_reduce_(1, block[None, :, None].expand(2, -1, HK), x.abs().amax(-1), "amax")
    scale = (top.clamp(min=1e-8) / 127.0)[:, block][..., None]
    full = (j // PAGE + 1) * PAGE <= (st["back"][1:] - st["back"][:-1])[seq2]
    x = torch.where(full[None, :, None, None], torch.round(x / scale).clamp(-127, 127) * scale, x).to(torch.bfloat16)
    return x[0], x[1]


def run(state):
    kind = state["case"]["kind"]
    if own:
        from mica_amd import attention, kv_cache
        st = state
        if kind == "packed":
            return attention.packed_attention(st["q"], st["k"], st["v"], st["starts"], longest=st["longest"])
        cache = kv_cache.PagedKV(st["data"], st["scales"], st["recent"])
        if kind == "paged":
            return kv_cache.paged_attention(st["q"], cache, st["starts"], st["lens"], st["table"], longest=st["longest"])
        if kind == "read":
            return kv_cache.read_kv(cache, st["rows"], st["starts"], st["lens"], st["table"], longest=st["longest"])
        kv_cache.append_kv(cache, st["k"], st["v"], st["starts"], st["lens"], st["table"], longest=st["longest"],
                           rope=(st["cos"], st["sin"]), norm=(st["weight"], 1.0, EPS))
        return kv_cache.read_kv(cache, st["back_rows"], st["back"], st["after"], st["table"], longest=st["back_longest"])
    return {"packed": _packed, "append": _append, "paged": _paged, "read": _read}[kind](state)


# --------------------------------------------------------------------------------------------------- work
def _stored(keys):
    """Bytes of a head's keys and values in the cache."""
    return 2 * (keys // PAGE * (PAGE * HD + 4) + keys % PAGE * HD * 2)


def work(case):
    new, held = _counts(case)
    HK, T = case["heads"], sum(new)
    HQ, row = GROUP * HK, 2 * HD                 # bytes of a head's bf16 row
    if case["kind"] == "packed":
        return dict(bytes=row * 2 * (HQ + HK) * T, flops=4 * HQ * HD * sum(n * (n + 1) // 2 for n in new))
    if case["kind"] == "paged":
        shared = case["shared"]
        return dict(bytes=row * 2 * HQ * T + HK * (_stored(shared) + sum(_stored(n) - _stored(shared) for n in held)),
                    flops=4 * HQ * HD * sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, held)))
    if case["kind"] == "read":
        return dict(bytes=HK * (2 * row * T + sum(_stored(m) - _stored((m - n) // PAGE * PAGE) for n, m in zip(new, held))), flops=0)
    # in: the new rows and those that wait; out: what is stored; then what is stored in and the touched blocks' rows out
    back = sum(h % PAGE + n for h, n in zip(held, new))
    kept = sum(_stored(h % PAGE + n) for h, n in zip(held, new))
    waits = sum(h % PAGE for h, n in zip(held, new) if h % PAGE + n >= PAGE)
    return dict(bytes=HK * (2 * row * (T + waits + back) + 2 * kept), flops=12 * HK * HD * T)


# ------------------------------------------------------------------------------------ 64-bit evaluation
def _exact_head(q, k, v, first):
    """Attention of one head in float64: q [n, HD] at positions first, first + 1, ...; k / v [S, HD]."""
    z = q @ k.t() * HD ** -0.5
    at = first + torch.arange(q.shape[0], device=DEV)
    z.masked_fill_(torch.arange(k.shape[0], device=DEV)[None] > at[:, None], -math.inf)
    w = torch.exp(z - z.max(1, keepdim=True).values)
    return (w @ v) / w.sum(1, keepdim=True)


def _exact_rows(st, b, first, last):
    """Positions first .. last - 1 of sequence b as the cache holds them, float64 [2, heads, rows, HD]."""
    out, n = [], int(st["lens"][b])
    token = torch.arange(PAGE, device=DEV)
    byte = 4 * torch.tensor([0, 4, 2, 6, 1, 5, 3, 7], device=DEV)[token // 4] + token % 4       # where a token's value lies
    for block in range(first // PAGE, -(-last // PAGE)):
        if block < n // PAGE:
            page = int(st["table"][b, block])
            x = st["data"][page].double()
            k = x[0].permute(0, 2, 1, 3).reshape(x.shape[1], PAGE, HD)
            v = x[1][..., byte].reshape(x.shape[1], HD, PAGE).transpose(1, 2)
            out.append(torch.stack((k, v)) * st["scales"][page].double()[..., None, None])
        else:
            out.append(st["recent"][b].double())
    at = first // PAGE * PAGE
    return torch.cat(out, 2)[:, :, first - at:last - at]


def exact(case, seed):
    st = prepare(case, seed)
    new, held = _counts(case)
    HK = case["heads"]
    if case["kind"] in ("packed", "paged"):
        out, lo = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV), 0
        for b, n in enumerate(new):
            if case["kind"] == "packed":
                k, v = (st[x][lo:lo + n].double().transpose(0, 1) for x in "kv")
            else:
                k, v = _exact_rows(st, b, 0, held[b])
            for h in range(GROUP * HK):
                out[lo:lo + n, h] = _exact_head(st["q"][lo:lo + n, h].double(), k[h // GROUP], v[h // GROUP], k.shape[1] - n)
            lo += n
        return out
    if case["kind"] == "read":
        x = torch.cat([_exact_rows(st, b, m - n, m) for b, (n, m) in enumerate(zip(new, held))], 2).transpose(1, 2)
        return x[0], x[1]
    rows, lo = [], 0
    for b, (n, h) in enumerate(zip(new, held)):
        k, v = st["k"][lo:lo + n].double(), st["v"][lo:lo + n].double()
        k = k * (k.square().mean(-1, keepdim=True) + EPS).rsqrt() * (1.0 + st["weight"].double())
        turn = torch.complex(st["cos"][h:h + n].double(), st["sin"][h:h + n].double())[:, None]
        pairs = torch.complex(k[..., :ROT // 2], k[..., ROT // 2:ROT]) * turn
        k = torch.cat((pairs.real, pairs.imag, k[..., ROT:]), -1).to(torch.bfloat16).double()      # the rows' type, before any block
        x = torch.cat((st["recent"][b, :, :, :h % PAGE].double(), torch.stack((k, v)).transpose(1, 2)), 2)
        for j in range(0, x.shape[2] // PAGE * PAGE, PAGE):
            y = x[:, :, j:j + PAGE]
            s = y.abs().amax((2, 3), keepdim=True).clamp(min=1e-8) / 127
            x[:, :, j:j + PAGE] = torch.round(y / s) * s
        rows.append(x)
        lo += n
    x = torch.cat(rows, 2).transpose(1, 2)
    return x[0], x[1]
