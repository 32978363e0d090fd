"""Cases of three operators that a scorer of candidate answers needs beside the prefill path:

  logprobs   readout.token_logprobs      log probabilities of given tokens, entropy and top alternatives of logit rows
  tree       attention.tree_attention    a tree of candidate tokens that attends to its ancestors and to cached keys
  window     attention.window_attention  causal attention within a sliding window and over a few first tokens (sinks)

``run`` computes them in plain torch, in float32, or with ``own`` set through the package.  The head layout is that of
the 4B configuration (16 query and 4 key/value heads of 256), the vocabulary its 151936; other sizes are generic.
"""
import math

import torch

own = False

DEV = "cuda"
HQ, HK, HD = 16, 4, 256
VOCAB = 151936
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the next token of one request: where only latency counts
        dict(name="lp_next_token", kind="logprobs", rows=1, vocab=VOCAB, dtype="bf16", top=5, given=1, pad=0, masked=False),
        # eight candidate tokens at each of 64 positions, fp32 logits of a W8A8 head
        dict(name="lp_candidates", kind="logprobs", rows=64, vocab=VOCAB, dtype="fp32", top=20, given=8, pad=0, masked=False),
        # odd everything: rows of a padded table, part of the vocabulary ruled out, fp16
        dict(name="lp_odd", kind="logprobs", rows=517, vocab=32003, dtype="fp16", top=7, given=1, pad=61, masked=True),
        # every token of a prompt with its alternatives
        dict(name="lp_prompt_top", kind="logprobs", rows=2048, vocab=VOCAB, dtype="bf16", top=20, given=1, pad=0, masked=False),
        # every token of a packed batch, without alternatives: the largest
        dict(name="lp_packed", kind="logprobs", rows=4096, vocab=VOCAB, dtype="bf16", top=0, given=1, pad=0, masked=False),
        # a handful of candidates after a short prompt
        dict(name="tree_short", kind="tree", batch=1, nodes=8, cache=500, ragged=False, shared=False, roots=1, branch=2),
        # a draft of 64 tokens after one long state
        dict(name="tree_long", kind="tree", batch=1, nodes=64, cache=32768, ragged=False, shared=False, roots=1, branch=3),
        # drafts of many requests with caches of different lengths
        dict(name="tree_batch", kind="tree", batch=32, nodes=16, cache=4096, ragged=True, shared=False, roots=2, branch=1),
        # every option of four questions about one state, whose cache they share
        dict(name="tree_options", kind="tree", batch=4, nodes=255, cache=2048, ragged=False, shared=True, roots=100, branch=1),
        # one new token of each of 64 requests
        dict(name="win_step", kind="window", batch=64, queries=1, keys=8192, window=4096, sinks=4, ragged=True),
        # a small batch of odd prompts
        dict(name="win_odd", kind="window", batch=3, queries=1111, keys=1111, window=200, sinks=5, ragged=False),
        # a long state
        dict(name="win_long", kind="window", batch=1, queries=16384, keys=16384, window=2048, sinks=4, ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("logprobs", "tree", "window"))
    if kind == "logprobs":
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        vocab = rng.choice((VOCAB, _log(rng, 300, 200000)))
        rows = _log(rng, 1, min(8192, 4096 * VOCAB * 2 // (vocab * SIZES[dtype])))
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, top=rng.choice((0, rng.randint(1, 20))),
                    given=rng.choice((1, rng.randint(2, 40))), pad=rng.choice((0, rng.randint(1, 64))),
                    masked=rng.random() < 0.3)
    if kind == "tree":
        batch, nodes = _log(rng, 1, 48), _log(rng, 1, 255)
        cache = rng.choice((0, _log(rng, 1, 32768), _log(rng, 1, 32768), _log(rng, 1, 32768)))
        while batch * nodes * (cache + nodes) > 4 * 255 * 2304 or batch * cache > 32 * 4096:
            batch, cache = max(1, batch - 1), cache * 3 // 4
        return dict(kind=kind, batch=batch, nodes=nodes, cache=cache, ragged=rng.random() < 0.5,
                    shared=rng.random() < 0.3, roots=rng.randint(1, 4), branch=rng.randint(1, 4))
    batch, window, sinks = _log(rng, 1, 64), _log(rng, 1, 8192), rng.choice((0, rng.randint(1, 40)))
    queries = rng.choice((1, _log(rng, 1, 16384)))
    keys = queries if rng.random() < 0.5 else queries + _log(rng, 1, 16384)
    while batch * queries * min(keys, window + sinks) > 16384 * 2052 or batch * keys > 64 * 8192 or \
            batch * queries * keys > 16384 * 16384:
        batch, queries, keys = max(1, batch - 2), max(1, queries * 3 // 4), max(1, keys * 3 // 4)
    return dict(kind=kind, batch=batch, queries=queries, keys=max(keys, queries), window=window, sinks=sinks,
                ragged=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case, longest):
    """Key counts of a batch: equal, or from the longest down to half of it."""
    B = case["batch"]
    return [longest - (longest * b // (2 * B) if case["ragged"] else 0) for b in range(B)]


def _parents(case):
    """`roots` nodes that follow the cache, every later node the child of an earlier one, `branch` children each."""
    return [-1 if i < case["roots"] else (i - case["roots"]) // case["branch"] for i in range(case["nodes"])]


def _ancestors(case):
    """Boolean [N, N]: node i sees node j (itself and its ancestors)."""
    sees, par = torch.eye(case["nodes"], dtype=torch.bool), _parents(case)
    for i, p in enumerate(par):
        if p >= 0:
            sees[i] |= sees[p]
    return sees


def _words(sees):
    """The rows of a boolean [N, N] as int64 words, 64 nodes a word, the lowest bit first."""
    n = sees.shape[0]
    bits = torch.zeros(n, -(-n // 64) * 64, dtype=torch.int64)
    bits[:, :n] = sees
    return (bits.view(n, -1, 64) << torch.arange(64)).sum(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    st = dict(case=case)
    if case["kind"] == "logprobs":
        T, V = case["rows"], case["vocab"]
        table = torch.empty(T, V + case["pad"], device=DEV, dtype=DTYPES[case["dtype"]])
        for lo in range(0, T, 1024):
            table[lo:lo + 1024] = torch.randn(min(1024, T - lo), V + case["pad"], generator=g, device=DEV) * 2.5
        logits = table[:, :V]
        if case["masked"]:                 # a grammar or a stop list rules a tenth of the vocabulary out
            logits[:, torch.randperm(V, generator=g, device=DEV)[:V // 10]] = -math.inf
        shape = (T,) if case["given"] == 1 else (T, case["given"])
        st.update(logits=logits, tokens=torch.randint(0, V, shape, generator=g, device=DEV))
        return st
    B = case["batch"]
    n = case["nodes"] if case["kind"] == "tree" else case["queries"]
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    if case["kind"] == "tree":
        # the new tokens' heads as a fused QKV projection leaves them, the cache as a prefix is kept
        st["q"], st["k"], st["v"] = rn(B, n, HQ + 2 * HK, HD).split((HQ, HK, HK), dim=2)
        C = case["cache"]
        rows = 1 if case["shared"] else B
        st["cache"] = tuple(rn(rows, C, HK, HD).expand(B, -1, -1, -1) for _ in range(2))
        st["sees"] = _ancestors(case).to(DEV)
        st["tree"] = _words(_ancestors(case)).to(DEV)
        st["lens"] = torch.tensor(_lengths(case, C), dtype=torch.int32, device=DEV)
        return st
    st["q"] = rn(B, n, HQ, HD)
    st["k"], st["v"] = rn(B, case["keys"], 2 * HK, HD).split((HK, HK), dim=2)
    st["lens"] = torch.tensor(_lengths(case, case["keys"]), dtype=torch.int32, device=DEV) if case["ragged"] else None
    return st


# --------------------------------------------------------------------------------------------- plain forms
def _logprobs(x, tokens, top):
    x = x.float()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True)
    norm = m + torch.log(s)
    entropy = norm - (torch.where(e > 0, e * x, 0.0).sum(1, keepdim=True) / s)
    got = x.gather(1, tokens.view(x.shape[0], -1)) - norm
    # ordered by the value, then by the lowest index: the value's bits as a whole number above the index's
    bits = (x + 0.0).view(torch.int32).long()
    key = (torch.where(bits < 0, -(bits & 0x7fffffff), bits) << 32) - torch.arange(x.shape[1], device=x.device)
    ids = -(key.topk(top, 1).values << 32 >> 32) if top else key[:, :0]
    return got.view(tokens.shape), entropy[:, 0], ids, x.gather(1, ids) - norm


def _attend(q, k, v, sees):
    """q [B, n, HQ, HD], k / v [B, S, HK, HD], sees [B or 1, n, S]: zeros for a query that sees no key."""
    B, n, S = q.shape[0], q.shape[1], k.shape[1]
    q = q.float().view(B, n, HK, HQ // HK, HD).permute(0, 2, 3, 1, 4).reshape(B, HK, HQ // HK * n, HD)
    k = k.float().permute(0, 2, 3, 1).contiguous()
    v = v.float().permute(0, 2, 1, 3).contiguous()
    z = (torch.matmul(q, k) / math.sqrt(HD)).view(B, HK, HQ // HK, n, S)
    z.masked_fill_(~sees[:, None, None], -math.inf)
    z -= z.amax(-1, keepdim=True).clamp_min(-3e38)
    z = z.exp_()
    s = z.sum(-1, keepdim=True)
    z /= torch.where(s > 0, s, 1.0)
    o = torch.matmul(z.view(B, HK, HQ // HK * n, S), v)
    return o.view(B, HQ, n, HD).transpose(1, 2)


def _tree_sees(st, case):
    B, C, n = case["batch"], case["cache"], case["nodes"]
    old = torch.arange(C, device=DEV)[None, None] < st["lens"][:, None, None]
    return torch.cat((old.expand(B, n, C), st["sees"][None].expand(B, n, n)), 2)


def _window_sees(st, case):
    lens = torch.tensor([case["keys"]], device=DEV) if st["lens"] is None else st["lens"]
    at = lens[:, None] - case["queries"] + torch.arange(case["queries"], device=DEV)[None]      # query positions
    at, key = at[:, :, None], torch.arange(case["keys"], device=DEV)[None, None]
    return (key <= at) & ((key > at - case["window"]) | (key < case["sinks"]))


def run(state):
    case = state["case"]
    if own:
        from mica_amd import attention, readout
        if case["kind"] == "logprobs":
            return tuple(readout.token_logprobs(state["logits"], state["tokens"], top=case["top"]))
        if case["kind"] == "tree":
            return attention.tree_attention(state["q"], state["k"], state["v"], state["tree"], cache=state["cache"],
                                            cache_len=state["lens"])
        return attention.window_attention(state["q"], state["k"], state["v"], case["window"], sinks=case["sinks"],
                                          kv_len=state["lens"])
    if case["kind"] == "logprobs":
        return _logprobs(state["logits"], state["tokens"], case["top"])
    if case["kind"] == "tree":
        k, v = (torch.cat((c, new), 1) for c, new in zip(state["cache"], (state["k"], state["v"])))
        return _attend(state["q"], k, v, _tree_sees(state, case)).to(torch.bfloat16)
    return _attend(state["q"], state["k"], state["v"], _window_sees(state, case)).to(torch.bfloat16)


# --------------------------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "logprobs":
        T, V = case["rows"], case["vocab"]
        # a subtraction, an exponential, the two sums; out: a value for each given token, the entropy, id and value
        return dict(bytes=T * V * SIZES[case["dtype"]] + T * (12 * case["given"] + 4 + 12 * case["top"]), flops=6 * T * V)
    B = case["batch"]
    row = 2 * HD                                       # bytes of a head's row
    if case["kind"] == "tree":
        n, lens = case["nodes"], _lengths(case, case["cache"])
        kept = max(lens) if case["shared"] else sum(lens)
        pairs = n * sum(lens) + B * int(_ancestors(case).sum())
        return dict(bytes=row * (2 * HK * (kept + B * n) + 2 * HQ * B * n) + 8 * n * -(-n // 64),
                    flops=4 * HQ * HD * pairs)
    n, pairs, rows = case["queries"], 0, 0
    for length in _lengths(case, case["keys"]):
        seen = lambda p: min(p + 1, case["window"] + min(case["sinks"], max(0, p + 1 - case["window"])))  # noqa: E731
        first = max(0, length - n)
        pairs += sum(seen(p) for p in range(first, length))
        oldest = max(0, first - case["window"] + 1)
        rows += length - oldest + min(case["sinks"], oldest)
    return dict(bytes=row * (2 * HK * rows + 2 * HQ * B * n), flops=4 * HQ * HD * pairs)


# ------------------------------------------------------------------------------------ 64-bit evaluation
def _exact_head(q, k, v, sees):
    """softmax(q k^T / 16) v of one head in float64; q [n, HD], k / v [S, HD], sees [n, S]."""
    z = torch.where(sees, q.double() @ k.double().t() * HD ** -0.5, -math.inf)
    top = z.max(1, keepdim=True).values
    w = torch.exp(z - torch.where(torch.isfinite(top), top, 0.0))
    total = w.sum(1, keepdim=True)
    return torch.where(total > 0, (w @ v.double()) / total, 0.0)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "logprobs":
        got, entropy, ids, best = [], [], [], []
        for x, t in zip(st["logits"].split(256), st["tokens"].split(256)):
            x = x.double()
            logp = x - torch.logsumexp(x, 1, keepdim=True)
            got.append(logp.gather(1, t.view(x.shape[0], -1)).view(t.shape))
            entropy.append(torch.special.entr(torch.exp(logp)).sum(1))
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            ids.append(order)
            best.append(logp.gather(1, order))
        return tuple(torch.cat(v) for v in (got, entropy, ids, best))
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(case["batch"]):
        if case["kind"] == "tree":
            n = int(st["lens"][b])
            sees = torch.cat((torch.ones(case["nodes"], n, dtype=torch.bool, device=DEV), st["sees"]), 1)
            k, v = (torch.cat((c[b, :n], new[b])) for c, new in zip(st["cache"], (st["k"], st["v"])))
        else:
            n = case["keys"] if st["lens"] is None else int(st["lens"][b])
            k, v = st["k"][b, :n], st["v"][b, :n]
            at = torch.arange(n - case["queries"], n, device=DEV)[:, None]
            gap = at - torch.arange(n, device=DEV)[None]
            sees = (gap >= 0) & ((gap < case["window"]) | (torch.arange(n, device=DEV)[None] < case["sinks"]))
        for h in range(HQ):
            out[b, :, h] = _exact_head(st["q"][b, :, h], k[:, h * HK // HQ], v[:, h * HK // HQ], sees)
    return out
