"""Prompts, their cache, and what is asked over it, as a model's layer runs them: packed prompt attention beside the append of
its keys and values, questions that share a state's pages, single tokens, drafts over the rows read back.

Each attention result is held against float64 over the rows that the layer made (the cache's own rounding of finished blocks
applied to them), within the bound derived beside kv_model.check; the rows that are read back are those of that model, so the
tree's result has the same bound."""
import pytest
import torch
from kv_model import attend, check, starts_of, stored

from mica_amd import fused_kernels as fk
from mica_amd.attention import packed_attention, tree_attention, tree_masks
from mica_amd.int8_runtime import QLinear
from mica_amd.kv_cache import PAGE, PagedKV, append_kv, paged_attention, read_kv

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
H, HQ, HK, D, V = 512, 8, 2, 256, 5003
STATE, OTHER = 230, 41                    # a state that three questions share, and a prompt of its own
QUESTIONS = [50, 7, 0, 33]                # of sequences 0 .. 2 about the state; sequence 3 goes on with its own prompt


class Layer:
    def __init__(self, gpu):
        g = torch.Generator(device=gpu).manual_seed(12)
        rn = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
        self.embed = rn(V, H).to(BF)
        self.qkv = QLinear.from_quantized(torch.randint(-127, 128, ((HQ + 2 * HK) * D, H), generator=g, device=gpu).to(torch.int8),
                                          torch.full(((HQ + 2 * HK) * D,), 1 / 73 / H ** 0.5, device=gpu))
        ang = torch.arange(1024, device=gpu)[:, None] * 10000.0 ** (-torch.arange(32, device=gpu) / 32)
        self.cos, self.sin = ang.cos().to(BF), ang.sin().to(BF)
        self.norm = (rn(D) * 0.1).to(BF)

    def heads(self, tokens, pos, keys=True):
        """q, k, v views of the fused projection's rows; the keys rotated as well, or left to the append."""
        rows = self.qkv(self.embed[tokens])
        fk.head_norm_rope(rows, D, (0, HQ), (HQ * D, HK if keys else 0), rot_dim=64, cos_tab=self.cos, sin_tab=self.sin,
                          pos=pos.to(torch.int32).contiguous())
        return rows.view(-1, HQ + 2 * HK, D).split((HQ, HK, HK), dim=1)


def place(starts, lens):
    """Positions of packed rows that follow `lens` tokens of their sequences."""
    n = (starts[1:] - starts[:-1]).long()
    b = torch.repeat_interleave(torch.arange(n.numel(), device=starts.device), n)
    return torch.arange(b.numel(), device=starts.device) - starts[b] + lens[b]


@pytest.fixture
def job(gpu):
    g = torch.Generator(device=gpu).manual_seed(9)
    return Layer(gpu), lambda n: torch.randint(0, V, (n,), generator=g, device=gpu)


def test_prompts_questions_steps_and_drafts(gpu, job):
    layer, draw = job
    cache = PagedKV.empty(40, 6, HK, gpu)
    g = torch.Generator().manual_seed(2)
    free = torch.randperm(40, generator=g).tolist()
    # two prompts: the state in slot 4, the other in slot 3 (sequence 3's own)
    starts, lens = starts_of([STATE, OTHER], gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    table = torch.tensor([free[:12], free[12:24]], dtype=torch.int32, device=gpu)
    q, k, v = layer.heads(draw(STATE + OTHER), place(starts, lens))
    o = packed_attention(q, k, v, starts, longest=STATE)
    append_kv(cache, k, v, starts, lens, table, torch.tensor([4, 3], dtype=torch.int32, device=gpu), longest=STATE)
    ks, vs = [list(x.split((STATE, OTHER))) for x in (k, v)]
    for b, x in enumerate((o.split((STATE, OTHER)), q.split((STATE, OTHER)))[1]):
        check(o.split((STATE, OTHER))[b], *attend(x, ks[b], vs[b], 0))

    # the questions' sequences: the state's finished blocks by their pages, its rest copied into each one's slot
    full = STATE // PAGE
    tables = torch.full((4, 12), -1, dtype=torch.int32)
    at = 24
    for b in range(3):
        tables[b, :full] = torch.tensor(free[:full])
        tables[b, full:full + 3] = torch.tensor(free[at:at + 3])
        at += 3
    tables[3] = torch.tensor(free[12:24])
    tables = tables.to(gpu)
    cache.recent[:3] = cache.recent[4]
    lens = torch.tensor([STATE] * 3 + [OTHER], dtype=torch.int32, device=gpu)
    kept = [cache.data[free[:full]].clone(), cache.scales[free[:full]].clone(), cache.recent[4, :, :, :STATE % PAGE].clone()]
    rows = [[ks[0], vs[0]] for _ in range(3)] + [[ks[1], vs[1]]]

    def call(counts):
        nonlocal lens
        starts = starts_of(counts, gpu)
        q, k, v = layer.heads(draw(sum(counts)), place(starts, lens))
        append_kv(cache, k, v, starts, lens, tables, longest=max(counts))
        lens = lens + (starts[1:] - starts[:-1])
        o = paged_attention(q, cache, starts, lens, tables, longest=max(counts))
        i = 0
        for b, n in enumerate(counts):
            rows[b] = [torch.cat((rows[b][0], k[i:i + n])), torch.cat((rows[b][1], v[i:i + n]))]
            check(o[i:i + n], *attend(q[i:i + n], stored(rows[b][0]), stored(rows[b][1]), rows[b][0].shape[0] - n))
            i += n
        assert i == o.shape[0]

    call(QUESTIONS)
    for _ in range(3):
        call([1, 1, 1, 1])
    call([0, 30, 1, 0])
    assert all(torch.equal(a, b) for a, b in zip(kept, (cache.data[free[:full]], cache.scales[free[:full]],
                                                       cache.recent[4, :, :, :STATE % PAGE])))

    # all rows back, and drafts over them: a chain, as the paged attention of the same rows says it
    n = lens.tolist()
    kb, vb = read_kv(cache, sum(n), starts_of(n, gpu), lens, tables, longest=max(n))
    for b, (x, y) in enumerate(zip(kb.split(n), vb.split(n))):
        assert torch.equal(x, stored(rows[b][0]).to(BF)) and torch.equal(y, stored(rows[b][1]).to(BF))
    wide = [torch.zeros(4, max(n), HK, D, dtype=BF, device=gpu) for _ in range(2)]
    for b in range(4):
        wide[0][b, :n[b]], wide[1][b, :n[b]] = kb.split(n)[b], vb.split(n)[b]
    masks = tree_masks([-1, 0, 1, 2], gpu)
    q, k, v = layer.heads(draw(16), (lens[:, None] + torch.arange(4, device=gpu)).reshape(-1))
    tree = tree_attention(*(x.reshape(4, 4, -1, D) for x in (q, k, v)), masks, cache=tuple(wide), cache_len=lens)
    for b in range(4):
        back = [torch.cat((stored(r).to(BF), x[4 * b:4 * b + 4])) for r, x in zip(rows[b], (k, v))]
        check(tree[b], *attend(q[4 * b:4 * b + 4], *back, n[b]))


def test_steps_replayed_from_a_graph(gpu, job):
    """A captured step (projection, append with norm and rotation, attention, lengths counted on) is replayed over the ends of
    blocks, with the eager step on a copy of the cache between the replays."""
    layer, draw = job
    B, begin = 5, [0, 31, 60, 95, 128]
    table = torch.randperm(B * 6, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(B, 6).to(gpu)
    starts = starts_of([1] * B, gpu)
    norm = (layer.norm, 1.0, 1e-6)

    def fresh():
        cache = PagedKV.empty(B * 6, B, HK, gpu)
        lens = torch.zeros(B, dtype=torch.int32, device=gpu)
        s = starts_of(begin, gpu)
        q, k, v = layer.heads(prompt, place(s, lens), keys=False)
        append_kv(cache, k, v, s, lens, table, rope=(layer.cos, layer.sin), norm=norm)
        lens += s[1:] - s[:-1]
        return cache, lens

    def step(cache, lens, tokens):
        q, k, v = layer.heads(tokens, lens, keys=False)
        append_kv(cache, k, v, starts, lens, table, longest=1, rope=(layer.cos, layer.sin), norm=norm)
        lens += 1
        return paged_attention(q, cache, starts, lens, table, longest=1)

    prompt, tokens = draw(sum(begin)), draw(B)
    (ca, la), (cb, lb), (cc, lc) = fresh(), fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cc, lc, tokens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(ca, la, tokens)
    for turn in range(40):
        tokens.copy_(draw(B))
        graph.replay()
        torch.cuda.synchronize()
        want = step(cb, lb, tokens)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(la, lb), f"step {turn}"
        assert not torch.isnan(want).any()
    n = lb.tolist()
    assert n == [x + 40 for x in begin]
    for x, y in zip(*(read_kv(c, sum(n), starts_of(n, gpu), ln, table) for c, ln in ((ca, la), (cb, lb)))):
        assert torch.equal(x, y)


def test_two_streams_at_once(gpu, job):
    """Two requests' layers on streams of their own, at the same time, over one cache: each as it is alone."""
    layer, draw = job
    cache = PagedKV.empty(200, 4, HK, gpu)
    table = torch.arange(200, dtype=torch.int32, device=gpu).view(4, 50)
    jobs = []
    for b, n in enumerate((700, 1500)):
        pos = torch.arange(n, device=gpu)
        jobs.append((*layer.heads(draw(n), pos), starts_of([n], gpu), torch.zeros(1, dtype=torch.int32, device=gpu),
                     torch.full((1,), n, dtype=torch.int32, device=gpu), table[b:b + 1], torch.full((1,), b, dtype=torch.int32, device=gpu)))

    def run(q, k, v, starts, none, lens, tab, slot):
        append_kv(cache, k, v, starts, none, tab, slot)
        return packed_attention(q, k, v, starts), paged_attention(q, cache, starts, lens, tab, slot), *read_kv(cache, q.shape[0], starts, lens, tab, slot)

    alone = [[x.clone() for x in run(*j)] for j in jobs]
    torch.cuda.synchronize()
    cache.data.zero_(), cache.scales.zero_(), cache.recent.zero_()
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    both = [[], []]
    for _ in range(4):
        for i, (st, j) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(st):
                both[i].append(run(*j))
    torch.cuda.synchronize()
    for i in range(2):
        for got in both[i]:
            assert all(torch.equal(x, y) for x, y in zip(got, alone[i]))
