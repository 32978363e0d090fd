"""The scoring of drafted continuations as a model's layer runs it: a prompt's attention within a window, a tree of drafts
over the prompt's keys, and the log probabilities of their tokens.

The layer quantizes and projects row by row, so a token has the same q / k / v bits wherever it stands at one position; two
attention results of the same numbers then differ by the roundings of both, 2 (2^-8 (A + |o|) + 2^-11 A) with
A <= max |v| of the head (the bound of one is derived beside the operators' own tests)."""
import pytest
import torch

from mica_amd import fused_kernels as fk
from mica_amd.attention import causal_gqa_attention, tree_attention, tree_masks, window_attention
from mica_amd.int8_runtime import QLinear
from mica_amd.readout import token_logprobs

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
H, HQ, HK, D, V = 512, 8, 2, 256, 5003
P, LENS = 150, (150, 97, 33)
PARENTS = [[-1, 0, 0, 1, 1, 2, 5, -1, 7, 8], [-1, 0, 1, 2, 3, 4, 5, 6, -2, -2], [-1, -1, -1, 0, 1, 2, 3, 3, 4, 6]]
N = len(PARENTS[0])


class Layer:
    def __init__(self, gpu):
        g = torch.Generator(device=gpu).manual_seed(11)
        rn = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
        self.embed = rn(V, H).to(BF)
        self.qkv = QLinear.from_quantized(torch.randint(-127, 128, ((HQ + 2 * HK) * D, H), generator=g, device=gpu).to(torch.int8),
                                          torch.full(((HQ + 2 * HK) * D,), 1 / 73 / H ** 0.5, device=gpu))
        self.head = (rn(V, HQ * D) * 0.02).to(BF)
        ang = torch.arange(512, device=gpu)[:, None] * 10000.0 ** (-torch.arange(32, device=gpu) / 32)
        self.cos, self.sin = ang.cos().to(BF), ang.sin().to(BF)

    def heads(self, tokens, pos):
        """q, k, v views of the fused projection's rows at positions `pos`."""
        B, n = tokens.shape
        rows = self.qkv(self.embed[tokens].view(B * n, H))
        fk.head_norm_rope(rows, D, (0, HQ), (HQ * D, HK), rot_dim=64, cos_tab=self.cos, sin_tab=self.sin,
                          pos=pos.reshape(-1).to(torch.int32).contiguous())
        rows = rows.view(B, n, HQ + 2 * HK, D)
        return rows[:, :, :HQ], rows[:, :, HQ:HQ + HK], rows[:, :, HQ + HK:]

    def logits(self, o):
        return (o.reshape(-1, HQ * D) @ self.head.t()).float()


@pytest.fixture
def job(gpu):
    g = torch.Generator(device=gpu).manual_seed(5)
    layer = Layer(gpu)
    prompt = torch.randint(0, V, (3, P), generator=g, device=gpu)
    drafts = torch.randint(0, V, (3, N), generator=g, device=gpu)
    lens = torch.tensor(LENS, dtype=torch.int32, device=gpu)
    depth = torch.zeros(3, N, dtype=torch.int64)
    for b, tree in enumerate(PARENTS):
        for i, p in enumerate(tree):
            depth[b, i] = depth[b, p] + 1 if p >= 0 else 0
    return layer, prompt, drafts, lens, tree_masks(PARENTS, gpu), depth.to(gpu)


def run(layer, prompt, drafts, lens, masks, depth, window=10 ** 6):
    at = torch.arange(P, device=prompt.device).expand(3, P)
    q, k, v = layer.heads(prompt, at)
    o = window_attention(q, k, v, window, 4)
    first = token_logprobs(layer.logits(o), prompt.roll(-1, 1).reshape(-1), 5)
    qt, kt, vt = layer.heads(drafts, lens[:, None] + depth)
    ot = tree_attention(qt, kt, vt, masks, (k, v), lens)
    second = token_logprobs(layer.logits(ot), drafts.roll(-1, 1).reshape(-1), 20)
    return o, first, ot, second


def test_a_branch_is_scored_like_the_plain_sequence(gpu, job):
    layer, prompt, drafts, lens, masks, depth = job
    _, _, ot, second = run(*job)
    x = layer.logits(ot)
    for b, tree in enumerate(PARENTS):
        for node, p in enumerate(tree):
            if p == -2:
                assert not ot[b, node].any()                    # no node: zeros, and the row's logits are equal
                assert (second.entropy.view(3, N)[b, node] - torch.tensor(float(V)).log()).abs() < 1e-5
                continue
            path = [node]
            while tree[path[0]] >= 0:
                path.insert(0, tree[path[0]])
            seq = torch.cat([prompt[b, :LENS[b]], drafts[b, path]])[None]
            q, k, v = layer.heads(seq, torch.arange(seq.shape[1], device=gpu)[None])
            got = ot[b, node].float()
            top = v[0].float().abs().amax((0, 1))
            for o in (window_attention(q, k, v, seq.shape[1]), causal_gqa_attention(q, k, v)):
                o = o[0, -1].float()
                d = (got - o).abs() - 2 * (2 ** -8 * (top + o.abs()) + 2 ** -11 * top)
                assert (d <= 0).all(), f"sequence {b}, node {node}: {d.max():.3g} over"
            lp = torch.log_softmax(x[b * N + node].double(), 0)
            t = drafts.roll(-1, 1)[b, node]
            assert abs(second.logprobs.view(3, N)[b, node] - lp[t]) < 1e-5 * (1 + abs(lp[t]))
            assert torch.equal(second.top_ids.view(3, N, 20)[b, node], torch.sort(lp, descending=True, stable=True).indices[:20])


def test_the_run_on_a_side_stream_and_replayed(gpu, job):
    """All of it in one captured graph, replayed on new drafts and lengths with the eager run between the replays."""
    layer, prompt, drafts, lens, masks, depth = job
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*job, window=40)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*job, window=40)
    g = torch.Generator(device=gpu).manual_seed(6)
    for turn in range(4):
        prompt.copy_(torch.randint(0, V, prompt.shape, generator=g, device=gpu))
        drafts.copy_(torch.randint(0, V, drafts.shape, generator=g, device=gpu))
        lens.copy_(torch.tensor([(turn * 61 + 40 * b) % P for b in range(3)], dtype=torch.int32, device=gpu))
        graph.replay()
        torch.cuda.synchronize()
        want = run(*job, window=40)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2])
        for a, b in ((out[1], want[1]), (out[3], want[3])):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
