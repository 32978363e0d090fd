"""The native launch path of the scoring operators against the Python path: the same bits, or the same refusal."""
import pytest
import torch
from test_gpu_native_path import BF, Sub, flat, outcome

from mica_amd import int8_kernels
from mica_amd.attention import tree_attention, tree_masks, window_attention
from mica_amd.readout import token_logprobs


def forms(gpu):
    g = torch.Generator(device=gpu).manual_seed(3)
    rn = lambda *s, dt=BF: torch.randn(*s, generator=g, device=gpu).to(dt)  # noqa: E731
    x, tok = rn(5, 9000), torch.randint(0, 9000, (5, 3), device=gpu)
    wide = rn(5, 9100)
    q, k, v = rn(2, 40, 24, 256).split((16, 4, 4), dim=2)
    kc, vc = rn(2, 300, 4, 256), rn(2, 300, 4, 256)
    m = tree_masks([-1] + [i // 2 for i in range(39)], gpu)
    m2 = torch.stack((m, m))
    n = torch.tensor([300, 20], dtype=torch.int32, device=gpu)
    lp, ta, wa = token_logprobs, tree_attention, window_attention
    return {
        "lp": lambda: lp(x, tok, 5), "lp_0": lambda: lp(x, tok), "lp_1d": lambda: lp(x, tok[:, 0].contiguous(), 5),
        "lp_i32": lambda: lp(x, tok.int(), 5), "lp_fp32": lambda: lp(x.float(), tok, 20), "lp_fp16": lambda: lp(x.half(), tok, 20),
        "lp_strided": lambda: lp(wide[:, 7:9007], tok, 5), "lp_strided_tokens": lambda: lp(x, tok[:, 1], 5),
        "lp_t": lambda: lp(x.t(), tok, 5), "lp_one_row": lambda: lp(x[:1], tok[:1], 5), "lp_empty": lambda: lp(x[:0], tok[:0], 5),
        "lp_no_tokens": lambda: lp(x, tok[:, :0], 5), "lp_33": lambda: lp(x, tok, 33), "lp_minus": lambda: lp(x, tok, -1),
        "lp_top_float": lambda: lp(x, tok, 5.0), "lp_top_tensor": lambda: lp(x, tok, torch.tensor(4)), "lp_rows": lambda: lp(x, tok[:4], 5),
        "lp_cpu": lambda: lp(x.cpu(), tok, 5), "lp_tok_cpu": lambda: lp(x, tok.cpu(), 5), "lp_sub": lambda: lp(x.as_subclass(Sub), tok, 5),
        "lp_double": lambda: lp(x.double(), tok, 5), "lp_param": lambda: lp(torch.nn.Parameter(x), tok, 5), "lp_v1": lambda: lp(x[:, :1], tok, 1),
        "lp_3d": lambda: lp(x[None], tok, 5), "lp_overlap": lambda: lp(x[:1].expand(5, -1), tok, 5),
        "tree": lambda: ta(q, k, v, m, cache=(kc, vc)), "tree_len": lambda: ta(q, k, v, m2, cache=(kc, vc), cache_len=n),
        "tree_none": lambda: ta(q, k, v, m), "tree_scale": lambda: ta(q, k, v, m, (kc, vc), None, 0.3), "tree_shared": lambda: ta(q, k, v, m, cache=[kc[0], vc[0]]),
        "tree_shared_4d": lambda: ta(q, k, v, m, cache=(kc[:1], vc[:1])), "tree_bhsd": lambda: ta(q, k, v, m, cache=tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kc, vc))),
        "tree_iter": lambda: ta(q, k, v, m, cache=iter((kc, vc))), "tree_node": lambda: ta(q[:, :1], k[:, :1], v[:, :1], m[:1], cache=(kc, vc)),
        "tree_c0": lambda: ta(q, k, v, m, cache=(kc[:, :0], vc[:, :0])), "tree_b0": lambda: ta(q[:0], k[:0], v[:0], m, cache=(kc[:0], vc[:0])),
        "tree_bad_mask": lambda: ta(q, k, v, m[:9], cache=(kc, vc)), "tree_mask_t": lambda: ta(q, k, v, m2.transpose(0, 1), cache=(kc, vc)),
        "tree_heads": lambda: ta(q[:, :, :8], k, v, m), "tree_kc_heads": lambda: ta(q, k, v, m, cache=(kc[:, :, :2], vc[:, :, :2])),
        "tree_neg": lambda: ta(q, k, v, m, scale=-1.0), "tree_fp16": lambda: ta(q.half(), k, v, m), "tree_len64": lambda: ta(q, k, v, m, cache=(kc, vc), cache_len=n.long()),
        "tree_sub": lambda: ta(q.as_subclass(Sub), k, v, m), "tree_cpu": lambda: ta(q, k, v, m.cpu()), "tree_rows_shared": lambda: ta(q, k[:, :1].expand(-1, 40, -1, -1), v, m),
        "win": lambda: wa(q, kc, vc, 100, 4), "win_len": lambda: wa(q, kc, vc, 100, 4, kv_len=n), "win_one": lambda: wa(q[:, :1], kc, vc, 200),
        "win_scale": lambda: wa(q, kc, vc, 100, scale=1.0), "win_self": lambda: wa(q, k, v, 7), "win_huge": lambda: wa(q, kc, vc, 2 ** 70, 2 ** 66),
        "win_0": lambda: wa(q, kc, vc, 0), "win_sinks": lambda: wa(q, kc, vc, 5, -1), "win_float": lambda: wa(q, kc, vc, 50.0), "win_b": lambda: wa(q[:1], kc, vc, 5),
        "win_no_keys": lambda: wa(q, kc[:, :0], vc[:, :0], 5), "win_no_queries": lambda: wa(q[:, :0], kc, vc, 5), "win_len_short": lambda: wa(q, kc, vc, 5, kv_len=n[:1]),
        "win_misaligned": lambda: wa(q.contiguous().view(-1)[4:4 + 2 * 39 * 16 * 256].view(2, 39, 16, 256), kc, vc, 5),
        "win_shared_keys": lambda: wa(q, kc[:1].expand(2, -1, -1, -1), vc[:1].expand(2, -1, -1, -1), 50),
    }


@pytest.mark.gpu
def test_native_path_equals_python_path(gpu, monkeypatch):
    monkeypatch.setattr(int8_kernels, "STRICT", False)
    for name, fn in forms(gpu).items():
        a, b = outcome(fn, True), outcome(fn, False)
        assert a[1:] == b[1:], (name, a[1:], b[1:])
        fa, fb = flat(a[0]), flat(b[0])
        assert len(fa) == len(fb), name
        for s, t in zip(fa, fb):
            assert (s is None and t is None) or (s.dtype == t.dtype and s.shape == t.shape
                                                 and torch.equal(torch.nan_to_num(s), torch.nan_to_num(t))), name
