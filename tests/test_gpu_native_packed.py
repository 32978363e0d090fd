"""The native launch path of the packed and paged operators against the Python path: the same bits, or the same refusal."""
import pytest
import torch
from kv_model import Cache, starts_of
from test_gpu_native_path import BF, Sub, flat, outcome

from mica_amd import int8_kernels
from mica_amd.attention import packed_attention
from mica_amd.kv_cache import append_kv, paged_attention, read_kv


def forms(gpu):
    g = torch.Generator(device=gpu).manual_seed(4)
    rn = lambda *s, dt=BF: torch.randn(*s, generator=g, device=gpu).to(dt)  # noqa: E731
    q, k, v = rn(1100, 24, 256).split((16, 4, 4), dim=1)
    s, one = starts_of([30, 0, 70], gpu), starts_of([1100], gpu)
    held = [rn(n, 4, 256) for n in (300, 7, 96)]
    c = Cache(gpu, held, held, extra=5, slots=[2, 0, 1])
    kv, a = c.kv(), (s, c.lens, c.table, c.slots)
    ang = torch.rand(500, 32, generator=g, device=gpu)
    cos, sin, w, pos = ang.cos().to(BF), ang.sin().to(BF), rn(256), torch.arange(1100, dtype=torch.int32, device=gpu)
    out = torch.zeros(1100, 16, 256, dtype=BF, device=gpu)
    pk, pa = packed_attention, paged_attention

    def ap(*args, cache=kv, **kw):
        """What the call has stored, and that it returned its cache."""
        mine = type(cache)(*(t.clone() for t in cache))
        r = append_kv(mine, *args, **kw)
        return [r is mine, *mine]

    def into(f):
        o = out[:100].clone()
        r = f(o)
        return [r is o, o]

    k1, v1, q1 = k[:100], v[:100], q[:100]
    return {
        "pk": lambda: pk(q, k, v, s), "pk_hint": lambda: pk(q, k, v, s, 70), "pk_one": lambda: pk(q, k, v, one, 1100), "pk_none": lambda: pk(q, k, v, s[:1]),
        "pk_scale": lambda: pk(q, k, v, s, None, 0.3), "pk_hint_wide": lambda: pk(q, k, v, s, 2 ** 70), "pk_hint_minus": lambda: pk(q, k, v, s, -2),
        "pk_hint_float": lambda: pk(q, k, v, s, 70.0), "pk_hint_tensor": lambda: pk(q, k, v, s, torch.tensor(70)), "pk_scale_0": lambda: pk(q, k, v, s, scale=0.0),
        "pk_out": lambda: into(lambda o: pk(q1, k1, v1, s, out=o)), "pk_out_shape": lambda: pk(q, k, v, s, out=out[:9]), "pk_out_fp32": lambda: pk(q, k, v, s, out=out.float()),
        "pk_out_view": lambda: pk(q1, k1, v1, s, out=out.view(-1)[:100 * 16 * 272].view(100, 16, 272)[..., 8:264]),
        "pk_out_heads_first": lambda: pk(q1, k1, v1, s, out=out[:100].view(16, 100, 256).transpose(0, 1)),
        "pk_out_overlap": lambda: pk(q1, k1, v1, s, out=out.view(-1)[:256 * 115].as_strided((100, 16, 256), (256, 256, 1))),
        "pk_out_overlap_rows": lambda: pk(q1, k1, v1, s, out=out.view(-1).as_strided((100, 16, 256), (512, 256, 1))),
        "pk_empty": lambda: pk(q[:0], k[:0], v[:0], s), "pk_row": lambda: pk(q[:1], k[:1], v[:1], s), "pk_heads": lambda: pk(q[:, :8], k, v, s),
        "pk_rows": lambda: pk(q, k[:9], v[:9], s), "pk_kv": lambda: pk(q, k, v[:, :2], s), "pk_s64": lambda: pk(q, k, v, s.long()), "pk_s_cpu": lambda: pk(q, k, v, s.cpu()),
        "pk_s_strided": lambda: pk(q, k, v, torch.stack((s, s), 1)[:, 0]), "pk_fp16": lambda: pk(q.half(), k, v, s), "pk_cpu": lambda: pk(q.cpu(), k, v, s),
        "pk_k_cpu": lambda: pk(q, k.cpu(), v, s), "pk_sub": lambda: pk(q.as_subclass(Sub), k, v, s), "pk_param": lambda: pk(torch.nn.Parameter(q), k, v, s),
        "pk_odd": lambda: pk(q.contiguous().view(-1)[4:4 + 99 * 4096].view(99, 16, 256), k[:99], v[:99], s), "pk_rows_meet": lambda: pk(q, k[:1].expand(1100, -1, -1), v, s),
        "ap": lambda: ap(k1, v1, *a), "ap_hint": lambda: ap(k1, v1, *a, 70), "ap_no_slots": lambda: ap(k1, v1, *a[:3]), "ap_norm": lambda: ap(k1, v1, *a, norm=(w, 1.0, 1e-6)),
        "ap_norm_int": lambda: ap(k1, v1, *a, norm=(w, 1, 1e-6)), "ap_rope": lambda: ap(k1, v1, *a, rope=(cos, sin)), "ap_rope_pos": lambda: ap(k1, v1, *a, rope=(cos, sin, pos[:100])),
        "ap_rope_none": lambda: ap(k1, v1, *a, rope=(cos, sin, None)), "ap_rope_fp32": lambda: ap(k1, v1, *a, rope=(cos.float(), sin.float()), norm=(w, 0.0, 1e-5)),
        "ap_rope_types": lambda: ap(k1, v1, *a, rope=(cos.float(), sin)), "ap_rope_24": lambda: ap(k1, v1, *a, rope=(cos[:, :12].contiguous(), sin[:, :12].contiguous())),
        "ap_rope_view": lambda: ap(k1, v1, *a, rope=(cos[:, :16], sin[:, :16])), "ap_pos_short": lambda: ap(k1, v1, *a, rope=(cos, sin, pos[:99])),
        "ap_pos_64": lambda: ap(k1, v1, *a, rope=(cos, sin, pos[:100].long())), "ap_norm_short": lambda: ap(k1, v1, *a, norm=(w[:128], 1.0, 1e-6)),
        "ap_empty": lambda: ap(k[:0], v[:0], *a), "ap_kv": lambda: ap(k1, v[:9], *a), "ap_heads": lambda: ap(k1[:, :2], v1[:, :2], *a), "ap_lens_none": lambda: ap(k1, v1, s, None, c.table),
        "ap_lens_64": lambda: ap(k1, v1, s, c.lens.long(), c.table), "ap_table_64": lambda: ap(k1, v1, s, c.lens, c.table.long()), "ap_table_1d": lambda: ap(k1, v1, s, c.lens, c.table[0]),
        "ap_table_view": lambda: ap(k1, v1, s, c.lens, torch.cat((c.table, c.table), 1)[:, :c.table.shape[1]], c.slots), "ap_table_t": lambda: ap(k1, v1, s, c.lens, c.table.t()),
        "ap_table_0": lambda: ap(k1, v1, s, c.lens, c.table[:, :0], c.slots), "ap_slots_2": lambda: ap(k1, v1, s, c.lens, c.table, c.slots[:2]), "ap_cpu": lambda: ap(k1.cpu(), v1, *a),
        "ap_scales_16": lambda: ap(k1, v1, *a, cache=kv._replace(scales=c.scales.half())), "ap_sub": lambda: ap(k1.as_subclass(Sub), v1, *a),
        "ap_data_view": lambda: ap(k1, v1, *a, cache=kv._replace(data=c.data.transpose(3, 4).contiguous().transpose(3, 4))),
        "ap_tuple": lambda: append_kv(tuple(kv), k[:0], v[:0], *a)[0] is kv[0],
        "rd": lambda: read_kv(kv, 100, *a), "rd_hint": lambda: read_kv(kv, 100, *a, 70), "rd_no_slots": lambda: read_kv(kv, 100, *a[:3]), "rd_0": lambda: read_kv(kv, 0, *a),
        "rd_more": lambda: read_kv(kv, 130, *a), "rd_less": lambda: read_kv(kv, 50, *a), "rd_minus": lambda: read_kv(kv, -1, *a), "rd_float": lambda: read_kv(kv, 100.0, *a),
        "rd_wide": lambda: read_kv(kv, 2 ** 40, *a), "rd_tensor": lambda: read_kv(kv, torch.tensor(100), *a), "rd_none": lambda: read_kv(kv, 40, s[:1], c.lens[:0], c.table[:0]),
        "rd_s64": lambda: read_kv(kv, 100, s.long(), c.lens, c.table), "rd_slots": lambda: read_kv(kv, 100, s, c.lens, c.table, c.slots.float()),
        "pa": lambda: pa(q1, kv, *a), "pa_hint": lambda: pa(q1, kv, *a, 70), "pa_few": lambda: pa(q[:9], kv, starts_of([4, 3, 2], gpu), *a[1:], 4), "pa_scale": lambda: pa(q1, kv, *a, None, 0.2),
        "pa_no_slots": lambda: pa(q1, kv, *a[:3]), "pa_out": lambda: into(lambda o: pa(q1, kv, *a, out=o)), "pa_out_shape": lambda: pa(q1, kv, *a, out=out[:9]),
        "pa_out_overlap": lambda: pa(q1, kv, *a, out=out.view(-1).as_strided((100, 16, 256), (256, 256, 1))), "pa_none": lambda: pa(q, kv, s[:1], c.lens[:0], c.table[:0]),
        "pa_empty": lambda: pa(q[:0], kv, *a), "pa_row": lambda: pa(q[:1], kv, starts_of([1, 0, 0], gpu), *a[1:]), "pa_heads": lambda: pa(q1[:, :8], kv, *a), "pa_fp16": lambda: pa(q1.half(), kv, *a),
        "pa_cpu": lambda: pa(q1.cpu(), kv, *a), "pa_sub": lambda: pa(q1.as_subclass(Sub), kv, *a), "pa_neg": lambda: pa(q1, kv, *a, scale=-1.0), "pa_table_0": lambda: pa(q1, kv, s, c.lens, c.table[:, :0], c.slots),
        "pa_lens_none": lambda: pa(q1, kv, s, None, c.table), "pa_lens_cpu": lambda: pa(q1, kv, s, c.lens.cpu(), c.table), "pa_tuple": lambda: pa(q1, tuple(kv), *a),
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
            if isinstance(s, torch.Tensor):
                assert s.dtype == t.dtype and s.shape == t.shape and torch.equal(torch.nan_to_num(s), torch.nan_to_num(t)), name
            else:
                assert s is t, name


@pytest.mark.gpu
def test_outputs_that_overlap_are_refused(gpu):
    q, k, v = torch.zeros(100, 24, 256, dtype=BF, device=gpu).split((16, 4, 4), dim=1)
    c = Cache(gpu, [torch.zeros(200, 4, 256, dtype=BF, device=gpu)], [torch.zeros(200, 4, 256, dtype=BF, device=gpu)])
    mem = torch.zeros(100 * 16 * 256 + 4096, dtype=BF, device=gpu)
    for strides in ((256, 256), (2048, 256), (256, 2048), (4096, 264), (4096, 128)):
        out = mem.as_strided((100, 16, 256), (*strides, 1))
        with pytest.raises(ValueError, match="overlap"):
            packed_attention(q, k, v, starts_of([100], gpu), out=out)
        with pytest.raises(ValueError, match="overlap"):
            paged_attention(q, c.kv(), starts_of([100], gpu), c.lens, c.table, out=out)
    for strides in ((4096, 256), (256, 25600)):
        out = mem.as_strided((100, 16, 256), (*strides, 1))
        assert packed_attention(q, k, v, starts_of([100], gpu), out=out) is out
        assert paged_attention(q, c.kv(), starts_of([100], gpu), c.lens, c.table, out=out) is out
