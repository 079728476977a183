"""The router's and the FP8 rows' refusals that need no GPU: nothing is enqueued, so the addresses are made up (and the tests
are for machines without a GPU, where a call that is not refused ends with no device)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from exl3b200.native import Native, RouterDesc  # noqa: E402

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses")
E_SHAPE, E_DTYPE, E_ALIGN, E_STRIDE, E_INVAL, E_DEVICE = -1, -2, -3, -4, -12, -6


def router(**kw):
    d = dict(n_tok=40, n_expert=256, top_k=8, dtype=1, score=1, n_group=8, group_keep=4, group_top=2, renorm=1, scale=2.5,
             logits=4096, logits_pitch=256, bias=4096, ids=4096, w=4096, n_local=256, expert_base=0, sorted_tok=4096,
             expert_offset=4096, work=4096)
    desc = RouterDesc(**{**d, **kw})
    return Native().lib.exl3b200_router(C.addressof(desc), None)


@pytest.mark.parametrize("want,kw", [
    (E_DTYPE, dict(dtype=0)), (E_DTYPE, dict(dtype=1024 + 0x3B8)), (E_INVAL, dict(score=2)), (E_INVAL, dict(score=-1)),
    (E_INVAL, dict(scale=float("nan"))), (E_INVAL, dict(scale=float("inf"))), (E_SHAPE, dict(n_tok=-1)),
    (E_SHAPE, dict(n_tok=1 << 31)), (E_SHAPE, dict(n_expert=0)), (E_SHAPE, dict(n_expert=2049, n_group=1, group_keep=1)),
    (E_SHAPE, dict(n_expert=257)), (E_SHAPE, dict(top_k=0)), (E_SHAPE, dict(top_k=33)), (E_SHAPE, dict(n_group=0)),
    (E_SHAPE, dict(n_expert=264, n_group=33)), (E_SHAPE, dict(group_keep=0)), (E_SHAPE, dict(group_keep=9)),
    (E_SHAPE, dict(group_top=0)), (E_SHAPE, dict(group_top=3)), (E_SHAPE, dict(n_expert=16, logits_pitch=16, top_k=9)),
    (E_SHAPE, dict(n_expert=2040, logits_pitch=2040, n_group=5, group_keep=3)), (E_SHAPE, dict(n_local=0)),
    (E_SHAPE, dict(n_local=16385)), (E_INVAL, dict(sorted_tok=None)), (E_INVAL, dict(expert_offset=None)),
    (E_INVAL, dict(n_tok=4096, work=None)), (E_INVAL, dict(logits=None)), (E_INVAL, dict(ids=None)), (E_INVAL, dict(w=None)),
    (E_STRIDE, dict(logits_pitch=255)), (E_ALIGN, dict(logits=4098)), (E_ALIGN, dict(dtype=3, logits=4097)),
    (E_ALIGN, dict(bias=4097)), (E_ALIGN, dict(ids=4097)), (E_ALIGN, dict(w=4098)), (E_ALIGN, dict(sorted_tok=4097)),
    (E_ALIGN, dict(expert_offset=4097)), (E_ALIGN, dict(work=4097)),
    (E_DEVICE, dict()), (E_DEVICE, dict(bias=None, sorted_tok=None, expert_offset=None, work=None, n_local=0)),
    (E_DEVICE, dict(dtype=3, logits=4098)), (E_DEVICE, dict(n_expert=2048, logits_pitch=2048)),
    (E_DEVICE, dict(n_expert=96, n_group=3, group_keep=2))])
def test_router_refuses(want, kw):
    assert router(**kw) == want


def test_router_without_a_description():
    assert Native().lib.exl3b200_router(None, None) == E_INVAL


F8 = dict(x=4096, dtype=3, x_pitch=640, rows=10, cols=640, codes=4096, codes_pitch=640, scales=4096, scales_pitch=5)


@pytest.mark.parametrize("want,kw", [
    (E_SHAPE, dict(rows=-1)), (E_SHAPE, dict(cols=0)), (E_SHAPE, dict(cols=636)), (E_SHAPE, dict(rows=(1 << 30) + 1)),
    (E_SHAPE, dict(cols=(1 << 30) + 8)), (E_SHAPE, dict(rows=1 << 30, cols=1 << 20)), (E_DTYPE, dict(dtype=0)),
    (E_INVAL, dict(x=None)), (E_INVAL, dict(codes=None)), (E_INVAL, dict(scales=None)), (E_STRIDE, dict(x_pitch=632)),
    (E_STRIDE, dict(codes_pitch=632)), (E_STRIDE, dict(scales_pitch=4)), (E_ALIGN, dict(x=4104)), (E_ALIGN, dict(x_pitch=644)),
    (E_ALIGN, dict(codes=4100)), (E_ALIGN, dict(codes_pitch=644)), (E_ALIGN, dict(scales=4098)), (0, dict(rows=0, x=None)),
    (E_DEVICE, dict()), (E_DEVICE, dict(codes=4104, cols=8))])
def test_f8_rows_refuse(want, kw):
    a = {**F8, **kw}
    lib = Native().lib
    assert lib.exl3b200_f8_quantize(a["x"], a["dtype"], a["x_pitch"], a["rows"], a["cols"], a["codes"], a["codes_pitch"],
                                    a["scales"], a["scales_pitch"], 0, None) == want
    assert lib.exl3b200_f8_dequantize(a["codes"], a["codes_pitch"], a["scales"], a["scales_pitch"], a["rows"], a["cols"],
                                      a["x"], a["dtype"], a["x_pitch"], None) == want


def test_an_fp8_block_carves_disjoint_buffers_and_refuses_before_its_first_step():
    from exl3b200.native import ExpertBlockDesc
    nat = Native()
    at = {n: 4096 for n in ("router_w", "gu_w", "dn_w", "gu_scales", "dn_scales", "pre_w")}
    d = ExpertBlockDesc(n_expert=64, hidden=2064, width=528, top_k=10, dtype=3, weights=1024 + 0x3B8, eps=1e-6, res_scale=1.0, **at)
    for T in (1, 33, 2048):
        P, base, n = T * 10, 0x7F0000000010, nat.expert_block_work_bytes(d, T)
        b = nat.expert_block_carve(d, T, base, n)
        codes = b.h + (P * 528 * 2 + 255) // 256 * 256
        spans = sorted((a, a + size) for a, size in (
            (b.xn, T * 2064 * 2), (b.x_codes, T * 2064), (b.x_scales, T * 20 * 4), (b.logits, T * 64 * 4), (b.ids, P * 4), (b.w, P * 4),
            (b.sorted_tok, P * 4), (b.expert_offset, 65 * 4), (b.h, P * 528 * 2), (codes, P * 528), (b.h_scales, P * 8 * 4),
            (b.y_rows, P * 2064 * 2), (b.branch, T * 2064 * 4), (b.scatter_work, nat.scatter_work_bytes(P, 64)),
            (b.gather_work, nat.gather_work_bytes(T, 10))))
        assert spans[0][0] >= base and spans[-1][1] <= base + n and all(a % 256 == 0 for a, _ in spans)
        assert all(e <= s for (_, e), (s, _) in zip(spans, spans[1:]))
    f = nat.lib.exl3b200_expert_block_forward_routed
    r = dict(score=1, n_group=8, group_keep=4, group_top=2, renorm=1, scale=2.5)
    for want, k in ((E_DEVICE, {}), (E_SHAPE, dict(n_group=7)), (E_SHAPE, dict(group_keep=1)), (E_INVAL, dict(score=3)),
                    (E_ALIGN, dict(bias=4097))):
        assert f(d, RouterDesc(**{**r, **k}), b, 4096, 4, 4096, None, None) == want
    assert f(d, None, b, 4096, 4, 4096, None, None) == E_DEVICE
    for name, v, want in (("gu_scales", 4098, E_ALIGN), ("dn_scales", None, E_INVAL), ("gu_w", 4104, E_ALIGN), ("hidden", 2056, E_SHAPE)):
        bad = ExpertBlockDesc.from_buffer_copy(d)
        setattr(bad, name, v)
        assert f(bad, None, b, 4096, 4, 4096, None, None) == want, name
