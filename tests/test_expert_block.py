"""The residual MoE block over f16 / bf16 / MXFP4 experts (exl3b200_expert_block_forward), and on the CPU its carve and
refusals.

On a GPU the block is checked in two ways. Against the composition of the entries it is made of, each of which has its own
test against 64 bits: to the bit, since it is the same calls. And against the whole formula in 64 bits with the routing the
block itself chose (its f32 logits are compared with 64 bits on their own, so that a near tie may go either way): the
stream's type is rounded six times on the way (norm, h, rows, gather, norm, out), each relative 2^-8 (bf16) of a value
that the following product mixes at random, so 2^-6 of the output's root mean square holds for 16-bit experts. MXFP4 h and x
round by up to a quarter of a value a block: there the composition is the test."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from exl3b200 import dense  # noqa: E402
from exl3b200.native import ExpertBlockBufs, ExpertBlockDesc, Native  # noqa: E402


def host_desc(**k):
    d = ExpertBlockDesc(n_expert=64, hidden=2048, width=512, top_k=10, dtype=3, weights=3, eps=1e-6, res_scale=1.0,
                        router_w=16, gu_w=16, dn_w=16, pre_w=16)
    for name, v in k.items():
        setattr(d, name, v)
    return d


@pytest.mark.parametrize("weights", [3, dense.MX4])
@pytest.mark.parametrize("T", [1, 33, 2048])
def test_carve_is_disjoint_and_in_bounds(weights, T):
    nat = Native()
    d = host_desc(weights=weights, gu_scales=16, dn_scales=16)
    E, H, W, P = d.n_expert, d.hidden, d.width, T * d.top_k
    mx = weights == dense.MX4
    n = nat.expert_block_work_bytes(d, T)
    base = 0x7F0000000010
    b = nat.expert_block_carve(d, T, base, n)
    size = {"xn": T * H * 2, "logits": T * E * 4, "ids": P * 4, "w": P * 4, "sorted_tok": P * 4, "expert_offset": (E + 1) * 4,
            "scatter_work": int(nat.lib.exl3b200_moe_scatter_work_bytes(P, E)), "h": P * W // 2 if mx else P * W * 2,
            "y_rows": P * H * 2, "branch": T * H * 4, "gather_work": nat.gather_work_bytes(T, d.top_k)}
    if mx:
        size |= {"x_codes": T * H // 2, "x_scales": T * H // 32, "h_scales": P * W // 32}
    else:
        assert not b.x_codes and not b.x_scales and not b.h_scales
    spans = sorted((getattr(b, k), getattr(b, k) + v) for k, v in size.items())
    assert spans[0][0] >= base and spans[-1][1] <= base + n and all(a % 256 == 0 for a, _ in spans)
    assert all(e <= s for (_, e), (s, _) in zip(spans, spans[1:]))
    assert b.max_tokens == T
    assert nat.lib.exl3b200_expert_block_carve(d, T, base, n - 1, b) == -5


def test_refusals_before_anything_is_enqueued():
    nat = Native()
    for k in (dict(n_expert=60), dict(n_expert=0), dict(n_expert=4096), dict(top_k=0), dict(top_k=33), dict(hidden=2044),
              dict(hidden=65536), dict(width=4), dict(dtype=1), dict(weights=2), dict(router_w=0), dict(gu_w=0),
              dict(dn_w=0), dict(pre_w=0), dict(weights=dense.MX4), dict(weights=dense.MX4, gu_scales=16, dn_scales=16, width=520)):
        d = host_desc(**k)
        assert nat.lib.exl3b200_expert_block_work_bytes(d, 8) == -1, k
        assert nat.lib.exl3b200_expert_block_forward(d, ExpertBlockBufs(max_tokens=8), 16, 1, 16, None, None) < 0, k
    d, b = host_desc(), ExpertBlockBufs(max_tokens=8)
    assert nat.lib.exl3b200_expert_block_work_bytes(d, 0) == -1
    assert nat.lib.exl3b200_expert_block_work_bytes(d, 1 << 24) == -1
    f = nat.lib.exl3b200_expert_block_forward
    assert f(d, b, 16, 9, 16, None, None) == -12 and f(d, b, 16, -1, 16, None, None) == -12
    assert f(d, b, None, 1, 16, None, None) == -12 and f(d, b, 16, 1, None, None, None) == -12
    assert f(d, b, 16, 1, 16, 16, None) == -12              # a next norm without its weight
    assert f(d, b, None, 0, None, None, None) == 0


def make(E, H, W, k, dtype, mx, seed, max_tokens):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(s, generator=g, device="cuda") * scale)  # noqa: E731
    t = {"router_w": r(E, H, scale=H ** -0.5).to(dtype), "pre_w": (1 + r(H, scale=0.1)).to(dtype),
         "post_w": (1 + r(H, scale=0.1)).to(dtype), "gate": r(H).to(dtype), "next_w": (1 + r(H, scale=0.1)).to(dtype)}
    gu, dn = r(E, 2 * W, H, scale=H ** -0.5), r(E, H, W, scale=W ** -0.5)
    if mx:
        for name, w in (("gu", gu), ("dn", dn)):
            q, s = dense.mx4_empty(w.shape[0] * w.shape[1], w.shape[2])
            dense.mx4_quantize(w.reshape(-1, w.shape[2]), q, s, torch.cuda.current_stream().cuda_stream)
            t[name + "_w"] = q.reshape(*w.shape[:2], -1)
            t[name + "_scales"] = s.reshape(*w.shape[:2], -1).contiguous()
    else:
        t |= {"gu_w": gu.to(dtype), "dn_w": dn.to(dtype)}
    return t, dense.ExpertBlock(top_k=k, eps=1e-6, res_scale=0.5, max_tokens=max_tokens, **t)


def composed(t, block, x, k, mx):
    """The same block from its entries, each called by itself."""
    T, H = x.shape
    E, W = t["router_w"].shape[0], block.desc.width
    st, dt, dev, nat = torch.cuda.current_stream().cuda_stream, x.dtype, x.device, dense.native()
    new = lambda *s, dtype: torch.empty(s, dtype=dtype, device=dev)  # noqa: E731
    xn = new(T, H, dtype=dt)
    q, s = dense.mx4_empty(T, H) if mx else (None, None)
    dense.BlockNorm(res=x, pre_w=t["pre_w"], pre_eps=1e-6, y=xn, y_codes=q, y_scales=s).run(st)
    logits = new(T, E, dtype=torch.float32)
    dense.GroupedMm(x=xn, w=t["router_w"][None], y=logits).run(st)
    ids, w, tok = new(T, k, dtype=torch.int32), new(T, k, dtype=torch.float32), new(T * k, dtype=torch.int32)
    off, work = new(E + 1, dtype=torch.int32), new(nat.scatter_work_bytes(T * k, E), dtype=torch.uint8)
    nat.router_scatter(logits.data_ptr(), T, E, k, ids.data_ptr(), w.data_ptr(), E, 0, tok.data_ptr(), off.data_ptr(),
                       work.data_ptr(), st)
    rows = new(T * k, H, dtype=torch.bfloat16)
    kw = dict(expert_offset=off, sorted_tok=tok)
    if mx:
        h, hs = dense.mx4_empty(T * k, W)
        dense.GroupedMm(x=q, x_scales=s, w=t["gu_w"], w_scales=dense.mx4_tile_scales(t["gu_scales"], "silu_mul"), y=h,
                        y_scales=hs, top_k=k, act="silu_mul", **kw).run(st)
        dense.GroupedMm(x=h, x_scales=hs, w=t["dn_w"], w_scales=dense.mx4_tile_scales(t["dn_scales"]), y=rows, **kw).run(st)
    else:
        h = new(T * k, W, dtype=dt)
        dense.GroupedMm(x=xn, w=t["gu_w"], y=h, top_k=k, act="silu_mul", **kw).run(st)
        dense.GroupedMm(x=h, w=t["dn_w"], y=rows, **kw).run(st)
    branch, gw = new(T, H, dtype=torch.float32), new(nat.gather_work_bytes(T, k), dtype=torch.uint8)
    nat.moe_gather(rows.data_ptr(), H, tok.data_ptr(), T * k, w.data_ptr(), T, k, H, branch.data_ptr(), gw.data_ptr(), st)
    out, nxt = new(T, H, dtype=dt), new(T, H, dtype=dt)
    dense.BlockNorm(branch=branch, post_w=t["post_w"], post_eps=1e-6, gate=t["gate"], gate_kind="channel", res=x,
                    res_scale=0.5, out=out, pre_w=t["next_w"], pre_eps=1e-6, y=nxt).run(st)
    return out, nxt, logits, ids, w


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 17, 300])
@pytest.mark.parametrize("dtype,mx", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True),
                                      (torch.float16, True)])
def test_block_is_its_entries_and_its_formula(T, dtype, mx):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    E, H, W, k = 32, 512, 256, 4
    t, block = make(E, H, W, k, dtype, mx, 5, 300)
    x = torch.randn((T, H), generator=torch.Generator(device="cuda").manual_seed(T), device="cuda").to(dtype)
    st = torch.cuda.current_stream().cuda_stream
    out, nxt = torch.empty_like(x), torch.empty_like(x)
    block.forward(x, out, nxt, st)
    want, want_next, logits, ids, w = composed(t, block, x, k, mx)
    assert torch.equal(out, want) and torch.equal(nxt, want_next)
    # in place, and without the next norm
    y = x.clone()
    block.forward(y, y, stream=st)
    assert torch.equal(y, want)
    # the formula
    rms = lambda v: v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)  # noqa: E731
    xd = x.double()
    xn = rms(xd) * t["pre_w"].double()
    z = xn @ t["router_w"].double().T
    # each logit sums 512 products of normed values (rounded to 2^-8 or 2^-11) and weights: random signs, 6 sigma
    sigma = 2.0 ** (-8 if dtype == torch.bfloat16 else -11) * ((xn * xn) @ (t["router_w"].double() ** 2).T).sqrt()
    assert bool(((logits.double() - z).abs() <= 6 * sigma + 1e-5).all())
    assert torch.equal(w, torch.softmax(logits, 1).gather(1, ids.long())) or \
        torch.allclose(w, torch.softmax(logits, 1).gather(1, ids.long()), rtol=1e-5, atol=0)
    if not mx:
        br = torch.zeros_like(xd)
        for s in range(k):
            e = ids[:, s].long()
            gu = torch.einsum("th,tnh->tn", xn, t["gu_w"].double()[e])
            h = gu[:, :W] * torch.sigmoid(gu[:, :W]) * gu[:, W:]
            br += w[:, s:s + 1].double() * torch.einsum("tw,thw->th", h, t["dn_w"].double()[e])
        r = 0.5 * xd + t["gate"].double() * rms(br) * t["post_w"].double()
        assert float((out.double() - r).norm() / r.norm()) <= 2.0 ** -6
        nx = rms(r) * t["next_w"].double()
        assert float((nxt.double() - nx).norm() / nx.norm()) <= 2.0 ** -6
    assert dense.native().read_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("mx", [False, True])
def test_block_replays_in_a_cuda_graph(mx):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    t, block = make(64, 2048, 512, 10, torch.bfloat16, mx, 9, 64)
    x = torch.randn((64, 2048), device="cuda").to(torch.bfloat16)
    out = torch.empty_like(x)
    block.forward(x, out, stream=torch.cuda.current_stream().cuda_stream)
    ref = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.forward(x, out, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, ref)


@pytest.mark.gpu
def test_block_refuses_what_does_not_fit():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    t, block = make(8, 64, 64, 2, torch.bfloat16, False, 1, 4)
    x = torch.zeros((5, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):
        block.forward(x, torch.empty_like(x))
    with pytest.raises(ValueError):
        block.forward(x[:4], torch.empty((4, 64), device="cuda"))
    with pytest.raises(ValueError):
        block.forward(x[:4, ::2], x[:4, ::2])
    with pytest.raises(ValueError):
        dense.ExpertBlock(top_k=2, **dict(t, dn_w=t["dn_w"][:4]))
