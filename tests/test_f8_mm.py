"""grouped_mm over FP8 operands on a GPU, against a plain implementation in 64 bits.

Tolerance, from the arithmetic alone: a block's 128 products of two 4-bit significands are exact, their sum in f32 -- any order
of rounded or truncated additions -- is within 128 * 2^-23 of the sum of magnitudes; the product of two scales is rounded once
and each block added with one rounding, (ceil(K / 128) + 2) * 2^-24 of the magnitudes so far at most, and a split k adds its up to
four parts with three more. silu_mul carries the two sums' errors through |silu'| <= 1.1 and |silu(g)| <= |g| and adds 2^-19 of
the value (its approximate exponential and quotient); an output type of p bits adds 2^-p of the value."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402
from test_dense import close, counts_of, gen, randn, routing, stream  # noqa: E402

F32, F16, BF16, F8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()
    assert dense.native().read_error() == 0


def codes(g, *shape):
    """e4m3 codes of N(0, 60): both signs, the subnormal ones too."""
    return (60 * torch.randn(shape, generator=g, device="cuda")).clamp(-448, 448).to(F8)


def scales(g, *shape):
    """About 1, four powers of two apart, every significand."""
    return torch.exp2(4 * torch.rand(shape, generator=g, device="cuda") - 2)


def weight_blocks(N, act):
    return -(-N // 128) * (2 if act == "silu_mul" else 1)


def values_of(w, ws, N):
    """A weight's values in 64 bits: block r / 128 of gate's rows, then of up's."""
    E, rows, K = w.shape
    r, c = torch.arange(rows, device="cuda"), torch.arange(K, device="cuda") // 128
    block = torch.where(r < N, r // 128, -(-N // 128) + (r - N) // 128)
    return w.double() * ws.double()[:, block][:, :, c]


def operands(seed, E, rows, K, N, act):
    g = gen(seed)
    x, (xq, xs) = codes(g, rows, K), dense.f8_empty(rows, K)
    xq.copy_(x)
    xs.copy_(scales(g, *xs.shape))
    w = codes(g, E, N * (2 if act == "silu_mul" else 1), K)
    ws = scales(g, E, weight_blocks(N, act), -(-K // 128)) / (60 * 60 * K ** 0.5)
    xv = xq.double() * xs.double()[:, torch.arange(K, device="cuda") // 128]
    return xq, xs, w, ws, xv


def case(seed, counts, K, N, act, top_k=1, out=F32, before=0, after=0, dropped=()):
    """Runs one product; returns what it wrote, the plan, and (the wanted values, the tolerance)."""
    g = gen(seed)
    tok, off, n = routing(counts, before, after, dropped, g=g)
    x_rows = max(1, (n + top_k - 1) // top_k)
    xq, xs, w, ws, xv = operands(seed, len(counts), x_rows, K, N, act)
    y = torch.full((n, N), float("nan"), dtype=out, device="cuda")
    plan = dense.GroupedMm(x=xq, x_scales=xs, w=w, w_scales=ws, expert_offset=off, sorted_tok=tok, top_k=top_k, act=act, y=y)
    plan.run(stream())
    return y, plan, plain(xv, values_of(w, ws, N), tok, off, top_k, act, N), (xq, xs, w, ws, tok, off)


def plain(xv, wv, tok, off, top_k, act, N, dx=None):
    """(y, its tolerance without the output type's) in 64 bits; dx: what each x may be off by besides."""
    unit = (128 + -(-xv.shape[1] // 128) + 5) * 2.0 ** -23
    y = torch.zeros((len(tok), N), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(y)
    o = off.tolist()
    for e in range(len(o) - 1):
        rows = torch.arange(o[e], o[e + 1], device="cuda")
        rows = rows[tok[rows] >= 0]
        if not rows.numel():
            continue
        t = tok[rows].long() // top_k if top_k else rows
        d = unit * xv[t].abs() + (dx[t] if dx is not None else 0)
        z, s = xv[t] @ wv[e].T, d @ wv[e].abs().T
        if act == "none":
            y[rows], tol[rows] = z, s
        else:
            g, u, sg, su = z[:, :N], z[:, N:], s[:, :N], s[:, N:]
            v = g * torch.sigmoid(g) * u
            y[rows], tol[rows] = v, 1.1 * sg * (u.abs() + su) + (g.abs() + sg) * su + 2.0 ** -19 * v.abs()
    return y, tol


@pytest.mark.parametrize("kind", ["one", "empty", "few", "ragged", "large", "many"])
@pytest.mark.parametrize("K,N", [(16, 8), (144, 40), (512, 200), (2048, 512), (640, 2560), (1040, 136)])
@pytest.mark.parametrize("act", ["none", "silu_mul"])
def test_grouped_mm_f8(kind, K, N, act):
    counts = counts_of(kind, gen(K + N))
    for out in (F32, F16, BF16) if K == 512 else (F32,):
        y, _, (want, tol), _ = case(K * 3 + N, counts, K, N, act, top_k=2, out=out)
        close(y, want, tol, out)


FORMS = {"split": ([1, 3], 1024, 128), "narrow": ([5] * 40, 512, 512),
         "wide": ([300, 0, 41, 700, 128, 257, 90, 500], 1024, 1280)}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("act", ["none", "silu_mul"])
@pytest.mark.parametrize("out", [F32, F16, BF16])
def test_every_form_with_dropped_slots_and_rows_outside(form, act, out):
    counts, K, N = FORMS[form]
    live = sum(counts)
    dropped = sorted({0, live // 2, live - 1} | set(range(live // 3, live // 3 + 3 if live > 8 else live // 3)))
    y, _, (want, tol), t = case(7, counts, K, N, act, out=out, before=3, after=5, dropped=[3 + d for d in dropped])
    tok = t[4]
    dead = (tok < 0) | (torch.arange(len(tok), device="cuda") < 3) | (torch.arange(len(tok), device="cuda") >= 3 + live)
    assert dead.sum() >= 8 and not y[dead].any()
    close(y[~dead], want[~dead], tol[~dead], out)


@pytest.mark.parametrize("rows", [1, 31, 33, 97, 255, 257, 1024, 2869, 4100, 9001])
@pytest.mark.parametrize("N,act", [(248, "silu_mul"), (512, "none"), (1064, "none"), (192, "silu_mul")])
def test_one_expert_of_many_rows(rows, N, act):
    y, _, (want, tol), _ = case(rows, [rows], 272, N, act)
    close(y, want, tol, F32)


@pytest.mark.parametrize("K", [16, 272, 640, 3824])
@pytest.mark.parametrize("form", ["narrow", "wide", "split"])
@pytest.mark.parametrize("shift,extra", [(0, 0), (1, 0), (3, 2), (4, 4), (2, 5)])
def test_scales_at_any_alignment(K, form, shift, extra):
    """x's scales any number of floats into their memory and any pitch apart, poison between them."""
    rows, N, E = {"narrow": (50, 1048, 20), "wide": (2100, 2048, 2), "split": (9, 128, 2)}[form]
    xq, xs, w, ws, xv = operands(K + shift, E, rows, K, N, "none")
    kb = -(-K // 128)
    mem = torch.full((shift + rows * (kb + extra),), float("nan"), device="cuda")
    odd = mem[shift:].view(rows, kb + extra)[:, :kb]
    odd.copy_(xs)
    off = torch.tensor([rows * e // E for e in range(E + 1)], dtype=torch.int32, device="cuda")
    y = torch.full((rows, N), float("nan"), device="cuda")
    dense.GroupedMm(x=xq, x_scales=odd, w=w, w_scales=ws, expert_offset=off, y=y).run(stream())
    tok, wv = torch.arange(rows, dtype=torch.int32, device="cuda"), values_of(w, ws, N)
    close(y, *plain(xv, wv, tok, off, 0, "none", N), F32)


@pytest.mark.parametrize("N,counts", [(136, [40, 7, 90]), (1096, [40, 3000, 7, 900])])
def test_strided_operands_and_neighbours_left_alone(N, counts):
    K = 272
    y, _, (want, tol), (xq, xs, w, ws, tok, off) = case(5, counts, K, N, "none")
    bx = torch.full((xq.shape[0], K + 48), 0x7F, dtype=torch.uint8, device="cuda")
    bw = torch.full((len(counts), N + 5, K + 16), 0x7F, dtype=torch.uint8, device="cuda")
    bx[:, 16:16 + K] = xq.view(torch.uint8)
    bw[:, :N, :K] = w.view(torch.uint8)
    by = torch.full((len(tok) + 2, N + 8), 7.0, device="cuda")
    dense.GroupedMm(x=bx[:, 16:16 + K].view(F8), x_scales=xs, w=bw[:, :N, :K].view(F8), w_scales=ws, expert_offset=off,
                    sorted_tok=tok, top_k=1, y=by[1:-1, :N]).run(stream())
    assert torch.equal(by[1:-1, :N], y)
    assert (by[[0, -1]] == 7).all() and (by[:, N:] == 7).all()


@pytest.mark.parametrize("many,N", [(0, 264), (3000, 1032)])
def test_values_that_are_no_numbers_stay_in_their_rows(many, N):
    """A row whose scale is NaN, an expert with a NaN code in one weight row; zero scales; an expert of many rows besides."""
    counts, K = [30, 50, 20] + [many] * (many > 0), 384
    y, _, (want, tol), (xq, xs, w, ws, tok, off) = case(9, counts, K, N, "none")
    xs[tok[10].item()] = float("nan")
    xs[tok[12].item(), 1] = 0
    w.view(torch.uint8)[1, 100, 5] = 0x7F
    ws[2] = 0
    got = torch.empty_like(y)
    dense.GroupedMm(x=xq, x_scales=xs, w=w, w_scales=ws, expert_offset=off, sorted_tok=tok, top_k=1, y=got).run(stream())
    assert got[10].isnan().all() and got[30:80, 100].isnan().all() and not got[80:100].any()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[[10, 12]] = keep[80:100] = False
    keep[30:80, 100] = False
    assert torch.equal(got[keep], y[keep])


@pytest.mark.parametrize("E,n,N", [(5, 1, 264), (5, 40, 264), (3, 900, 1056), (3, 5000, 1056)])
@pytest.mark.parametrize("start", [0, 1])
def test_no_expert_has_a_row(E, n, N, start):
    xq, xs, w, ws, _ = operands(E + n, E, n, 512, N, "none")
    off = torch.full((E + 1,), start, dtype=torch.int32, device="cuda")
    tok = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    y = torch.full((n, N), float("nan"), dtype=BF16, device="cuda")
    dense.GroupedMm(x=xq, x_scales=xs, w=w, w_scales=ws, expert_offset=off, sorted_tok=tok, top_k=1, y=y).run(stream())
    assert torch.equal(y, torch.zeros_like(y))


def test_one_group_without_routing():
    xq, xs, w, ws, xv = operands(3, 1, 77, 256, 104, "none")
    y = torch.empty((77, 104), device="cuda")
    dense.GroupedMm(x=xq, x_scales=xs, w=w, w_scales=ws, y=y).run(stream())
    tok, off = torch.arange(77, dtype=torch.int32, device="cuda"), torch.tensor([0, 77], dtype=torch.int32, device="cuda")
    close(y, *plain(xv, values_of(w, ws, 104), tok, off, 0, "none", 104), F32)


@pytest.mark.parametrize("K", [64, 256])
def test_all_units_past_the_table(K):
    """More units a CTA than its table holds, in the narrow form (K 64) and the wide one: 40,000 rows of one expert over a wide
    output; rows repeat, and so do results."""
    n, N = 40000, 16384
    g = gen(4)
    xq16, xs16, w, ws, xv = operands(4, 1, 16, K, N, "none")
    pick = torch.randint(0, 16, (n,), generator=g, device="cuda")
    xq, xs = dense.f8_empty(n, K)
    xq.view(torch.uint8).copy_(xq16.view(torch.uint8)[pick])
    xs.copy_(xs16[pick])
    y = torch.empty((n, N), dtype=F16, device="cuda")
    dense.GroupedMm(x=xq, x_scales=xs, w=w, w_scales=ws, y=y).run(stream())
    tok, off = torch.arange(16, dtype=torch.int32, device="cuda"), torch.tensor([0, 16], dtype=torch.int32, device="cuda")
    want, tol = plain(xv, values_of(w, ws, N), tok, off, 0, "none", N)
    first = torch.stack([y[(pick == i).nonzero()[0, 0]] for i in range(16)])
    close(first, want, tol, F16)
    for r in range(0, n, 5000):
        assert torch.equal(y[r:r + 5000], first[pick[r:r + 5000]])


@pytest.mark.parametrize("rows,N", [(3, 32), (2100, 2048)])
def test_offsets_past_32_bits(rows, N):
    """Experts, input rows and output rows that lie over 4 GiB into their tensors, in the split and the wide form."""
    K, far = 128, 4_600_000_000
    xq, xs, w, ws, xv = operands(6, 2, rows, K, N, "none")
    wbuf = torch.empty(far + N * K, dtype=torch.uint8, device="cuda")
    wf = torch.as_strided(wbuf, (2, N, K), (far, K, 1))
    wf.copy_(w.view(torch.uint8))
    pitch = 4_800_000_000 // rows // 16 * 16
    xbuf = torch.empty((rows - 1) * pitch + K, dtype=torch.uint8, device="cuda")
    x = torch.as_strided(xbuf, (rows, K), (pitch, 1))
    x.copy_(xq.view(torch.uint8))
    ybuf = torch.empty((rows - 1) * (pitch // 2) + N, dtype=F16, device="cuda")
    y = torch.as_strided(ybuf, (rows, N), (pitch // 2, 1))
    tok = torch.randperm(rows, generator=gen(2), device="cuda").to(torch.int32)
    off = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device="cuda")
    dense.GroupedMm(x=x.view(F8), x_scales=xs, w=wf.view(F8), w_scales=ws, y=y, expert_offset=off, sorted_tok=tok,
                    top_k=1).run(stream())
    close(y, *plain(xv, values_of(w, ws, N), tok, off, 1, "none", N), F16)


def test_repeats_to_the_bit_on_streams_and_in_graphs():
    for counts, K, N in FORMS.values():
        y, plan, _, _ = case(12, counts, K, N, "silu_mul", out=BF16)
        ref = y.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y.zero_()
            plan.run()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(y, ref)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run(stream())
        for _ in range(3):
            y.zero_()
            graph.replay()
            assert torch.equal(y, ref)


@pytest.mark.parametrize("K", [1 << 26, (1 << 26) - 16])
def test_the_longest_k(K):
    """A row of zeros but for a few ones, times small whole numbers, scales powers of two: the sum is exact in f32."""
    g = gen(1)
    at = torch.tensor([0, 1, 127, 128, K // 2, K - 129, K - 128, K - 17, K - 1], device="cuda")
    w = torch.randint(-8, 9, (1, 8, K), generator=g, device="cuda", dtype=torch.int8).to(F8)
    kb = -(-K // 128)
    ws = torch.exp2(torch.randint(-3, 4, (1, 1, kb), generator=g, device="cuda").float())
    xq, xs = dense.f8_empty(1, K)
    xq.zero_()
    xs.copy_(torch.exp2(torch.randint(-3, 4, (1, kb), generator=g, device="cuda").float()))
    xq[0, at] = torch.ones(len(at), device="cuda").to(F8)
    y = torch.empty((1, 8), device="cuda")
    dense.GroupedMm(x=xq, x_scales=xs, w=w, w_scales=ws, y=y).run(stream())
    want = (w[0][:, at].double() * (ws[0, 0, at // 128] * xs[0, at // 128]).double()).sum(1)
    assert torch.equal(y[0].double(), want)


def test_a_layer_of_fp8_experts():
    """Router with groups, FP8 rows, gate and up, FP8 rows, down, the weighted sum: the steps as a layer takes them, against
    the same steps in 64 bits on what each of them was given."""
    T, E, k, H, W = 75, 32, 4, 512, 256
    g = gen(21)
    x, logits, bias = randn(g, T, H, dtype=BF16), randn(g, T, E), 0.1 * randn(g, E)
    _, _, gu, gus, _ = operands(22, E, 1, H, W, "silu_mul")
    _, _, dn, dns, _ = operands(23, E, 1, W, H, "none")
    P = T * k
    ids, w = torch.empty((T, k), dtype=torch.int32, device="cuda"), torch.empty((T, k), device="cuda")
    tok, off = torch.empty(P, dtype=torch.int32, device="cuda"), torch.empty(E + 1, dtype=torch.int32, device="cuda")
    (xq, xs), (hq, hs) = dense.f8_empty(T, H), dense.f8_empty(P, W)
    h, y = torch.empty((P, W), dtype=BF16, device="cuda"), torch.empty((P, H), dtype=BF16, device="cuda")
    out = torch.empty((T, H), device="cuda")
    work = torch.empty(dense.native().gather_work_bytes(T, k), dtype=torch.uint8, device="cuda")
    router = dense.Router(logits=logits, top_k=k, ids=ids, w=w, score="sigmoid", bias=bias, groups=8, keep_groups=3, group_top=2,
                          renorm=True, scale=2.5, sorted_tok=tok, expert_offset=off)
    up = dense.GroupedMm(x=xq, x_scales=xs, w=gu, w_scales=gus, expert_offset=off, sorted_tok=tok, top_k=k, act="silu_mul", y=h)
    down = dense.GroupedMm(x=hq, x_scales=hs, w=dn, w_scales=dns, expert_offset=off, sorted_tok=tok, y=y)

    def layer():
        router.run()
        dense.f8_quantize(x, xq, xs)
        up.run()
        dense.f8_quantize(h, hq, hs)
        down.run()
        dense.native().moe_gather(y.data_ptr(), H, tok.data_ptr(), P, w.data_ptr(), T, k, H, out.data_ptr(), work.data_ptr(), stream())

    layer()
    spread = lambda q, s: q.double() * s.double()[:, torch.arange(q.shape[1], device="cuda") // 128]  # noqa: E731
    gv, dv = values_of(gu, gus, W), values_of(dn, dns, H)
    close(h, *plain(spread(xq, xs), gv, tok, off, k, "silu_mul", W), BF16)
    close(y, *plain(spread(hq, hs), dv, tok, off, 0, "none", H), BF16)
    place = torch.empty(P, dtype=torch.long, device="cuda")
    place[tok.long()] = torch.arange(P, device="cuda")
    rows = y.double()[place].view(T, k, H) * w.double()[..., None]
    assert bool(((out.double() - rows.sum(1)).abs() <= 2 * k * 2.0 ** -24 * rows.abs().sum(1)).all())
    # what the codes lose: each x within half a step of its value, 2^-4 of it, or of the smallest step, 2^-10 scales
    lost = x.double().abs() * 2.0 ** -4 + spread(torch.ones_like(x), xs) * 2.0 ** -10
    close(h, *plain(x.double(), gv, tok, off, k, "silu_mul", W, lost), BF16)
    graph = torch.cuda.CUDAGraph()
    keep = out.clone()
    with torch.cuda.graph(graph):
        layer()
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, keep)


def test_f8_products_refuse():
    xq, xs, w, ws, _ = operands(1, 2, 4, 256, 32, "none")
    off, y = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.full((4, 32), 5.0, dtype=F16, device="cuda")
    kw = dict(x=xq, x_scales=xs, w=w, w_scales=ws, expert_offset=off, y=y)
    for bad in (dict(x_scales=None), dict(w_scales=None), dict(x_scales=xs[:, :1]), dict(w_scales=ws[:, :, :1]),
                dict(w_scales=ws.double()), dict(x_scales=xs.half()), dict(x=xq.view(torch.uint8)), dict(act="silu_mul"),
                dict(w_scales=torch.cat((ws, ws), 1)[:, ::2]), dict(x=xq.view(torch.float8_e5m2))):
        with pytest.raises(ValueError):
            dense.GroupedMm(**{**kw, **bad})
    with pytest.raises(RuntimeError):
        dense.GroupedMm(**{**kw, "y": torch.empty((4, 16), dtype=torch.uint8, device="cuda"),
                           "y_scales": torch.empty((4, 1), dtype=torch.uint8, device="cuda")}).run()
    assert (y == 5).all()


@pytest.mark.parametrize("routed", [False, True, "masked"])
@pytest.mark.parametrize("T", [1, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_an_fp8_block_is_its_entries(T, dtype, routed):
    """The residual block over FP8 experts, with its own router, with grouped routing, and with a bias that leaves a token fewer
    experts than slots, against the entries it is made of, to the bit; and in a graph."""
    E, H, W, k = 32, 528, 272, 4
    g = gen(T)
    t = {"router_w": randn(g, E, H, dtype=dtype) * H ** -0.5, "pre_w": randn(g, H, dtype=dtype), "post_w": randn(g, H, dtype=dtype),
         "gate": randn(g, H, dtype=dtype), "next_w": randn(g, H, dtype=dtype)}
    _, _, t["gu_w"], t["gu_scales"], _ = operands(1, E, 1, H, W, "silu_mul")
    _, _, t["dn_w"], t["dn_scales"], _ = operands(2, E, 1, W, H, "none")
    routing = dict(score="sigmoid", bias=0.1 * randn(g, E), groups=8, keep_groups=3, group_top=2, renorm=True, scale=2.5)
    if routed == "masked":
        routing["bias"][2:] = -float("inf")
    block = dense.ExpertBlock(top_k=k, res_scale=0.5, max_tokens=300, router=routing if routed else None, **t)
    x = randn(g, T, H, dtype=dtype)
    out, nxt = torch.empty_like(x), torch.empty_like(x)
    block.forward(x, out, nxt)
    new = lambda *s, dt=dtype: torch.empty(s, dtype=dt, device="cuda")  # noqa: E731
    P, nat = T * k, dense.native()
    xn, logits, h, rows = new(T, H), new(T, E, dt=F32), new(P, W), new(P, H, dt=BF16)
    ids, w, tok, off = new(T, k, dt=torch.int32), new(T, k, dt=F32), new(P, dt=torch.int32), new(E + 1, dt=torch.int32)
    dense.BlockNorm(res=x, pre_w=t["pre_w"], y=xn).run()
    dense.GroupedMm(x=xn, w=t["router_w"][None], y=logits).run()
    if routed:
        dense.Router(logits=logits, top_k=k, ids=ids, w=w, sorted_tok=tok, expert_offset=off, **routing).run()
        assert routed != "masked" or ((ids[:, 2:] == -1).all() and (ids[:, :2] >= 0).all() and (tok == -1).sum() == 2 * T)
    else:
        work = new(nat.scatter_work_bytes(P, E), dt=torch.uint8)
        nat.router_scatter(logits.data_ptr(), T, E, k, ids.data_ptr(), w.data_ptr(), E, 0, tok.data_ptr(), off.data_ptr(),
                           work.data_ptr(), stream())
    (xq, xs), (hq, hs) = dense.f8_empty(T, H), dense.f8_empty(P, W)
    dense.f8_quantize(xn, xq, xs)
    dense.GroupedMm(x=xq, x_scales=xs, w=t["gu_w"], w_scales=t["gu_scales"], expert_offset=off, sorted_tok=tok, top_k=k,
                    act="silu_mul", y=h).run()
    dense.f8_quantize(h, hq, hs)
    dense.GroupedMm(x=hq, x_scales=hs, w=t["dn_w"], w_scales=t["dn_scales"], expert_offset=off, sorted_tok=tok, y=rows).run()
    branch, gw = new(T, H, dt=F32), new(nat.gather_work_bytes(T, k), dt=torch.uint8)
    nat.moe_gather(rows.data_ptr(), H, tok.data_ptr(), P, w.data_ptr(), T, k, H, branch.data_ptr(), gw.data_ptr(), stream())
    want, want_next = torch.empty_like(x), torch.empty_like(x)
    dense.BlockNorm(branch=branch, post_w=t["post_w"], gate=t["gate"], gate_kind="channel", res=x, res_scale=0.5, out=want,
                    pre_w=t["next_w"], y=want_next).run()
    assert torch.equal(out, want) and torch.equal(nxt, want_next)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.forward(x, out, nxt)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)


def test_a_block_refuses_a_router_that_does_not_fit():
    _, _, gu, gus, _ = operands(1, 16, 1, 64, 32, "silu_mul")
    _, _, dn, dns, _ = operands(2, 16, 1, 32, 64, "none")
    one = torch.ones(64, dtype=BF16, device="cuda")
    t = dict(router_w=torch.zeros((16, 64), dtype=BF16, device="cuda"), gu_w=gu, gu_scales=gus, dn_w=dn, dn_scales=dns, pre_w=one,
             top_k=4, max_tokens=8)
    x = torch.zeros((8, 64), dtype=BF16, device="cuda")
    out = torch.full_like(x, 5)
    for bad in (dict(groups=3), dict(groups=8, keep_groups=1), dict(scale=float("inf"))):
        with pytest.raises(RuntimeError):
            dense.ExpertBlock(**t, router=bad).forward(x, out)
    assert (out == 5).all()
    for bad in (dict(router=dict(top=1)), dict(router=dict(bias=one)), dict(gu_scales=gus[:, :1]), dict(dn_scales=dns.double()),
                dict(dn_w=dn.view(torch.uint8))):
        with pytest.raises(ValueError):
            dense.ExpertBlock(**{**t, **bad})


@pytest.mark.parametrize("T,pad", [(1, 7), (40, 65), (300, 900)])
def test_beside_exl3_experts_in_one_buffer(T, pad):
    """Trailing experts in FP8 behind a layer's EXL3 ones: grouped_mm over their part of the offsets, which clears the rows
    before them, then the EXL3 ops over their live rows alone, which leave the others."""
    from exl3b200 import load_plugin
    from exl3b200.layer import MoeLayer
    lay = MoeLayer(load_plugin(), n_expert=16, hidden=2048, width=512, top_k=4, bits_gu=3, bits_dn=4, max_tokens=T, seed=3,
                   max_rows=T * 4 + pad)
    R, K, H, g = T * lay.k, 512, lay.H, gen(4)
    lay.x.copy_(randn(g, *lay.x.shape, dtype=F16))
    lay.logits.copy_(randn(g, *lay.logits.shape))
    n = R + pad
    lay.forward(T, stream())
    lay.experts(T, n, stream(), live=True)    # alone, over as many rows: their number chooses the ops' form
    torch.cuda.synchronize()
    want = lay.y_rows[:R].view(torch.int16).clone()
    off = torch.tensor([R, R + pad // 3, n], dtype=torch.int32, device="cuda")
    y = lay.y_rows[:n].view(BF16)
    xq, xs, w, ws, xv = operands(5, 2, n, K, H, "none")
    dense.GroupedMm(x=xq, x_scales=xs, w=w, w_scales=ws, expert_offset=off, y=y).run(stream())
    alone = y[R:].clone()
    rows = torch.arange(n, dtype=torch.int32, device="cuda")
    close(y, *plain(xv, values_of(w, ws, H), rows, off, 0, "none", H), BF16)
    assert not y[:R].any()
    lay.experts(T, n, stream(), live=True)
    torch.cuda.synchronize()
    assert torch.equal(y[R:], alone) and torch.equal(lay.y_rows[:R].view(torch.int16), want)
