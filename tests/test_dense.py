"""grouped_mm, block_norm and the MXFP4 conversions on a GPU, against plain implementations in 64 bits.

Tolerances, from the arithmetic alone:
- A product sums K exact products of 8- or 11-bit significands (MXFP4: 4-bit ones, scaled by powers of two) in f32. Any
  order of K rounded or truncated additions is within K * 2^-23 * sum |x w| of the sum; an output type of p bits adds
  2^-p of the value. silu_mul carries the two sums' errors through |silu'| <= 1.1 and |silu(g)| <= |g|, and its own f32
  arithmetic (an approximate exponential and a division) adds 2^-19 of the value.
- block_norm's sums run over at most 32 values a thread, then two trees: relative 2^-17 covers each norm with its root,
  and every output is rounded once. The error of r is relative to |res_scale res| + |g n|.
- MXFP4 values are exact: compared bit for bit."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ULP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}      # half of the last place at the bottom of the range


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()
    assert dense.native().read_error() == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def stream():
    return torch.cuda.current_stream().cuda_stream


def padded(t, extra, fill=float("nan")):
    """t as a view of rows `extra` elements longer, the rest filled."""
    big = torch.full((*t.shape[:-1], t.shape[-1] + extra), fill if t.dtype.is_floating_point else 0xEE, dtype=t.dtype,
                     device=t.device)
    big[..., :t.shape[-1]] = t
    return big[..., :t.shape[-1]], big


# ------------------------------------------------------------------------------------------------ MXFP4
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def mx4_plain(x):
    """(values, scale bytes) by the definition, in numpy's 64 bits; x [rows, cols]."""
    b = x.double().cpu().numpy().reshape(x.shape[0], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    a = np.abs(np.where(np.isfinite(b), b, 0))
    top = a.max(-1)
    e = np.where(top > 0, np.frexp(top)[1] - 1 - 2, -127)
    e = np.maximum(e, -127)
    r = a / np.ldexp(1.0, e)[..., None]
    d = np.abs(r[..., None] - GRID)
    even = np.array([0, 1, 0, 1, 0, 1, 0, 1]) * 1e-9             # a tie goes to the even mantissa
    v = GRID[np.argmin(d + even, -1)]
    v = np.where(r >= 6, 6.0, v) * np.ldexp(1.0, e)[..., None] * np.where(np.signbit(b), -1, 1)
    v[bad] = np.nan
    code = np.where(bad, 255, e + 127)
    return v.reshape(x.shape), code.astype(np.uint8)


def decode(codes, scales):
    c = codes.cpu().numpy()
    n = np.stack((c & 15, c >> 4), -1).reshape(*c.shape[:-1], -1)
    v = GRID[n & 7] * np.where(n > 7, -1, 1)
    s = scales.cpu().numpy().astype(np.int64)
    f = np.where(s == 255, np.nan, np.ldexp(1.0, np.where(s == 255, 0, s - 127)))
    return v * np.repeat(f, 32, -1)


@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 64), (3, 96), (5, 2048), (64, 2080), (700, 4096)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_quantize_is_exact(rows, cols, dtype):
    g = gen(rows * 7 + cols)
    x = randn(g, rows, cols) * torch.exp2(torch.randint(-12, 12, (rows, cols // 32, 1), generator=g, device="cuda").float()
                                          ).expand(-1, -1, 32).reshape(rows, cols)
    # multiples of an eighth of each block's scale: every midpoint of the grid among them
    x[:, ::2] = torch.round(x[:, ::2] * 8) / 8
    x, _ = padded(x.to(dtype), 8)
    codes, cbig = padded(torch.zeros((rows, cols // 2), dtype=torch.uint8, device="cuda"), 16)
    scales, sbig = padded(torch.zeros((rows, cols // 32), dtype=torch.uint8, device="cuda"), 3)
    dense.mx4_quantize(x, codes, scales, stream())
    want, code = mx4_plain(x)
    assert np.array_equal(scales.cpu().numpy(), code)
    assert np.array_equal(decode(codes, scales), want)
    assert (cbig[:, cols // 2:] == 0xEE).all() and (sbig[:, cols // 32:] == 0xEE).all()
    for out in (F32, F16, BF16):
        y = dense.mx4_dequantize(codes, scales, torch.empty((rows, cols), dtype=out, device="cuda"), stream())
        assert torch.equal(y, torch.from_numpy(want).cuda().to(out))


def test_quantize_midpoints_saturation_and_special_values():
    x = torch.zeros((9, 32))
    mids = torch.tensor([0., .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.99])
    for row, f in ((0, 1.0), (1, 2.0 ** 40), (2, 2.0 ** -100)):
        x[row, :17], x[row, 17:32] = mids * f, -mids[:15] * f
    x[3, 0] = 2.0 ** -126                       # the smallest normal: its scale is below the range, 2^-127 serves
    x[4, 0] = 2.0 ** -149
    x[5, 0], x[5, 1] = float("inf"), 1.0
    x[6, 31], x[6, 0] = float("nan"), 1.0
    x[7, 3] = torch.finfo(F32).max
    x[8, 5], x[8, 6] = -torch.finfo(F32).max, -0.0
    x = x.cuda()
    codes, scales = dense.mx4_empty(9, 32)
    dense.mx4_quantize(x, codes, scales, stream())
    want, code = mx4_plain(x)
    assert np.array_equal(scales.cpu().numpy(), code)
    assert scales[5, 0] == 255 and scales[6, 0] == 255 and not codes[5:7].any()
    assert np.array_equal(decode(codes, scales), want, equal_nan=True)


def test_dequantize_every_code_and_scale():
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").reshape(16, 16).repeat(16, 1)     # 256 rows of 32
    scales = torch.arange(256, dtype=torch.uint8, device="cuda").reshape(256, 1)
    y = dense.mx4_dequantize(codes, scales, torch.empty((256, 32), device="cuda"), stream())
    want = decode(codes, scales)
    assert np.array_equal(y.double().cpu().numpy(), want.astype(np.float32).astype(np.float64), equal_nan=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_dequantize_every_code_and_scale_rounds_once(dtype):
    """Below the type's range the values round (to nearest, ties to even), above it they are infinite. A code has two
    significant bits: 64 bits, then 32, then the type round no differently from 64 bits to the type at once."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").reshape(16, 16).repeat(16, 1)
    scales = torch.arange(256, dtype=torch.uint8, device="cuda").reshape(256, 1)
    y = dense.mx4_dequantize(codes, scales, torch.empty((256, 32), dtype=dtype, device="cuda"), stream())
    want = torch.from_numpy(decode(codes, scales)).cuda().to(F32).to(dtype)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.nan_to_num(y), torch.nan_to_num(want))


def test_quantize_of_no_rows_and_refusals():
    n, u8 = dense.native(), torch.uint8
    x = torch.zeros((4, 64), device="cuda")
    codes, scales = dense.mx4_empty(4, 64)
    dense.mx4_quantize(x[:0], codes[:0], scales[:0], stream())
    args = dict(x=x.data_ptr(), dt=1, xp=64, rows=4, cols=64, c=codes.data_ptr(), cp=32, s=scales.data_ptr(), sp=2)

    def call(**k):
        a = dict(args, **k)
        return n.lib.exl3b200_mx4_quantize(a["x"], a["dt"], a["xp"], a["rows"], a["cols"], a["c"], a["cp"], a["s"], a["sp"],
                                           stream())
    assert call() == 0
    for want, k in ((-1, dict(cols=48)), (-1, dict(rows=-1)), (-1, dict(cols=0)), (-2, dict(dt=9)), (-12, dict(x=0)),
                    (-12, dict(s=0)), (-4, dict(xp=32)), (-4, dict(cp=31)), (-4, dict(sp=1)),
                    (-3, dict(x=x.data_ptr() + 4)), (-3, dict(c=codes.data_ptr() + 1)), (-3, dict(xp=66))):
        assert call(**k) == want, k
    assert n.lib.exl3b200_mx4_tiled_bytes(1, 7, 64, 1) == -1 and n.lib.exl3b200_mx4_tiled_bytes(1, 8, 48, 0) == -1
    with pytest.raises(ValueError):
        dense.mx4_quantize(x, codes, scales.t().contiguous().t(), stream())


# ------------------------------------------------------------------------------------------------ grouped_mm
def routing(counts, before=0, after=0, dropped=(), top_k=1, g=None):
    """sorted_tok over a shuffled slot order, expert_offset starting at `before`; `dropped` rows carry -1."""
    live = sum(counts)
    n = before + live + after
    tok = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    off = torch.tensor(np.cumsum([before, *counts]), dtype=torch.int32, device="cuda")
    for i in dropped:
        tok[i] = -1
    return tok, off, n


def plain(x, w, tok, off, top_k, act, n_out):
    """(y, its tolerance without the output type's) in 64 bits."""
    n, E = tok.numel(), w.shape[0]
    y = torch.zeros((n, n_out), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(y)
    K = x.shape[1]
    o = off.tolist()
    for e in range(E):
        rows = torch.arange(o[e], o[e + 1], device="cuda")
        rows = rows[tok[rows] >= 0]
        if not rows.numel():
            continue
        xe = x[(tok[rows].long() // top_k) if top_k else rows].double()
        we = w[e].double()
        z, s = xe @ we.T, xe.abs() @ we.abs().T * (K * 2.0 ** -23)
        if act == "none":
            y[rows], tol[rows] = z, s
        else:
            g, u, sg, su = z[:, :n_out], z[:, n_out:], s[:, :n_out], s[:, n_out:]
            v = g * torch.sigmoid(g) * u
            y[rows] = v
            tol[rows] = 1.1 * sg * (u.abs() + su) + (g.abs() + sg) * su + 2.0 ** -19 * v.abs()
    return y, tol


def close(got, want, tol, dtype):
    err = (got.double() - want).abs()
    bound = tol + ULP[dtype] * (want.abs() + tol) + TINY[dtype]
    worst = float((err / bound.clamp_min(1e-300)).max()) if err.numel() else 0.0
    assert bool((err <= bound).all()), worst


def counts_of(kind, g):
    return {"one": [1], "empty": [0, 0, 3, 0], "few": [1, 0, 2, 1, 0, 5], "ragged": [17, 0, 33, 129, 16, 1, 64],
            "large": [300, 0, 515], "many": torch.randint(0, 4, (300,), generator=g, device="cuda").tolist()}[kind]


def case_tensors(kind, K, N, act, dtype, top_k, seed, before=0, after=0, dropped=()):
    g = gen(seed)
    counts = counts_of(kind, g)
    tok, off, n = routing(counts, before, after, dropped, g=g)
    x_rows = n if top_k == 0 else (n + top_k - 1) // top_k
    wn = N * (2 if act == "silu_mul" else 1)
    x = randn(g, x_rows, K, dtype=dtype if dtype != "mx4" else F32)
    w = randn(g, len(counts), wn, K) * (K ** -0.5)
    return x, (w if dtype == "mx4" else w.to(dtype)), tok, off, n


def mx4_of(x):
    q, s = dense.mx4_empty(x[..., 0].numel(), x.shape[-1])
    dense.mx4_quantize(x.reshape(-1, x.shape[-1]).contiguous(), q, s, stream())
    v = torch.from_numpy(decode(q, s)).cuda().reshape(x.shape)
    return q.reshape(*x.shape[:-1], -1), s.reshape(*x.shape[:-1], -1), v


@pytest.mark.parametrize("kind", ["one", "empty", "few", "ragged", "large", "many"])
@pytest.mark.parametrize("K,N", [(8, 8), (72, 40), (512, 200), (2048, 512), (640, 2560)])
@pytest.mark.parametrize("act", ["none", "silu_mul"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_grouped_mm(kind, K, N, act, dtype):
    top_k = {"one": 1, "few": 3, "ragged": 0}.get(kind, 2)
    x, w, tok, off, n = case_tensors(kind, K, N, act, dtype, top_k, K + N)
    want, tol = plain(x, w, tok, off, top_k, act, N)
    outs = {}
    for yd in (F32, dtype):
        y, ybig = padded(torch.zeros((n, N), dtype=yd, device="cuda"), 16, 7.0)
        y.fill_(float("nan"))
        dense.GroupedMm(x=x, w=w, y=y, expert_offset=off, sorted_tok=tok, top_k=top_k, act=act).run(stream())
        close(y, want, tol, yd)
        assert (ybig[:, N:] == 7).all()
        outs[yd] = y
    assert torch.equal(outs[F32].to(dtype), outs[dtype])            # the same sums, rounded once


@pytest.mark.parametrize("kind", ["one", "empty", "few", "ragged", "large", "many"])
@pytest.mark.parametrize("K,N", [(32, 8), (96, 40), (544, 200), (2048, 512), (640, 2560)])
@pytest.mark.parametrize("act", ["none", "silu_mul"])
def test_grouped_mm_mx4(kind, K, N, act):
    top_k = {"one": 1, "few": 3, "ragged": 0}.get(kind, 2)
    x, w, tok, off, n = case_tensors(kind, K, N, act, "mx4", top_k, K + N)
    xq, xs, xv = mx4_of(x)
    wq, ws, wv = mx4_of(w)
    want, tol = plain(xv, wv, tok, off, top_k, act, N)
    tiled = dense.mx4_tile_scales(ws, act)
    outs = {}
    for yd in (F32, F16, BF16):
        y = torch.full((n, N), float("nan"), dtype=yd, device="cuda")
        dense.GroupedMm(x=xq, x_scales=xs, w=wq, w_scales=tiled, y=y, expert_offset=off, sorted_tok=tok, top_k=top_k,
                        act=act).run(stream())
        close(y, want, tol, yd)
        outs[yd] = y
    assert torch.equal(outs[F32].to(F16), outs[F16]) and torch.equal(outs[F32].to(BF16), outs[BF16])


@pytest.mark.parametrize("dtype", [F16, "mx4"])
@pytest.mark.parametrize("kind", ["few", "ragged"])
@pytest.mark.parametrize("act", ["none", "silu_mul"])
def test_mx4_output_is_the_f32_output_quantised(dtype, kind, act):
    K, N = 256, 352
    x, w, tok, off, n = case_tensors(kind, K, N, act, dtype, 1, 5, before=3, after=9, dropped=(4, 6))
    kw = dict(expert_offset=off, sorted_tok=tok, top_k=1, act=act)
    if dtype == "mx4":
        xq, xs, _ = mx4_of(x)
        wq, ws, _ = mx4_of(w)
        kw |= dict(x=xq, x_scales=xs, w=wq, w_scales=dense.mx4_tile_scales(ws, act))
    else:
        kw |= dict(x=x, w=w)
    y = torch.empty((n, N), device="cuda")
    dense.GroupedMm(y=y, **kw).run(stream())
    want_q, want_s = dense.mx4_empty(n, N)
    dense.mx4_quantize(y, want_q, want_s, stream())
    q, qbig = padded(torch.zeros((n, N // 2), dtype=torch.uint8, device="cuda"), 16)
    s, sbig = padded(torch.zeros((n, N // 32), dtype=torch.uint8, device="cuda"), 5)
    q.fill_(0x11)
    s.fill_(0x11)
    dense.GroupedMm(y=q, y_scales=s, **kw).run(stream())
    assert torch.equal(s, want_s) and np.array_equal(decode(q, s), decode(want_q, want_s))
    assert (qbig[:, N // 2:] == 0xEE).all() and (sbig[:, N // 32:] == 0xEE).all()


@pytest.mark.parametrize("dtype", [BF16, "mx4"])
def test_rows_outside_the_runs_dropped_slots_and_poison(dtype):
    """Rows before, after and dropped are zero; NaN in rows, weights and padding that no live row reads stays there."""
    K, N, before, after = 192, 136, 5, 40
    dropped = (7, 20, 21)
    x, w, tok, off, n = case_tensors("ragged", K, N, "silu_mul", dtype, 1, 9, before, after, dropped)
    live = torch.zeros(n, dtype=torch.bool, device="cuda")
    live[before:n - after] = True
    live[list(dropped)] = False
    x[tok[~live & (tok >= 0)].long()] = float("nan")
    w[1] = float("inf")                                             # the expert without rows
    if dtype == "mx4":
        xq, xs, xv = mx4_of(x)
        wq, ws, wv = mx4_of(w)
        kw = dict(x=xq, x_scales=xs, w=wq, w_scales=dense.mx4_tile_scales(ws, "silu_mul"))
    else:
        xv, wv = x, w
        kw = dict(x=padded(x, 24)[0], w=padded(w, 8)[0])
    want, tol = plain(torch.where(torch.isnan(xv), 0, xv), torch.where(torch.isfinite(wv), wv, 0), tok,
                      off, 1, "silu_mul", N)
    y = torch.full((n, N), float("nan"), dtype=BF16, device="cuda")
    dense.GroupedMm(y=y, expert_offset=off, sorted_tok=tok, top_k=1, act="silu_mul", **kw).run(stream())
    want[~live], tol[~live] = 0, 0
    assert not y[~live].any() and torch.isfinite(y).all()
    close(y, want, tol, BF16)
    # a NaN in one live row is that row's alone
    r = int(tok[before + 30])
    assert r >= 0
    if dtype == "mx4":
        xs[r, 2] = 255
    else:
        kw["x"][r, 3] = float("nan")
    y2 = torch.empty_like(y)
    dense.GroupedMm(y=y2, expert_offset=off, sorted_tok=tok, top_k=1, act="silu_mul", **kw).run(stream())
    assert torch.isnan(y2[before + 30]).all()
    y[before + 30] = y2[before + 30] = 0
    assert torch.equal(y, y2)


@pytest.mark.parametrize("dtype", [F16, "mx4"])
def test_one_group_without_routing(dtype):
    g = gen(3)
    x, w = randn(g, 77, 256), randn(g, 1, 104, 256) * 0.06
    if dtype == "mx4":
        (x, xs, xv), (w, ws, wv) = mx4_of(x), mx4_of(w)
        kw = dict(x_scales=xs, w_scales=dense.mx4_tile_scales(ws))
    else:
        x, w = x.to(F16), w.to(F16)
        xv, wv, kw = x, w, {}
    y = torch.empty((77, 104), device="cuda")
    dense.GroupedMm(x=x, w=w, y=y, **kw).run(stream())
    off = torch.tensor([0, 77], dtype=torch.int32, device="cuda")
    want, tol = plain(xv, wv, torch.arange(77, device="cuda"), off, 0, "none", 104)
    close(y, want, tol, F32)


def test_many_groups_of_one_expert_and_all_units_past_the_table():
    """More units a CTA than its table holds: 40,000 rows of one expert over a wide output."""
    g = gen(4)
    n, K, N = 40000, 64, 16384
    x, w = randn(g, n, K, dtype=F16), randn(g, 1, N, K, dtype=F16)
    y = torch.empty((n, N), dtype=F16, device="cuda")
    dense.GroupedMm(x=x, w=w, y=y).run(stream())
    for r in (0, 12345, n - 1):
        z = x[r].double() @ w[0].double().T
        s = x[r].double().abs() @ w[0].double().abs().T
        close(y[r], z, K * 2.0 ** -23 * s, F16)
    z = x.double() @ w[0, N - 3].double()
    close(y[:, N - 3], z, K * 2.0 ** -23 * (x.double().abs() @ w[0, N - 3].double().abs()), F16)


def test_offsets_past_32_bits():
    """Experts, input rows and output rows that lie over 4 GiB into their tensors."""
    g = gen(6)
    K, N, far = 64, 32, 2_300_000_000
    wbuf = torch.empty(far + N * K, dtype=F16, device="cuda")
    w = torch.as_strided(wbuf, (2, N, K), (far, K, 1))
    w.copy_(randn(g, 2, N, K))
    pitch = 1_200_000_008
    xbuf = torch.empty(2 * pitch + K, dtype=F16, device="cuda")
    x = torch.as_strided(xbuf, (3, K), (pitch, 1))
    x.copy_(randn(g, 3, K))
    ybuf = torch.empty(2 * pitch + N, dtype=F16, device="cuda")
    y = torch.as_strided(ybuf, (3, N), (pitch, 1))
    tok = torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda")
    off = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    dense.GroupedMm(x=x, w=w, y=y, expert_offset=off, sorted_tok=tok, top_k=1).run(stream())
    want, tol = plain(x, w, tok, off, 1, "none", N)
    close(y, want, tol, F16)


def test_grouped_mm_repeats_to_the_bit_on_streams_and_in_graphs():
    x, w, tok, off, n = case_tensors("ragged", 320, 264, "silu_mul", BF16, 2, 12)
    y = torch.empty((n, 264), dtype=BF16, device="cuda")
    plan = dense.GroupedMm(x=x, w=w, y=y, expert_offset=off, sorted_tok=tok, top_k=2, act="silu_mul")
    plan.run(stream())
    ref = y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y.zero_()
        plan.run(side.cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(stream())
    for _ in range(3):
        y.zero_()
        graph.replay()
        assert torch.equal(y, ref)


def test_grouped_mm_refusals():
    x, w = torch.zeros((4, 64), dtype=F16, device="cuda"), torch.zeros((2, 32, 64), dtype=F16, device="cuda")
    off, y = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.full((4, 32), 5.0, dtype=F16, device="cuda")
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    lib = dense.native().lib

    def status(**k):
        plan = dense.GroupedMm(x=x, w=w, y=y, expert_offset=off, sorted_tok=tok, top_k=1)
        for name, v in k.items():
            setattr(plan.desc, name, v)
        return lib.exl3b200_grouped_mm(plan._addr, stream())
    for want, k in ((-2, dict(dtype=1)), (-2, dict(y_dtype=11)), (-12, dict(act=2)), (-1, dict(n_expert=0)),
                    (-1, dict(n_expert=2049)), (-1, dict(n_rows=-1)), (-1, dict(n_in=60)), (-1, dict(n_out=4)),
                    (-1, dict(top_k=-1)), (-1, dict(top_k=0, x_rows=3)), (-1, dict(x_rows=0)), (-12, dict(x=0)),
                    (-12, dict(w=0)), (-12, dict(y=0)), (-12, dict(expert_offset=0)), (-12, dict(dtype=dense.MX4)),
                    (-1, dict(y_dtype=dense.MX4, n_out=40)), (-12, dict(y_dtype=dense.MX4)), (-4, dict(x_pitch=56)),
                    (-4, dict(w_pitch=32)), (-4, dict(y_pitch=24)), (-4, dict(w_expert_pitch=64)),
                    (-3, dict(x=x.data_ptr() + 2)), (-3, dict(x_pitch=66)), (-3, dict(y=y.data_ptr() + 8)),
                    (-3, dict(y_pitch=36)), (-1, dict(n_rows=1 << 30, n_out=1 << 29))):
        assert status(**k) == want, k
    assert lib.exl3b200_grouped_mm(None, stream()) == -12
    assert status(n_rows=0) == 0
    torch.cuda.synchronize()
    assert (y == 5).all()
    with pytest.raises(ValueError):
        dense.GroupedMm(x=x.to(BF16), w=w, y=y, expert_offset=off)
    with pytest.raises(ValueError):
        dense.GroupedMm(x=x, w=w, y=y, expert_offset=off[:2])
    with pytest.raises(ValueError):
        dense.GroupedMm(x=x.t().contiguous().t(), w=w, y=y, expert_offset=off)


# ------------------------------------------------------------------------------------------------ block_norm
def norm_plain(branch, post_w, gate, kind, res, rs, pre_w, eps):
    """(r, its scale, y, its scale) in 64 bits."""
    n = torch.zeros_like(res, dtype=torch.float64) if branch is None else branch.double()
    if post_w is not None:
        n = n / torch.sqrt((n * n).mean(1, keepdim=True) + eps) * post_w.double()
    if kind == "token":
        n = n * torch.sigmoid(gate.double())[:, None]
    elif kind == "channel":
        n = n * gate.double()
    elif kind == "element":
        n = n * torch.sigmoid(gate.double())
    base = res.double() * rs if res is not None else torch.zeros_like(n)
    r, size = base + n, base.abs() + n.abs()
    if pre_w is None:
        return r, size, None, None
    root = torch.sqrt((r * r).mean(1, keepdim=True) + eps)
    # y: r's own error over the root, and the root's, whose relative error is that of the sizes over it
    spread = (size * size).mean(1, keepdim=True).sqrt() / root
    w = pre_w.double()
    return r, size, r / root * w, (size / root + (r / root).abs() * spread) * w.abs()


def near(got, want, size, dtype):
    err = (got.double() - want).abs()
    bound = size * 2.0 ** -17 + ULP[dtype] * (want.abs() + size * 2.0 ** -17) + TINY[dtype]
    assert bool((err <= bound).all()), float((err / bound.clamp_min(1e-300)).max())


NORMS = [(1, 1), (3, 7), (2, 33), (5, 100), (1, 2048), (4, 2560), (130, 640), (9, 4096), (3, 8200), (2, 12001), (2, 32768)]


@pytest.mark.parametrize("T,H", NORMS)
@pytest.mark.parametrize("dtype,bd", [(BF16, F32), (F16, F16), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("kind", ["none", "token", "channel", "element"])
def test_block_norm(T, H, dtype, bd, kind):
    g = gen(T * 31 + H)
    branch, res = randn(g, T, H, dtype=bd) * 3, randn(g, T, H, dtype=dtype)
    post_w, pre_w = randn(g, H, dtype=dtype), randn(g, H, dtype=dtype)
    gate = {"none": lambda: None, "token": lambda: randn(g, T), "channel": lambda: randn(g, H, dtype=dtype),
            "element": lambda: randn(g, T, H, dtype=dtype)}[kind]()
    out, obig = padded(torch.zeros((T, H), dtype=dtype, device="cuda"), 3, 7.0)
    y = torch.full((T, H), float("nan"), dtype=dtype, device="cuda")
    dense.BlockNorm(branch=branch, post_w=post_w, post_eps=1e-5, gate=gate, gate_kind=kind, res=res, res_scale=0.5,
                    out=out, pre_w=pre_w, pre_eps=1e-5, y=y).run(stream())
    r, size, want, ysize = norm_plain(branch, post_w, gate, kind, res, 0.5, pre_w, 1e-5)
    near(out, r, size, dtype)
    near(y, want, ysize, dtype)
    assert (obig[:, H:] == 7).all()


@pytest.mark.parametrize("H", [8, 250, 2048])
def test_block_norm_parts_alone(H):
    g = gen(H)
    T, dt = 6, BF16
    branch, res, w = randn(g, T, H, dtype=dt), randn(g, T, H, dtype=dt), randn(g, H, dtype=dt)
    y = torch.empty((T, H), dtype=dt, device="cuda")
    # the norm before a block alone, on the stream and on a branch
    dense.BlockNorm(res=res, pre_w=w, pre_eps=1e-6, y=y).run(stream())
    r, size, want, ysize = norm_plain(None, None, None, "none", res, 1.0, w, 1e-6)
    near(y, want, ysize, dt)
    dense.BlockNorm(branch=branch, pre_w=w, pre_eps=1e-6, y=y).run(stream())
    near(y, *norm_plain(branch, None, None, "none", None, 1.0, w, 1e-6)[2:], dt)
    # a plain residual add, in place
    keep = res.clone()
    dense.BlockNorm(branch=branch, res=res, out=res).run(stream())
    near(res, keep.double() + branch.double(), keep.double().abs() + branch.double().abs(), dt)
    # in place, with the norm behind the block and the one before the next
    r, size, want, ysize = norm_plain(branch, w, None, "none", keep, 2.0, w, 1e-6)
    res.copy_(keep)
    dense.BlockNorm(branch=branch, post_w=w, res=res, res_scale=2.0, out=res, pre_w=w, y=y).run(stream())
    near(res, r, size, dt)
    near(y, want, ysize, dt)


def test_block_norm_zero_rows_infinities_and_nan():
    H, dt = 512, F16
    branch = torch.ones((5, H), dtype=dt, device="cuda")
    res, w = torch.ones((5, H), dtype=dt, device="cuda"), torch.ones(H, dtype=dt, device="cuda")
    branch[0], res[0] = 0, 0
    branch[1, 7] = float("nan")
    branch[2, 9] = float("inf")
    res[3, 1] = torch.finfo(dt).max
    gate = torch.tensor([0., 0., 0., float("-inf"), 200.], device="cuda")
    out, y = torch.empty_like(res), torch.empty_like(res)
    codes, scales = dense.mx4_empty(5, H)
    dense.BlockNorm(branch=branch, post_w=w, gate=gate, gate_kind="token", res=res, out=out, pre_w=w, y=y, y_codes=codes,
                    y_scales=scales).run(stream())
    assert not out[0].any() and not y[0].any() and not scales[0].any()
    assert torch.isnan(out[1]).all() and torch.isnan(y[1]).all() and (scales[1] == 255).all()
    assert torch.isnan(out[2, 9]) and torch.equal(out[2, :9], res[2, :9])        # inf / inf, and 1 / inf
    assert torch.equal(out[3], res[3]) and torch.isfinite(y[3]).all()            # a closed gate
    assert torch.equal(out[4], 2 * res[4])


@pytest.mark.parametrize("T,H", [(1, 32), (7, 96), (33, 2048), (3, 8224), (2, 32768)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_block_norm_mx4_is_its_f32_output_quantised(T, H, dtype):
    g = gen(H)
    branch, res = randn(g, T, H, dtype=dtype), randn(g, T, H, dtype=dtype)
    w = randn(g, H, dtype=dtype)
    codes, scales = dense.mx4_empty(T, H)
    y = torch.empty((T, H), dtype=dtype, device="cuda")
    kw = dict(branch=branch, post_w=w, res=res, pre_w=w, y=y)
    dense.BlockNorm(y_codes=codes, y_scales=scales, **kw).run(stream())
    alone, s2 = dense.mx4_empty(T, H)
    dense.BlockNorm(branch=branch, post_w=w, res=res, pre_w=w, y_codes=alone, y_scales=s2).run(stream())
    assert torch.equal(alone, codes) and torch.equal(s2, scales)
    if dtype == F32:
        want, s2 = dense.mx4_empty(T, H)
        dense.mx4_quantize(y, want, s2, stream())
        assert torch.equal(scales, s2) and torch.equal(codes, want)
    else:                                                            # of the f32 value, not of its rounded one
        v = torch.from_numpy(decode(codes, scales)).cuda()
        top = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
        assert bool(((v - y.double()).abs() <= top * 1.0 + (y.double().abs() - 6 * top).clamp_min(0) + 2 * ULP[dtype] * y.double().abs()).all())


def test_block_norm_refusals():
    x = torch.zeros((2, 64), dtype=BF16, device="cuda")
    w, out = torch.ones(64, dtype=BF16, device="cuda"), torch.full((2, 64), 5.0, dtype=BF16, device="cuda")
    codes, scales = dense.mx4_empty(2, 64)
    lib = dense.native().lib

    def status(**k):
        plan = dense.BlockNorm(branch=x, post_w=w, res=x, out=out, pre_w=w, y=out, y_codes=codes, y_scales=scales)
        for name, v in k.items():
            setattr(plan.desc, name, v)
        return lib.exl3b200_block_norm(plan._addr, stream())
    for want, k in ((-1, dict(rows=-1)), (-1, dict(cols=0)), (-1, dict(cols=32769)), (-2, dict(dtype=11)),
                    (-2, dict(branch_dtype=0)), (-12, dict(branch=0, res=0)), (-12, dict(branch=0)),
                    (-12, dict(out=0, y=0, y_codes=0, y_scales=0)), (-12, dict(pre_w=0)), (-12, dict(y=0, y_codes=0, y_scales=0)),
                    (-12, dict(y_scales=0)), (-12, dict(gate_kind=4)), (-12, dict(gate_kind=1)),
                    (-12, dict(gate=x.data_ptr())), (-12, dict(post_eps=-1.0)), (-12, dict(pre_eps=float("nan"))),
                    (-4, dict(branch_pitch=32)), (-4, dict(out_pitch=63)), (-4, dict(y_codes_pitch=31)),
                    (-4, dict(y_scales_pitch=1)), (-1, dict(cols=48)), (-3, dict(res=x.data_ptr() + 1)),
                    (-3, dict(res=x.data_ptr() + 2)), (-3, dict(y_codes=codes.data_ptr() + 2))):
        assert status(**k) == want, k
    assert lib.exl3b200_block_norm(None, stream()) == -12
    assert status(rows=0) == 0
    torch.cuda.synchronize()
    assert (out == 5).all()
    with pytest.raises(ValueError):
        dense.BlockNorm(branch=x, res=x.float(), out=x)
    with pytest.raises(ValueError):
        dense.BlockNorm(branch=x, res=x[:1], out=x)
    with pytest.raises(KeyError):
        dense.BlockNorm(branch=x, gate=w, gate_kind="row", out=x)


# ------------------------------------------------------------------------------------------------ forms, chains
# (counts, K, N): few units over a long k; a few rows an expert; hundreds of rows an expert in pairs of CTAs, in units cut
# short to fill the SMs and, over more outputs, in whole ones
FORMS = {"split": ([3, 0, 2], 1024, 96), "narrow": ([5, 0, 33, 1, 17, 12, 0, 0, 0, 0, 0, 0] * 9, 320, 352),
         "pair": ([600, 0, 715, 257], 320, 544), "wide": ([600, 0, 715, 257], 64, 4128)}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("act", ["none", "silu_mul"])
@pytest.mark.parametrize("dtype", [F16, BF16, "mx4"])
def test_every_form_and_output_with_dropped_slots(form, act, dtype):
    """Rows outside the runs on both sides, single dropped slots, a whole slice of them and an expert's all."""
    counts, K, N = FORMS[form]
    before, after = 70, 333
    g = gen(N)
    n = before + sum(counts) + after
    dropped = sorted({before, before + 3, n - after - 1} | set(range(before + 48, min(before + 70, n - after)))
                     | set(range(n - after - counts[-1], n - after)))
    tok, off, n = routing(counts, before, after, dropped, g=g)
    x, w = randn(g, n, K), randn(g, len(counts), N * (2 if act == "silu_mul" else 1), K) * K ** -0.5
    kw = dict(expert_offset=off, sorted_tok=tok, top_k=1, act=act)
    if dtype == "mx4":
        (xq, xs, xv), (wq, ws, wv) = mx4_of(x), mx4_of(w)
        kw |= dict(x=xq, x_scales=xs, w=wq, w_scales=dense.mx4_tile_scales(ws, act))
    else:
        xv, wv = x.to(dtype), w.to(dtype)
        kw |= dict(x=xv, w=wv)
    want, tol = plain(xv, wv, tok, off, 1, act, N)
    y32 = torch.full((n, N), float("nan"), device="cuda")
    dense.GroupedMm(y=y32, **kw).run(stream())
    close(y32, want, tol, F32)
    gone = (tok < 0) | (torch.arange(n, device="cuda") < before) | (torch.arange(n, device="cuda") >= n - after)
    assert not y32[gone].any()
    for yd in (F16, BF16):
        y = torch.full((n, N), float("nan"), dtype=yd, device="cuda")
        dense.GroupedMm(y=y, **kw).run(stream())
        assert torch.equal(y, y32.to(yd))
    want_q, want_s = dense.mx4_empty(n, N)
    dense.mx4_quantize(y32, want_q, want_s, stream())
    q, s = torch.full_like(want_q, 0x11), torch.full((n, N // 32), 0x11, dtype=torch.uint8, device="cuda")
    dense.GroupedMm(y=q, y_scales=s, **kw).run(stream())
    assert torch.equal(s, want_s) and np.array_equal(decode(q, s), decode(want_q, want_s))


@pytest.mark.parametrize("rows", [1, 63, 97, 1024, 2869, 4100])
@pytest.mark.parametrize("N,act", [(248, "silu_mul"), (512, "none"), (1064, "none")])
@pytest.mark.parametrize("dtype", [BF16, "mx4"])
def test_one_expert_of_many_rows(rows, N, act, dtype):
    """Where one expert's units would leave SMs without one, they are cut shorter."""
    g, K = gen(rows), 416
    x, w = randn(g, rows, K), randn(g, 1, N * (2 if act == "silu_mul" else 1), K) * K ** -0.5
    if dtype == "mx4":
        (x, xs, xv), (w, ws, wv) = mx4_of(x), mx4_of(w)
        kw = dict(x_scales=xs, w_scales=dense.mx4_tile_scales(ws, act))
    else:
        x, w = x.to(BF16), w.to(BF16)
        xv, wv, kw = x, w, {}
    y = torch.full((rows, N), float("nan"), dtype=BF16, device="cuda")
    dense.GroupedMm(x=x, w=w, y=y, act=act, **kw).run(stream())
    every = torch.arange(rows, device="cuda", dtype=torch.int32)
    want, tol = plain(xv, wv, every, torch.tensor([0, rows]), 0, act, N)
    close(y, want, tol, BF16)


@pytest.mark.parametrize("K", [32, 288, 544, 3808])
@pytest.mark.parametrize("form", ["narrow", "pair"])
@pytest.mark.parametrize("shift,extra", [(0, 0), (1, 0), (3, 2), (4, 4), (8, 8), (16, 5)])
def test_scales_at_any_alignment(K, form, shift, extra):
    """Row scales `shift` bytes behind a 16-byte boundary, `extra` between the rows, nothing behind the last: the same
    bits as scales on 16-byte rows."""
    counts, _, N = FORMS[form]
    g = gen(K)
    tok, off, n = routing(counts, g=g)
    xq, xs, _ = mx4_of(randn(g, n, K))
    wq, ws, _ = mx4_of(randn(g, len(counts), N, K))
    kw = dict(x=xq, w=wq, w_scales=dense.mx4_tile_scales(ws), expert_offset=off, sorted_tok=tok, top_k=1)
    want, y = (torch.full((n, N), float("nan"), dtype=BF16, device="cuda") for _ in range(2))
    dense.GroupedMm(y=want, x_scales=xs, **kw).run(stream())
    pitch = K // 32 + extra
    flat = torch.full((shift + (n - 1) * pitch + K // 32,), 255, dtype=torch.uint8, device="cuda")
    at = flat[shift:].as_strided((n, K // 32), (pitch, 1))
    at.copy_(xs)
    dense.GroupedMm(y=y, x_scales=at, **kw).run(stream())
    assert torch.equal(y, want)


@pytest.mark.parametrize("form", ["split", "narrow", "pair"])
@pytest.mark.parametrize("graph", [False, True])
def test_a_chain_waits_for_each_predecessor(form, graph):
    """Norm, quantisation, two products and the way back, each reading what the last one wrote and the first overwriting
    what the last reads, many times without a pause: the same bits as with a synchronisation after every call."""
    counts, K, _ = FORMS[form]
    H, W = K, 2 * K
    g = gen(K)
    tok, off, n = routing(counts, 3, 20, (5,), g=g)
    w1, w2 = randn(g, len(counts), 2 * W, H) * H ** -0.5, randn(g, len(counts), H, W) * W ** -0.5
    (q1, s1, _), w2 = mx4_of(w1), w2.to(BF16)
    start, norm_w = randn(g, n, H, dtype=BF16), randn(g, H, dtype=BF16)
    route = dict(expert_offset=off, sorted_tok=tok, top_k=1)
    x, xn, h, branch = (torch.empty((n, c), dtype=BF16, device="cuda") for c in (H, H, W, H))
    xq, xs = dense.mx4_empty(n, H)
    pre = dense.BlockNorm(res=x, pre_w=norm_w, y=xn)
    up = dense.GroupedMm(x=xq, x_scales=xs, w=q1, w_scales=dense.mx4_tile_scales(s1, "silu_mul"), y=h, act="silu_mul", **route)
    down = dense.GroupedMm(x=h, w=w2, y=branch, expert_offset=off, sorted_tok=tok, top_k=0)
    post = dense.BlockNorm(branch=branch, post_w=norm_w, res=x, res_scale=0.5, out=x)

    def steps(st):
        yield lambda: pre.run(st)
        yield lambda: dense.mx4_quantize(xn, xq, xs, st)
        yield lambda: up.run(st)
        yield lambda: down.run(st)
        yield lambda: dense.mx4_dequantize(xq, xs, xn, st)
        yield lambda: post.run(st)

    x.copy_(start)
    for _ in range(12):
        for call in steps(stream()):
            call()
            torch.cuda.synchronize()
    want = [t.clone() for t in (x, xn, h, branch)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            x.copy_(start)
            if graph:
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured, stream=side):
                    for _ in range(12):
                        for call in steps(torch.cuda.current_stream().cuda_stream):
                            call()
                x.copy_(start)
                captured.replay()
            else:
                for _ in range(12):
                    for call in steps(side.cuda_stream):
                        call()
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip((x, xn, h, branch), want))
