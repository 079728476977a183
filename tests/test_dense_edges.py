"""The dense and MXFP4 expert operators where they can go wrong at their edges: the longest k, calls in which no expert has
a row, rows beside those of EXL3 experts."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402
from test_dense import decode, gen, mx4_of, randn, stream  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()
    assert dense.native().read_error() == 0


def places(K):
    """Columns at the first and last stages of k, around the middle, and at the row's two ends."""
    at = [0, 1, 255, 256, K // 2 - 1, K // 2, K - 257, K - 256, K - 65, K - 64, K - 1]
    return torch.tensor(sorted(set(at)), device="cuda")


@pytest.mark.parametrize("K", [1 << 26, (1 << 26) - 8, (1 << 26) - 200])
def test_the_longest_k_16_bit(K):
    """A row of zeros but for a few small whole numbers, times small whole numbers: the sum is exact in f32."""
    g, at = gen(1), places(K)
    w = torch.randint(-8, 9, (1, 8, K), generator=g, device="cuda", dtype=torch.int8).to(F16)
    x = torch.zeros((1, K), dtype=F16, device="cuda")
    x[0, at] = torch.arange(1, len(at) + 1, device="cuda").to(F16)
    y = torch.empty((1, 8), device="cuda")
    dense.GroupedMm(x=x, w=w, y=y).run(stream())
    assert torch.equal(y[0].double(), w[0][:, at].double() @ x[0, at].double())


@pytest.mark.parametrize("K", [1 << 26, (1 << 26) - 32])
def test_the_longest_k_mxfp4(K):
    """The same in MXFP4, every block with a scale of its own: values of two bits times powers of two within 2^8 of one
    another, a dozen of them, are exact in f32."""
    g, at = gen(2), places(K)
    wq = torch.randint(0, 256, (1, 8, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    ws = torch.randint(124, 129, (1, 8, K // 32), generator=g, device="cuda", dtype=torch.uint8)
    xq, xs = dense.mx4_empty(1, K)
    xq.zero_()
    xs.copy_(torch.randint(125, 130, (1, K // 32), generator=g, device="cuda", dtype=torch.uint8))
    for c in at.tolist():
        xq[0, c // 2] |= 2 << (4 * (c & 1))                  # the code of 1
    y = torch.empty((1, 8), device="cuda")
    dense.GroupedMm(x=xq, x_scales=xs, w=wq, w_scales=dense.mx4_tile_scales(ws, stream=stream()), y=y).run(stream())
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device="cuda")
    codes = (wq[0][:, at // 2].int() >> (4 * (at & 1))) & 15
    e = ws[0][:, at // 32].double() - 127 + xs[0, at // 32].double() - 127
    assert torch.equal(y[0].double(), (grid[codes] * torch.exp2(e)).sum(1))


@pytest.mark.parametrize("dtype", [BF16, "mx4"])
@pytest.mark.parametrize("E,n,N", [(5, 1, 264), (5, 40, 264), (3, 900, 1056)])
@pytest.mark.parametrize("start", [0, 1])
def test_no_expert_has_a_row(dtype, E, n, N, start):
    """Every offset the same (nothing routed here), in the split, narrow and pair forms: all rows are zero."""
    g, K = gen(E + n), 512
    x, w = randn(g, n, K), randn(g, E, N, K)
    off = torch.full((E + 1,), start, dtype=torch.int32, device="cuda")
    tok = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    kw = dict(expert_offset=off, sorted_tok=tok, top_k=1)
    if dtype == "mx4":
        (x, xs, _), (w, ws, _) = mx4_of(x), mx4_of(w)
        kw |= dict(x_scales=xs, w_scales=dense.mx4_tile_scales(ws, stream=stream()))
    else:
        x, w = x.to(dtype), w.to(dtype)
    y = torch.full((n, N), float("nan"), dtype=BF16, device="cuda")
    dense.GroupedMm(x=x, w=w, y=y, **kw).run(stream())
    assert torch.equal(y, torch.zeros_like(y))
    if N % 32 == 0:
        q, s = dense.mx4_empty(n, N)
        q.fill_(0x11)
        s.fill_(0x11)
        dense.GroupedMm(x=x, w=w, y=q, y_scales=s, **kw).run(stream())
        assert not q.any() and not s.any() and not np.any(decode(q, s))


@pytest.mark.parametrize("T,pad", [(3, 3), (128, 96)])
def test_beside_exl3_experts_in_one_buffer(T, pad):
    """Trailing experts in bf16 behind a layer's EXL3 ones: grouped_mm over their part of the offsets, which clears the rows
    before them, then the EXL3 ops over their live rows alone, which leave the others."""
    from exl3b200 import load_plugin
    from exl3b200.layer import MoeLayer
    lay = MoeLayer(load_plugin(), n_expert=16, hidden=2048, width=512, top_k=4, bits_gu=3, bits_dn=4, max_tokens=T, seed=3,
                   max_rows=T * 4 + pad)
    g, R, K = gen(4), T * lay.k, 256
    lay.x.copy_(randn(g, *lay.x.shape, dtype=F16))
    lay.logits.copy_(randn(g, *lay.logits.shape))
    lay.forward(T, stream())
    torch.cuda.synchronize()
    want = lay.y_rows[:R].view(torch.int16).clone()
    n = R + pad
    off = torch.tensor([R, R + pad // 3, n], dtype=torch.int32, device="cuda")
    y = lay.y_rows[:n].view(BF16)
    x, w = randn(g, n, K, dtype=BF16), randn(g, 2, lay.H, K, dtype=BF16)
    dense.GroupedMm(x=x, w=w, y=y, expert_offset=off).run(stream())
    alone = y[R:].clone()
    assert alone.any() and not y[:R].any()
    lay.experts(T, n, stream(), live=True)
    torch.cuda.synchronize()
    assert torch.equal(y[R:], alone) and torch.equal(lay.y_rows[:R].view(torch.int16), want)
