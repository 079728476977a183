"""FP8 rows on a GPU: f8_quantize and f8_dequantize against their definition in numpy, bit for bit (numpy's f32 quotients and
products are rounded to nearest, as the definition's are)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402

F32, F16, BF16, F8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
# e4m3's values in the order of their codes 0 .. 126
CODES = np.array([(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 7) for e in range(16) for m in range(8)][:127])


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()
    assert dense.native().read_error() == 0


def nearest(v):
    """The code bytes of f32 values: to nearest, ties to the even code."""
    a = np.abs(v.astype(np.float64))
    mid = (CODES[1:] + CODES[:-1]) / 2
    lo, hi = np.searchsorted(mid, a, side="left"), np.searchsorted(mid, a, side="right")
    n = np.where(lo == hi, lo, np.where(lo % 2 == 0, lo, hi))
    return (n | (np.signbit(v) << 7)).astype(np.uint8)


def quantised(x, pow2):
    """(code bytes, scales)."""
    rows, cols = x.shape
    nb = -(-cols // 128)
    b = np.zeros((rows, nb * 128), np.float32)
    b[:, :cols] = x.float().cpu().numpy()
    b = b.reshape(rows, nb, 128)
    with np.errstate(invalid="ignore", over="ignore"):
        bad = ~np.isfinite(b).all(2)
        m = np.maximum(np.abs(np.where(np.isfinite(b), b, 0)).max(2), np.float32(2.0 ** -110))
        s = m / np.float32(448)
        if pow2:
            f, e = np.frexp(s)
            s = np.ldexp(np.float32(1), np.where(f == 0.5, e - 1, e)).astype(np.float32)
            v = b / s[..., None]
        else:
            v = b * (np.float32(448) / m)[..., None]
    assert s.dtype == v.dtype == np.float32
    q = np.where(bad[..., None], 0, nearest(np.where(np.isfinite(v), v, 0))).astype(np.uint8)
    return q.reshape(rows, -1)[:, :cols], np.where(bad, np.nan, s).astype(np.float32)


def values(q, s):
    c = np.where(q & 0x7F == 0x7F, np.nan, CODES[np.minimum(q & 0x7F, 126)]).astype(np.float32)
    c = np.where(q & 0x80, -c, c)
    return c * np.repeat(s, 128, axis=1)[:, :q.shape[1]]


def check(x, pow2=False, codes=None, scales=None):
    rows, cols = x.shape
    if codes is None:
        codes, scales = dense.f8_empty(rows, cols)
    dense.f8_quantize(x, codes, scales, pow2=pow2)
    q, s = quantised(x, pow2)
    assert np.array_equal(scales.cpu().numpy(), s, equal_nan=True)
    assert np.array_equal(codes.view(torch.uint8).cpu().numpy(), q)
    want = torch.from_numpy(values(q, s)).cuda()
    for dt in (F32, F16, BF16):
        y = torch.full((rows, (cols + 7) // 8 * 8 + 8), 9.0, dtype=dt, device="cuda")
        dense.f8_dequantize(codes, scales, y[:, :cols])
        assert torch.equal(y[:, :cols].isnan(), want.to(dt).isnan())
        assert torch.equal(y[:, :cols].nan_to_num(7.0), want.to(dt).nan_to_num(7.0))
        assert (y[:, cols:] == 9.0).all()


def randn(seed, rows, cols, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn((rows, cols), generator=g, device="cuda")).to(dtype)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 16), (5, 120), (1, 128), (7, 136), (64, 640), (33, 1000), (300, 2048)])
def test_rows_of_every_type_and_odd_sizes(rows, cols, dtype, pow2):
    check(randn(rows + cols, rows, cols, dtype), pow2)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_extremes_zeros_and_values_that_are_no_numbers(dtype, pow2):
    x = randn(1, 24, 256, dtype)
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    x[0] = 0
    x[1, 3] = torch.nan
    x[2, 200] = torch.inf
    x[3, 0] = -torch.inf
    x[4] = big
    x[5] = -big
    x[6, 7] = big
    x[7] = tiny
    x[8] = tiny / 4
    x[9, :128] = 0
    x[10] = x[10] * 2.0 ** -20
    x[11] = -0.0
    if dtype != F16:
        x[12:20] = x[12:20] * 2.0 ** -112                       # about the least maximum
        x[20:] = x[20:] * 2.0 ** 120
    check(x, pow2)
    check(x, pow2, torch.empty((24, 256), dtype=F8, device="cuda"), torch.empty((24, 2), device="cuda"))     # rows without gaps


def test_values_on_the_midpoints():
    """Maxima whose quotient by 448 is exact, and multiples of it on e4m3's midpoints: ties, which go to the even code; and
    maxima for which the quotient is rounded, whose products fall beside them."""
    x = torch.zeros((400, 128), device="cuda")
    for i in range(400):
        m = float(i % 200 + 1)
        x[i] = m / 448 * torch.linspace(0, 16, 128, device="cuda").mul(8).round().div(8)
        x[i, 0] = m if i < 200 else m * 1.125
        x[i, 1:30] = m * torch.arange(1, 30, device="cuda") * 3 / 64
    for dt in (F32, BF16):
        check(x.to(dt))


def test_strides_and_neighbours_left_alone():
    x = torch.full((40, 704), torch.nan, dtype=BF16, device="cuda")
    x[:, 8:648] = randn(2, 40, 640, BF16)
    codes = torch.full((42, 672), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((42, 9), 5.0, device="cuda")
    check(x[:, 8:648], False, codes[1:41, 16:656].view(F8), scales[1:41, 2:7])
    assert (codes[[0, 41]] == 0x55).all() and (codes[:, :16] == 0x55).all() and (codes[:, 656:] == 0x55).all()
    assert (scales[[0, 41]] == 5).all() and (scales[:, :2] == 5).all() and (scales[:, 7:] == 5).all()


def test_every_code_back():
    q = torch.arange(256, dtype=torch.uint8, device="cuda").view(2, 128)
    s = torch.tensor([[0.375], [3.0e-5]], device="cuda")
    y = torch.empty((2, 128), device="cuda")
    dense.f8_dequantize(q.view(F8), s, y)
    assert np.array_equal(y.cpu().numpy(), values(q.cpu().numpy(), s.cpu().numpy()), equal_nan=True)


def test_no_rows():
    codes, scales = dense.f8_empty(0, 128)
    dense.f8_quantize(torch.empty((0, 128), device="cuda"), codes, scales)
    dense.f8_dequantize(codes, scales, torch.empty((0, 128), device="cuda"))


def test_captured_and_replayed():
    x = randn(1, 100, 640, BF16)
    codes, scales = dense.f8_empty(100, 640)
    dense.f8_quantize(x, codes, scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dense.f8_quantize(x, codes, scales)
    x.copy_(randn(2, 100, 640, BF16))
    graph.replay()
    q, s = quantised(x, False)
    assert np.array_equal(codes.view(torch.uint8).cpu().numpy(), q) and np.array_equal(scales.cpu().numpy(), s)
