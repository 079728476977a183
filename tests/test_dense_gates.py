"""The gates of the dense expert operators over their whole range, against 64 bits.

silu_mul's sums are one product of a weight by one, exact, so that what is compared is its own arithmetic: 2^-19 of the
value, the output's one rounding, and half a last place at the bottom of the type's range -- also where e^-z or the value
without its factor is outside f32's range."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402
from test_dense import TINY, ULP, stream  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()
    assert dense.native().read_error() == 0


# rows and repetitions of the gates that take the split, narrow and pair forms
FORMS = {"split": (3, 1, 512), "narrow": (20, 4, 8), "pair": (600, 3, 8)}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype,up", [(F16, 1.0), (F16, -3e4), (BF16, 1.0), (BF16, 2.0 ** 60), (BF16, 2.0 ** -30)])
def test_silu_mul_over_the_whole_range(form, dtype, up):
    rows, reps, K = FORMS[form]
    z = torch.arange(-1680, 1680, device="cuda").double() / 16
    z[:8] = torch.tensor([0.0, -0.0, 2.0 ** -14, -(2.0 ** -20), 6e4, -6e4, 300.0, -300.0], device="cuda")
    if dtype == BF16:
        z[8:16] = torch.tensor([1e-30, -1e-30, 1e30, -1e30, 1e38, -1e38, 1e-37, -1e-37], device="cuda")
    z = z.to(dtype).repeat(reps)
    N = z.numel()
    w = torch.zeros((1, 2 * N, K), dtype=dtype, device="cuda")
    w[0, :N, K - 1], w[0, N:, K - 1] = z, up
    x = torch.zeros((rows, K), dtype=dtype, device="cuda")
    x[:, K - 1] = 1
    want = z.double() * torch.sigmoid(z.double()) * w[0, N, K - 1].double()
    for out in (F32, F16, BF16):
        y = torch.empty((rows, N), dtype=out, device="cuda")
        dense.GroupedMm(x=x, w=w, y=y, act="silu_mul").run(stream())
        ref = want.to(F32).to(out) if out == F16 else want.to(out)
        fits = torch.isfinite(ref) & (want.abs() < torch.finfo(out).max)
        bound = (2.0 ** -19 + ULP[out]) * want.abs() * (1 + 2.0 ** -18) + TINY[out]
        err = (y.double() - want).abs()
        bad = fits & ~(err <= bound)
        assert not bool(bad.any()), (out, z[bad[0]][:5].tolist(), y[bad][:5].tolist())
        assert bool((torch.isinf(y) | (y.abs() >= torch.finfo(out).max * (1 - ULP[out])))[:, ~fits].all())


@pytest.mark.parametrize("form", ["split", "narrow", "pair"])
def test_silu_mul_of_infinities_and_nan(form):
    rows, _, K = FORMS[form]
    z = torch.tensor([float("inf"), float("nan"), 1.0, -1.0], device="cuda").repeat(200)
    N = z.numel()
    w = torch.zeros((1, 2 * N, K), dtype=BF16, device="cuda")
    w[0, :N, K - 1], w[0, N:, K - 1] = z.to(BF16), 2
    x = torch.zeros((rows, K), dtype=BF16, device="cuda")
    x[:, K - 1] = 1
    y = torch.empty((rows, N), device="cuda")
    dense.GroupedMm(x=x, w=w, y=y, act="silu_mul").run(stream())
    y = y.reshape(rows, 200, 4)
    assert torch.isposinf(y[..., 0]).all() and torch.isnan(y[..., 1]).all() and torch.isfinite(y[..., 2:]).all()


@pytest.mark.parametrize("kind", ["token", "element"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("H", [2048, 2047, 12000])
@pytest.mark.parametrize("n", [1.0, -(2.0 ** 15)])
def test_sigmoid_gates_over_the_whole_range(kind, dtype, H, n):
    """sigmoid(g) * branch alone: the same bound."""
    T = 420 if kind == "token" else 2
    size = T if kind == "token" else T * H
    g = ((torch.arange(size, device="cuda") % 1680).double() / (4 if kind == "token" else 8) - 105)
    g[:6] = torch.tensor([0.0, -0.0, 300.0, -300.0, float("inf"), float("-inf")], device="cuda")
    g = g.to(F32) if kind == "token" else g.to(dtype).reshape(T, H)
    branch = torch.full((T, H), n, dtype=dtype, device="cuda")
    out = torch.empty((T, H), dtype=dtype, device="cuda")
    dense.BlockNorm(branch=branch, gate=g, gate_kind=kind, out=out).run(stream())
    want = torch.sigmoid(g.double()) * n
    want = want[:, None].expand(T, H) if kind == "token" else want
    err = (out.double() - want).abs()
    assert bool((err <= (2.0 ** -19 + ULP[dtype]) * want.abs() * (1 + 2.0 ** -18) + TINY[dtype]).all())
