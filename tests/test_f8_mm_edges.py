"""grouped_mm over FP8 operands on a GPU at the ends of its scales' range. Tolerances are those of test_f8_mm.py: its errors are
relative to the blocks' sums, whatever their scales."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402
from test_dense import close, stream  # noqa: E402
from test_f8_mm import FORMS, F32, gpu, operands, plain, values_of  # noqa: E402, F401


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("x_by,w_by", [(-118, -2), (-3, -112), (-60, -60), (119, -20), (100, 2), (1, 100)])
def test_scales_at_the_ends_of_their_range(form, x_by, w_by):
    """x's scales times 2^x_by and the weight's times 2^w_by: from the least that f8_quantize makes to the largest of bf16 rows, with
    products down to 2^-126 and values up to 2^120. A block of zeros may have a smaller product."""
    counts, K, N = FORMS[form]
    rows = sum(counts)
    xq, xs, w, ws, xv = operands(3, len(counts), rows, K, N, "none")
    ws *= 60 * 60 * K ** 0.5                                    # about 1, as x's
    xs *= 2.0 ** x_by
    ws *= 2.0 ** w_by
    xq[rows // 2, :128] = 0
    xs[rows // 2, 0] = 2.0 ** -118
    xv = xq.double() * xs.double()[:, torch.arange(K, device="cuda") // 128]
    product = xs.double().amax() * ws.double().amax(), xs[:, 1:].double().amin() * ws.double().amin()
    assert product[0] < 2.0 ** 128 and product[1] >= 2.0 ** -126
    off = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    y = torch.full((rows, N), float("nan"), device="cuda")
    dense.GroupedMm(x=xq, x_scales=xs, w=w, w_scales=ws, expert_offset=off, y=y).run(stream())
    tok = torch.arange(rows, dtype=torch.int32, device="cuda")
    close(y, *plain(xv, values_of(w, ws, N), tok, off, 0, "none", N), F32)
