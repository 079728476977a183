"""FP8 rows past 2^31 lanes on a GPU, where places are worked out in 64 bits: to the bit, on the rows around every border."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402
from test_f8 import BF16, F8, gpu, quantised, values  # noqa: E402, F401

STEP = 1 << 20                          # rows written at a time


def fill(x):
    """Rows of N(0, 1), then every row times a power of two of its own number's: no two neighbours alike."""
    g = torch.Generator(device="cuda").manual_seed(5)
    for r in range(0, x.shape[0], STEP):
        p = x[r:r + STEP]
        p.normal_(generator=g)
        p.mul_(torch.exp2((torch.arange(r, r + p.shape[0], device="cuda") % 7).float()).to(x.dtype)[:, None])


def around(rows, lanes):
    """Rows at both ends and around the row of lane 2^31, `lanes` a row."""
    at, block = (1 << 31) // lanes, 1024 // lanes
    near = {r for c in (0, block, at - block, at, rows // 2, rows - 1) for r in range(c - 2, c + 3)}
    return sorted(r for r in near if 0 <= r < rows)


def check(x, codes, scales, at):
    q, s = quantised(x[at], False)
    assert np.array_equal(codes.view(torch.uint8)[at].cpu().numpy(), q)
    assert np.array_equal(scales[at].cpu().numpy(), s)
    return q, s


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("less than 80 GiB free")
    yield
    torch.cuda.empty_cache()


def test_rows_that_lie_apart():
    """Sixteen lanes a row of eight values."""
    rows = (1 << 27) + 3
    x = torch.empty((rows, 8), dtype=BF16, device="cuda")
    fill(x)
    codes, scales = torch.empty((rows, 8), dtype=F8, device="cuda"), torch.empty((rows, 1), device="cuda")
    dense.f8_quantize(x, codes, scales)
    check(x, codes, scales, around(rows, 16))
    q, s = codes.view(torch.uint8), scales
    near = s >= x.float().abs().amax(1, keepdim=True) / 449        # all of them: every row was written, each from its own values
    assert bool(near.all()) and bool((s <= x.float().abs().amax(1, keepdim=True) / 447).all())
    assert bool(((q & 0x7F).amax(1) == 0x7E).all())                # a row's largest value is the largest code


def test_rows_without_gaps_there_and_back():
    """2^31 lanes of whole blocks, and as many vectors back."""
    rows, cols = (1 << 24) + 5, 1024
    x = torch.empty((rows, cols), dtype=BF16, device="cuda")
    fill(x)
    codes, scales = torch.empty((rows, cols), dtype=F8, device="cuda"), torch.empty((rows, cols // 128), device="cuda")
    dense.f8_quantize(x, codes, scales)
    at = around(rows, cols // 8)
    q, s = check(x, codes, scales, at)
    want = torch.from_numpy(values(q, s)).to(BF16)
    for r in range(0, rows, STEP):
        p = slice(r, r + STEP)
        top = x[p].view(-1, cols // 128, 128).abs().amax(2).float()
        assert bool(((scales[p] - top / 448).abs() <= 2.0 ** -23 * top / 448).all())
        assert bool(((codes[p].view(torch.uint8).view(-1, cols // 128, 128) & 0x7F).amax(2) == 0x7E).all())
    x.fill_(float("nan"))
    dense.f8_dequantize(codes, scales, x)
    assert torch.equal(x[at].cpu(), want)
    for r in range(0, rows, STEP):
        p = slice(r, r + STEP)
        v = codes[p].float().view(-1, cols // 128, 128) * scales[p][..., None]
        assert torch.equal(x[p], v.view(-1, cols).to(BF16))
