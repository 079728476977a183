"""grouped_mm over FP8 operands on a GPU at the ends of its scales' range, and in each form at sizes well inside its side of
the rule that chooses. Tolerances are those of test_f8_mm.py: its errors are relative to the blocks' sums, whatever their
scales."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402
from test_dense import close, stream  # noqa: E402
from test_f8_forms import form_of  # noqa: E402
from test_f8_mm import F8, F16, F32, FORMS, gpu, operands, plain, values_of  # noqa: E402, F401


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("x_by,w_by", [(-118, -2), (-3, -112), (-60, -60), (119, -20), (100, 2), (1, 100)])
def test_scales_at_the_ends_of_their_range(form, x_by, w_by):
    """x's scales times 2^x_by and the weight's times 2^w_by: from the least that f8_quantize makes to the largest of bf16 rows,
    with products down to 2^-126 and values up to 2^120. A block of zeros may have a smaller product."""
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


# form, experts, rows, n_out, n_in: well inside the form's side of the rule
FAR = [("wide", 2, 5000, 2048, 400), ("wide", 1, 9000, 1024, 144), ("narrow", 24, 200, 1048, 144), ("narrow", 24, 200, 520, 2064),
       ("split", 2, 9, 128, 2064)]


def form_here(E, rows, N, K):
    return form_of(E, rows, N, K, sms=torch.cuda.get_device_properties(0).multi_processor_count)


@pytest.mark.parametrize("form,E,rows,N,K", FAR)
@pytest.mark.parametrize("shift,extra", [(0, 0), (1, 0), (3, 2), (4, 4)])
def test_each_form_with_scales_at_any_alignment(form, E, rows, N, K, shift, extra):
    assert form_here(E, rows, N, K) == form
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


@pytest.mark.parametrize("form,E,rows,N,K", [("wide", 2, 5000, 2048, 384), ("narrow", 24, 200, 1048, 384)])
def test_each_form_past_32_bits(form, E, rows, N, K):
    """Weights, input rows and output rows that lie over 4 GiB into their tensors."""
    assert form_here(E, rows, N, K) == form
    far, pitch = 4_600_000_000 // (E - 1) // 16 * 16, 4_800_000_000 // rows // 16 * 16
    xq, xs, w, ws, xv = operands(6, E, rows, K, N, "none")
    wf = torch.as_strided(torch.empty((E - 1) * far + N * K, dtype=torch.uint8, device="cuda"), (E, N, K), (far, K, 1))
    wf.copy_(w.view(torch.uint8))
    x = torch.as_strided(torch.empty((rows - 1) * pitch + K, dtype=torch.uint8, device="cuda"), (rows, K), (pitch, 1))
    x.copy_(xq.view(torch.uint8))
    y = torch.as_strided(torch.empty((rows - 1) * (pitch // 2) + N, dtype=F16, device="cuda"), (rows, N), (pitch // 2, 1))
    tok = torch.randperm(rows, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(torch.int32)
    off = torch.tensor([rows * e // E for e in range(E + 1)], dtype=torch.int32, device="cuda")
    dense.GroupedMm(x=x.view(F8), x_scales=xs, w=wf.view(F8), w_scales=ws, y=y, expert_offset=off, sorted_tok=tok,
                    top_k=1).run(stream())
    close(y, *plain(xv, values_of(w, ws, N), tok, off, 1, "none", N), F16)


def test_the_narrow_forms_units_past_the_table():
    """A row for each of 2048 experts and 32 blocks of outputs: 221 units a CTA, of which its table holds 128."""
    E, N, K = 2048, 4096, 64
    assert form_here(E, E, N, K) == form_here(E, 2 * E, N, K) == "narrow"
    xq, xs, w, ws, xv = operands(8, E, E, K, N, "none")
    off = torch.arange(E + 1, dtype=torch.int32, device="cuda")
    y = torch.full((E, N), float("nan"), device="cuda")
    dense.GroupedMm(x=xq, x_scales=xs, w=w, w_scales=ws, expert_offset=off, y=y).run(stream())
    for e in range(0, E, 256):                  # experts at a time: a weight's values take eight bytes each
        s = slice(e, e + 256)
        wv = values_of(w[s], ws[s], N)
        want = torch.einsum("ek,enk->en", xv[s], wv)
        tol = (128 + 1 + 5) * 2.0 ** -23 * torch.einsum("ek,enk->en", xv[s].abs(), wv.abs())
        close(y[s], want, tol, F32)


@pytest.mark.parametrize("form,E,rows,N,K", FAR)
def test_each_form_without_a_sort(form, E, rows, N, K):
    """No sorted_tok: row i is slot i of token i / top_k, the last token's slots not all there."""
    xq, xs, w, ws, xv = operands(5, E, -(-rows // 7), K, N, "none")
    off = torch.tensor([rows * e // E for e in range(E + 1)], dtype=torch.int32, device="cuda")
    y = torch.full((rows, N), float("nan"), dtype=F16, device="cuda")
    dense.GroupedMm(x=xq, x_scales=xs, w=w, w_scales=ws, expert_offset=off, top_k=7, y=y).run(stream())
    tok = torch.arange(rows, dtype=torch.int32, device="cuda")
    close(y, *plain(xv, values_of(w, ws, N), tok, off, 7, "none", N), F16)
