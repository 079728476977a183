"""The dense and MXFP4 expert operators' refusals that need no GPU: nothing is enqueued, so the addresses are made up (and
the tests are for machines without a GPU, where a call that is not refused ends with no device)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from exl3b200 import dense  # noqa: E402
from exl3b200.native import ExpertBlockBufs, ExpertBlockDesc, GroupedMmDesc, Native  # noqa: E402

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses")
E_SHAPE, E_ALIGN, E_DEVICE = -1, -3, -6
LIMIT = 1 << 26                         # grouped_mm's n_in


def product(dtype, n_in):
    """One row times eight weight rows, otherwise within every limit."""
    return GroupedMmDesc(n_expert=1, n_rows=1, n_out=8, n_in=n_in, x_rows=1, top_k=0, dtype=dtype, y_dtype=1, act=0, x=4096,
                         x_pitch=n_in, x_scales=4096, x_scales_pitch=n_in // 32, w=4096, w_pitch=n_in, w_scales=4096,
                         y=4096, y_pitch=8)


@pytest.mark.parametrize("dtype,step", [(2, 8), (3, 8), (dense.MX4, 32)])
def test_grouped_mm_refuses_a_k_past_its_indices(dtype, step):
    """32 bits hold the offsets along k up to the limit; past it a call would read in front of its operands: MXFP4 scales
    (1 KB each 256 columns) from 2^29 + 1 on, 16-bit rows at 2^30."""
    lib = Native().lib
    for n_in in (LIMIT + step, (1 << 29) + 256, (1 << 30) - 64, (1 << 30) - 32, 1 << 30):
        d = product(dtype, n_in)
        assert lib.exl3b200_grouped_mm(C.addressof(d), None) == E_SHAPE, n_in
    for n in (LIMIT, 2 * LIMIT):        # what the limit is for: the last stage's offsets
        assert (n // 256 - 1) * 1024 < 1 << 31 and n * 2 < 1 << 31


@pytest.mark.parametrize("weights", [3, dense.MX4])
@pytest.mark.parametrize("name", ["out", "next", "router_w", "gu_w", "dn_w", "gu_scales", "dn_scales", "post_w", "gate", "next_w"])
def test_the_expert_block_refuses_misaligned_operands_before_its_first_step(weights, name):
    """Not when the step that reads them is reached, with the others enqueued."""
    nat = Native()
    at = {n: 4096 for n in ("router_w", "gu_w", "dn_w", "gu_scales", "dn_scales", "pre_w", "post_w", "gate", "next_w")}
    io = {"out": 4096, "next": 4096}
    odd = 4097 if name in ("out", "next", "post_w", "gate", "next_w") else 4096 + 8
    (io if name in io else at)[name] = odd
    d = ExpertBlockDesc(n_expert=64, hidden=2048, width=512, top_k=10, dtype=3, weights=weights, eps=1e-6, res_scale=1.0, **at)
    b = nat.expert_block_carve(d, 8, 4096, nat.expert_block_work_bytes(d, 8))
    rc = nat.lib.exl3b200_expert_block_forward(d, b, 4096, 4, io["out"], io["next"], None)
    assert rc == (E_DEVICE if weights == 3 and name in ("gu_scales", "dn_scales") else E_ALIGN)      # unread: 16-bit weights
