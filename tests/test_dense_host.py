"""The dense and MXFP4 expert operators' refusals that need no GPU: nothing is enqueued, so the addresses are made up."""
import ctypes as C

import pytest

pytest.importorskip("torch")

from exl3b200 import dense  # noqa: E402
from exl3b200.native import GroupedMmDesc, Native  # noqa: E402

E_SHAPE = -1
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
