"""Which form an FP8 product takes: that the tests named for a form run in it, on a B200's 148 SMs; the rule is host code, so this
needs no GPU."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from exl3b200.native import Native  # noqa: E402

B200 = 148


def form_of(n_expert, n_rows, n_out, n_in, act="none", sms=B200):
    """"wide", "narrow" or "split"."""
    f = Native().lib.exl3b_gmm8_form
    f.argtypes = [C.c_int64] * 4 + [C.c_int] * 2
    return {0: "wide", 1: "narrow"}.get(f(n_expert, n_rows, n_out, n_in, act == "silu_mul", sms), "split")


@pytest.mark.parametrize("act", ["none", "silu_mul"])
def test_the_forms_that_tests_are_named_for(act):
    from test_f8_mm import FORMS
    for name, (counts, K, N) in FORMS.items():
        assert form_of(len(counts), sum(counts), N, K, act) == name
        assert form_of(len(counts), sum(counts) + 8, N, K, act) == name         # with rows outside the runs
    for K in (272, 640, 3824):
        assert form_of(20, 50, 1048, K) == "narrow"
        assert form_of(2, 2100, 2048, K) == "wide"
    assert form_of(2, 9, 128, 3824) == "split"
    assert form_of(1, 40000, 16384, 256) == form_of(2, 2100, 2048, 128) == "wide"
    assert form_of(1, 40000, 16384, 64) == "narrow"


@pytest.mark.parametrize("sms", [132, B200, 160])
def test_sizes_far_from_the_rules_border(sms):
    """test_f8_mm_edges.py's: the same form for a tenth fewer or more SMs, and a fifth fewer rows or a quarter more."""
    from test_f8_mm_edges import FAR
    for form, E, rows, N, K in FAR:
        assert form_of(E, rows, N, K, sms=sms) == form
        if form == "wide":
            assert form_of(E, rows * 4 // 5, N, K, sms=sms) == form
        if form == "narrow":
            assert form_of(E, rows * 5 // 4, N, K, sms=sms) == form
