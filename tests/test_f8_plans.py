"""What exl3b200/dense.py's router, FP8 rows and FP8 products refuse before they call the library, and the streams they take, over
stand-ins for tensors: no GPU, none of them is read."""
import pytest

torch = pytest.importorskip("torch")

from exl3b200 import dense  # noqa: E402
from test_dense_plans import Fake, launched  # noqa: E402, F401

F32, I32, F8 = torch.float32, torch.int32, torch.float8_e4m3fn


def mm_tensors():
    return dict(x=Fake(4, 256, dtype=F8), x_scales=Fake(4, 2, dtype=F32), w=Fake(2, 64, 256, dtype=F8),
                w_scales=Fake(2, 1, 2, dtype=F32), y=Fake(4, 64), expert_offset=Fake(3, dtype=I32), sorted_tok=Fake(4, dtype=I32))


def router_tensors():
    return dict(logits=Fake(4, 16, dtype=F32), bias=Fake(16, dtype=F32), ids=Fake(4, 2, dtype=I32), w=Fake(4, 2, dtype=F32),
                sorted_tok=Fake(8, dtype=I32), expert_offset=Fake(17, dtype=I32))


def rows_tensors():
    return dict(x=Fake(4, 256), codes=Fake(4, 256, dtype=F8), scales=Fake(4, 2, dtype=F32))


MAKERS = {"mm": (mm_tensors, lambda t, *s: dense.GroupedMm(**t).run(*s)),
          "router": (router_tensors, lambda t, *s: dense.Router(top_k=2, **t).run(*s)),
          "quantize": (rows_tensors, lambda t, *s: dense.f8_quantize(t["x"], t["codes"], t["scales"], False, *s)),
          "dequantize": (rows_tensors, lambda t, *s: dense.f8_dequantize(t["codes"], t["scales"], t["x"], *s))}


def enqueued(launched):
    return [c for c in launched if c[0].startswith("exl3b200_")]


@pytest.mark.parametrize("kind,name", [(k, n) for k, (t, _) in MAKERS.items() for n in t()])
@pytest.mark.parametrize("dev", [-1, 1])
def test_a_calls_tensors_share_a_gpu(launched, kind, name, dev):
    tensors, call = MAKERS[kind]
    t = tensors()
    call(t, 5)
    assert len(enqueued(launched)) == 1
    t[name] = Fake(*t[name].shape, dtype=t[name].dtype, dev=dev)
    with pytest.raises(ValueError, match="GPU|cuda"):
        call(t, 5)
    assert len(enqueued(launched)) == 1


@pytest.mark.parametrize("kind", MAKERS)
def test_that_gpu_is_the_current_one(launched, kind):
    tensors, call = MAKERS[kind]
    with pytest.raises(ValueError, match="current"):
        call({n: Fake(*t.shape, dtype=t.dtype, dev=1) for n, t in tensors().items()}, 5)
    assert not enqueued(launched)


@pytest.mark.parametrize("kind,name", [(k, n) for k, (t, _) in MAKERS.items() for n in t()])
def test_types_and_shapes_that_do_not_fit(launched, kind, name):
    """int64 in every place; one more row (and for x and y of a product, whose rows may be more, one more column)."""
    tensors, call = MAKERS[kind]
    t = tensors()
    old = t[name]
    longer = (*old.shape[:-1], old.shape[-1] + 1) if (kind, name) in (("mm", "x"), ("mm", "y")) else (old.shape[0] + 1, *old.shape[1:])
    bad = [Fake(*old.shape, dtype=torch.int64)] + ([Fake(*longer, dtype=old.dtype)] if (kind, name) != ("router", "expert_offset") else
                                                   [Fake(1, dtype=I32), Fake(4, 4, dtype=I32)])
    for f in bad:
        with pytest.raises(ValueError):
            call({**t, name: f}, 5)
    assert not enqueued(launched)


@pytest.mark.parametrize("given", [None, 0, 5])
@pytest.mark.parametrize("kind", MAKERS)
def test_every_call_takes_the_same_default_stream(launched, kind, given):
    tensors, call = MAKERS[kind]
    call(tensors(), *([] if given is None else [given]))
    assert [s for _, s in enqueued(launched)] == [77 if given is None else given]


def test_a_router_sorts_with_both_arrays_or_neither(launched):
    t = router_tensors()
    for one in ("sorted_tok", "expert_offset"):
        with pytest.raises(ValueError):
            dense.Router(top_k=2, **{**t, one: None})
    dense.Router(top_k=2, **{**t, "sorted_tok": None, "expert_offset": None}).run()
    assert len(enqueued(launched)) == 1


@pytest.mark.parametrize("capturing", [False, True])
@pytest.mark.parametrize("T,waits", [(4, 0), (1024, 0), (1025, 1)])
def test_a_router_waits_for_its_work_buffer_only_where_it_has_one(launched, monkeypatch, T, waits, capturing):
    """Of up to 2048 pairs it has none; under capture there is nothing to wait for, and waiting would end the capture."""
    monkeypatch.setattr(dense._native, "scatter_work_bytes", lambda *a: 4096, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    plan = dense.Router(top_k=2, logits=Fake(T, 16, dtype=F32), ids=Fake(T, 2, dtype=I32), w=Fake(T, 2, dtype=F32),
                        sorted_tok=Fake(2 * T, dtype=I32), expert_offset=Fake(17, dtype=I32))
    assert [n for n, _ in launched].count("synchronize") == (0 if capturing else waits)
    assert bool(plan.desc.work) == bool(waits)
