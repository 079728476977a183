"""What exl3b200/dense.py refuses before it calls the library, over stand-ins for tensors: no GPU, none of them is read."""
import pytest

torch = pytest.importorskip("torch")

from exl3b200 import dense  # noqa: E402

F32, F16, BF16, U8, I32 = torch.float32, torch.float16, torch.bfloat16, torch.uint8, torch.int32


class Fake:
    """As much of a dense tensor on GPU `dev` (-1: on the CPU) as a plan asks for."""

    def __init__(self, *shape, dtype=BF16, dev=0):
        self.shape, self.dtype, self.dev = torch.Size(shape), dtype, dev
        self.is_cuda, self.device = dev >= 0, torch.device("cuda", dev) if dev >= 0 else torch.device("cpu")

    def get_device(self):
        return self.dev

    def dim(self):
        return len(self.shape)

    def stride(self, d=None):
        st, n = [], 1
        for s in reversed(self.shape):
            st.insert(0, n)
            n *= s
        return tuple(st) if d is None else st[d]

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096


@pytest.fixture
def launched(monkeypatch):
    """The calls that reach the library, which is not called, and their streams; the current device is GPU 0, its current
    stream 77."""
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append((name, a[-1])) or 0

    class Host(Lib):
        lib = Lib()

        def mx4_tiled_bytes(self, *a):
            return 4096

        def expert_block_work_bytes(self, *a):
            return 4096

        def expert_block_carve(self, *a):
            pass

    class Stream:
        cuda_stream = 77

        def synchronize(self):
            calls.append(("synchronize", 77))

    monkeypatch.setattr(dense, "_native", Host())
    monkeypatch.setattr(dense, "_several", True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: Stream())
    monkeypatch.setattr(torch, "empty", lambda n, dtype=None, device=None: Fake(n, dtype=dtype))
    return calls


def grouped(**k):
    t = dict(x=Fake(4, 64), w=Fake(2, 32, 64), y=Fake(4, 32), expert_offset=Fake(3, dtype=I32), sorted_tok=Fake(4, dtype=I32),
             top_k=1)
    return dense.GroupedMm(**dict(t, **k))


def grouped_mx4(**k):
    t = dict(x=Fake(4, 32, dtype=U8), x_scales=Fake(4, 2, dtype=U8), w=Fake(2, 32, 32, dtype=U8), w_scales=Fake(4096, dtype=U8),
             y=Fake(4, 16, dtype=U8), y_scales=Fake(4, 1, dtype=U8), expert_offset=Fake(3, dtype=I32))
    return dense.GroupedMm(**dict(t, **k))


def norm(**k):
    t = dict(branch=Fake(4, 64), post_w=Fake(64), gate=Fake(64), gate_kind="channel", res=Fake(4, 64), out=Fake(4, 64),
             pre_w=Fake(64), y=Fake(4, 64), y_codes=Fake(4, 32, dtype=U8), y_scales=Fake(4, 2, dtype=U8))
    return dense.BlockNorm(**dict(t, **k))


OTHER = {grouped: ("x", "w", "y", "expert_offset", "sorted_tok"), grouped_mx4: ("x_scales", "w_scales", "y_scales"),
         norm: ("branch", "post_w", "gate", "res", "out", "pre_w", "y", "y_codes", "y_scales")}


@pytest.mark.parametrize("make,name", [(m, n) for m, names in OTHER.items() for n in names])
@pytest.mark.parametrize("dev", [-1, 1])
def test_a_plans_tensors_share_a_gpu(launched, make, name, dev):
    base = {"x": Fake(4, 64), "w": Fake(2, 32, 64), "y": Fake(4, 32), "expert_offset": Fake(3, dtype=I32),
            "sorted_tok": Fake(4, dtype=I32)}
    if make is grouped_mx4:
        base = {"x_scales": Fake(4, 2, dtype=U8), "w_scales": Fake(4096, dtype=U8), "y_scales": Fake(4, 1, dtype=U8)}
    if make is norm:
        base = {n: Fake(4, 64) for n in ("branch", "res", "out", "y")} | {n: Fake(64) for n in ("post_w", "gate", "pre_w")} | {
            "y_codes": Fake(4, 32, dtype=U8), "y_scales": Fake(4, 2, dtype=U8)}
    t = base[name]
    make(**{name: t}).run(0)
    assert len(launched) == 1
    with pytest.raises(ValueError, match="GPU|cuda"):
        make(**{name: Fake(*t.shape, dtype=t.dtype, dev=dev)}).run(0)
    assert len(launched) == 1


@pytest.mark.parametrize("make", [grouped, grouped_mx4, norm])
def test_a_plan_runs_on_its_own_gpu_only(launched, monkeypatch, make):
    plan = make()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="cuda:0"):
        plan.run(0)
    assert not launched


def test_the_conversions_tensors_share_the_current_gpu(launched, monkeypatch):
    x, codes, scales = Fake(4, 64), Fake(4, 32, dtype=U8), Fake(4, 2, dtype=U8)
    dense.mx4_quantize(x, codes, scales, 0)
    dense.mx4_dequantize(codes, scales, x, 0)
    assert len(launched) == 2
    for bad in ((Fake(4, 64, dev=1), codes, scales), (x, Fake(4, 32, dtype=U8, dev=1), scales),
                (x, codes, Fake(4, 2, dtype=U8, dev=1)), (x, codes, Fake(4, 2, dtype=U8, dev=-1))):
        with pytest.raises(ValueError):
            dense.mx4_quantize(*bad, 0)
        with pytest.raises(ValueError):
            dense.mx4_dequantize(bad[1], bad[2], bad[0], 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (lambda: dense.mx4_quantize(x, codes, scales, 0), lambda: dense.mx4_dequantize(codes, scales, x, 0),
                 lambda: dense.mx4_tile_scales(Fake(2, 32, 2, dtype=U8), stream=0)):
        with pytest.raises(ValueError):
            call()
    assert len(launched) == 2


@pytest.mark.parametrize("make,missing", [(grouped_mx4, "x_scales"), (grouped_mx4, "w_scales"), (grouped_mx4, "y_scales")])
def test_mxfp4_without_its_scales(launched, make, missing):
    with pytest.raises(ValueError, match=missing):
        make(**{missing: None})


@pytest.mark.parametrize("gu,dn", [(False, True), (True, False)])
def test_an_mxfp4_block_without_its_scales(launched, gu, dn):
    U = lambda *s: Fake(*s, dtype=U8)  # noqa: E731
    with pytest.raises(ValueError, match="dn_scales" if gu else "gu_scales"):
        dense.ExpertBlock(router_w=Fake(8, 64), gu_w=U(8, 128, 32), dn_w=U(8, 64, 32), pre_w=Fake(64), top_k=2,
                          gu_scales=U(8, 128, 2) if gu else None, dn_scales=U(8, 64, 2) if dn else None)


@pytest.mark.parametrize("name,shape", [("x", (4, 64, 72)), ("x", (64,)), ("y", (4, 32, 40)), ("y", (32,)), ("w", (32, 64)),
                                        ("w", (2, 32, 64, 8))])
def test_grouped_mm_wants_matrices(launched, name, shape):
    """Rows of a third dimension were taken for rows of the second one's length."""
    with pytest.raises(ValueError):
        grouped(**{name: Fake(*shape)})


@pytest.mark.parametrize("shape", [(4, 64, 72), (64,)])
def test_norms_and_conversions_want_matrices(launched, shape):
    with pytest.raises(ValueError):
        norm(branch=Fake(*shape))
    with pytest.raises(ValueError):
        dense.mx4_quantize(Fake(*shape), Fake(4, 32, dtype=U8), Fake(4, 2, dtype=U8), 0)
    assert not launched


def block():
    U = lambda *s: Fake(*s, dtype=U8)  # noqa: E731
    return dense.ExpertBlock(router_w=Fake(8, 64), gu_w=U(8, 128, 32), dn_w=U(8, 64, 32), pre_w=Fake(64), top_k=2,
                             gu_scales=U(8, 128, 2), dn_scales=U(8, 64, 2))


@pytest.mark.parametrize("given", [None, 0, 5])
def test_every_call_takes_the_same_default_stream(launched, given):
    """torch's current stream, where the tensors were written; its side streams do not wait for the legacy one."""
    kw, want = ({}, 77) if given is None else (dict(stream=given), given)
    x, codes, scales = Fake(4, 64), Fake(4, 32, dtype=U8), Fake(4, 2, dtype=U8)
    b = block()
    launched.clear()
    dense.mx4_quantize(x, codes, scales, **kw)
    dense.mx4_dequantize(codes, scales, x, **kw)
    grouped().run(**kw)
    norm().run(**kw)
    b.forward(x, x, **kw)
    assert [s for _, s in launched] == [want] * 5
    if given is None:
        dense.mx4_tile_scales(Fake(2, 32, 2, dtype=U8))
        assert launched[-1][1] == 77


def test_a_block_is_ready_on_any_stream(launched):
    """Its scales are tiled, and its work block's earlier uses over, before the constructor returns."""
    block()
    assert [n for n, _ in launched] == ["mx4_tile_scales", "mx4_tile_scales", "synchronize"]


@pytest.mark.parametrize("given,want", [(None, None), (77, None), (5, 5), (0, 0)])
def test_tiled_scales_lie_in_their_streams_memory(launched, monkeypatch, given, want):
    """What is written on a stream is allocated there: memory of the current one's pool may still be in use on it."""
    inside, got = [], []

    class On:
        def __init__(self, s):
            self.s = s

        def __enter__(self):
            inside.append(self.s)

        def __exit__(self, *a):
            inside.pop()

    monkeypatch.setattr(torch.cuda, "stream", On)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda s, device=None: s)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda dev=None: 0)
    monkeypatch.setattr(torch, "empty", lambda n, dtype=None, device=None: got.append(inside[-1] if inside else None)
                        or Fake(n, dtype=dtype))
    dense.mx4_tile_scales(Fake(2, 32, 2, dtype=U8), stream=given)
    assert got == [want] and launched[-1][1] == (77 if given is None else given)
