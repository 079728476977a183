"""The dense and MXFP4 expert operators on streams other than the default one: what a call reads was written on the stream
it is enqueued on by default, and a block that was built on one stream runs on another."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from exl3b200 import dense  # noqa: E402
from test_dense import gen, randn  # noqa: E402
from test_expert_block import make  # noqa: E402

BF16 = torch.bfloat16
PAUSE = 100_000_000                     # clock cycles, some 50 ms


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()
    assert dense.native().read_error() == 0


def test_defaults_follow_the_current_stream():
    g, K, N = gen(1), 256, 264
    x, w = randn(g, 64, K, dtype=BF16), randn(g, 3, 2 * N, K) * K ** -0.5
    norm_w, off = randn(g, N, dtype=BF16), torch.tensor([0, 20, 20, 64], dtype=torch.int32, device="cuda")
    zeros = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731

    def chain(pause):
        """Each step's inputs are written on the current stream, the first of them after a pause."""
        xin, back, y, out = zeros(64, K), zeros(64, K), zeros(64, N), zeros(64, N)
        win = zeros(3 * 2 * N, K, dtype=torch.float32)
        (xq, xs), (wq, ws) = dense.mx4_empty(64, K), dense.mx4_empty(3 * 2 * N, K)
        for t in (xq, xs, wq, ws):
            t.zero_()
        torch.cuda.synchronize()
        if pause:
            torch.cuda._sleep(PAUSE)
        xin.copy_(x)
        win.copy_(w.reshape(-1, K))
        dense.mx4_quantize(xin, xq, xs)
        dense.mx4_quantize(win, wq, ws)
        dense.mx4_dequantize(xq, xs, back)
        tiled = dense.mx4_tile_scales(ws.reshape(3, 2 * N, -1), "silu_mul")
        dense.GroupedMm(x=xq, x_scales=xs, w=wq.reshape(3, 2 * N, -1), w_scales=tiled, y=y, expert_offset=off,
                        act="silu_mul").run()
        dense.BlockNorm(branch=y, post_w=norm_w, out=out).run()
        torch.cuda.synchronize()
        return back, y, out

    want = chain(False)
    assert want[2].any()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = chain(True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("mx", [False, True])
def test_a_block_built_on_one_stream_runs_on_another(mx):
    t, block = make(16, 256, 128, 2, BF16, mx, 3, 32)
    x = torch.randn((32, 256), device="cuda").to(BF16)
    want = block.forward(x, torch.empty_like(x))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        # memory that the second block is likely to get, still being written when it is built
        sizes = [k.numel() for k in block._keep[7:]] + [block.work.numel()]
        junk = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes]
        torch.cuda._sleep(PAUSE)
        for j in junk:
            j.fill_(0xFF)
        del j, junk
        again = dense.ExpertBlock(top_k=2, eps=1e-6, res_scale=0.5, max_tokens=32, **t)
    out = torch.empty_like(x)
    for st in (torch.cuda.current_stream(), side):
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            again.forward(x, out.fill_(float("nan")))
        st.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("legacy", [False, True])
def test_scales_tiled_on_another_stream_keep_their_memory(legacy):
    """A block of the current stream's memory, freed while it is still being written there, is not what they lie in."""
    ws = torch.randint(0, 255, (4, 256, 16), generator=gen(2), device="cuda", dtype=torch.uint8)
    want = dense.mx4_tile_scales(ws, "silu_mul")
    torch.cuda.synchronize()
    other = torch.cuda.default_stream() if legacy else torch.cuda.Stream()
    with torch.cuda.stream(torch.cuda.Stream()):
        junk = torch.empty_like(want)
        torch.cuda._sleep(PAUSE)
        junk.fill_(0xAA)
        del junk
        out = dense.mx4_tile_scales(ws, "silu_mul", stream=other.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
