"""Layers of EXL3 experts run from several threads at once on a GPU, each on a stream of its own: their kernels need different
amounts of shared memory, and no call fails another's."""
import threading

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)


@pytest.mark.parametrize("T", [2, 300])
def test_layers_of_different_sizes(T):
    from exl3b200 import load_plugin
    from exl3b200.layer import MoeLayer
    plugin, failed = load_plugin(), []
    layers = []
    for n_expert, width in ((16, 512), (200, 512), (32, 256)):
        lay = MoeLayer(plugin, n_expert=n_expert, hidden=512, width=width, top_k=4, max_tokens=T)
        lay.x.normal_()
        lay.logits.normal_()
        lay.forward(T, torch.cuda.current_stream().cuda_stream)
        layers.append((lay, torch.cuda.Stream(), lay.out[:T].clone()))
    torch.cuda.synchronize()
    assert all(want.any() and want.isfinite().all() for _, _, want in layers)

    def steps(lay, stream):
        for _ in range(500):
            try:
                lay.forward(T, stream.cuda_stream)
            except RuntimeError as e:
                failed.append(e)
                return

    threads = [threading.Thread(target=steps, args=(lay, s)) for lay, s, _ in layers]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed[0]
    assert layers[0][0].native.read_error() == 0
    for lay, _, want in layers:
        assert torch.equal(lay.out[:T], want)
