"""The serving example's decoder on its own stream."""

import pytest

from aero_b200 import native_cuda as nc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_lib):
    nc.require_gpu()


def test_decoder_stream_waits_for_the_weights(monkeypatch):
    """Work of the stream that makes the weights is still under way when the decoder is there: its own
    stream begins behind it. (Nothing is computed with weights that may not be there.)"""
    from aero_b200 import synth
    from aero_b200.pages import PagedCache
    from aero_b200.serve_example import PagedDecoder
    c = PagedCache(1, 4, 16, 2, 64, 1, 4)
    PagedDecoder(c, 8, 256, 100).close()  # kernels loaded
    opened = synth.open_layer

    def open_and_keep_busy(*a, **kw):
        layer = opened(*a, **kw)
        torch.cuda._sleep(int(4e8))  # some 0.2 s
        return layer

    monkeypatch.setattr(synth, "open_layer", open_and_keep_busy)
    made_on = torch.cuda.Stream()
    with torch.cuda.stream(made_on):
        net = PagedDecoder(c, 8, 256, 100)
        made = made_on.record_event()
    begins = net.stream.record_event()
    early, done = begins.query(), made.query()
    torch.cuda.synchronize()
    net.close()
    assert done or not early
    assert not done, "the weights were there too soon for this test to show anything"
