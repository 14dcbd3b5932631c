"""The paged cache's and the logits' entry points without a GPU: plans and refusals."""

import ctypes

import numpy as np
import pytest

from aero_b200 import native_cuda as nc


def desc(**kw):
    a = dict(n_layer=2, n_page=10, page_size=16, n_head_kv=4, head_dim=128, n_seq=3, max_pages=5, dtype=nc.TYPE_F16, device=0, reserved=0)
    a.update(kw)
    return nc.PagesDesc(**a)


def test_plan_bytes(cuda_lib):
    by = (ctypes.c_int64 * 2)()
    total = cuda_lib.aero_cuda_pages_plan_bytes(ctypes.byref(desc()), by)
    assert by[0] == 2 * 2 * 10 * 4 * 16 * 128 * 2 and total == by[0] + by[1] and by[1] > 0
    assert cuda_lib.aero_cuda_pages_plan_bytes(ctypes.byref(desc(dtype=nc.TYPE_BF16)), None) == total
    from aero_b200.pages import plan_bytes
    assert plan_bytes(2, 10, 16, 4, 128, 3, 5)["total"] == total
    with pytest.raises(ValueError):
        plan_bytes(2, 10, 17, 4, 128, 3, 5)


@pytest.mark.parametrize("bad", [
    dict(n_layer=0), dict(n_page=-1), dict(page_size=4), dict(page_size=24), dict(page_size=512), dict(head_dim=96),
    dict(head_dim=320), dict(dtype=nc.TYPE_F32), dict(dtype=8), dict(n_seq=0), dict(max_pages=0), dict(n_head_kv=0),
    dict(n_page=1 << 28), dict(n_seq=1 << 20, max_pages=1 << 20)])
def test_invalid_descriptions(cuda_lib, bad):
    assert cuda_lib.aero_cuda_pages_plan_bytes(ctypes.byref(desc(**bad)), None) == -1
    err = ctypes.create_string_buffer(256)
    assert not cuda_lib.aero_cuda_pages_open(ctypes.byref(desc(**bad)), err, 256) and err.value


def test_refuses_without_gpu(cuda_lib):
    if nc.gpu_count() > 0:
        pytest.skip("a GPU is visible")
    err = ctypes.create_string_buffer(256)
    assert not cuda_lib.aero_cuda_pages_open(ctypes.byref(desc()), err, 256) and b"no CUDA device" in err.value
    assert not cuda_lib.aero_cuda_pages_open(None, err, 256)
    torch = pytest.importorskip("torch")
    from aero_b200.logits import adjust
    from aero_b200.pages import PagedCache
    with pytest.raises(nc.CudaMoeUnavailable):
        PagedCache(1, 4, 16, 1, 64, 1, 2)
    with pytest.raises(nc.CudaMoeUnavailable):
        adjust(torch.zeros((1, 8)))


def test_null_handles(cuda_lib):
    assert cuda_lib.aero_cuda_pages_compact(None) == -1 and cuda_lib.aero_cuda_pages_status(None) == -1
    assert cuda_lib.aero_cuda_pages_buffers(None, None, None, None, None, None) == -1
    assert b"null" in cuda_lib.aero_cuda_pages_last_error(None)
    cuda_lib.aero_cuda_pages_close(None)
    host = np.zeros(8, np.float32)
    none = [None] * 8
    args = (host.ctypes.data, 8, 0, 1, 8, None, 0, *none, None, 0, host.ctypes.data, 8, None)
    assert cuda_lib.aero_cuda_logits_adjust(*args) == -1  # host memory (or no device at all)
