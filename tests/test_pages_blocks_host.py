"""The entry points of block selection and sampling without a GPU: plans and refusals."""

import ctypes

import numpy as np
import pytest

from aero_b200 import native_cuda as nc


def test_bounds_bytes(cuda_lib):
    d = nc.PagesDesc(2, 10, 16, 4, 128, 3, 5, nc.TYPE_F16, 0, 0)
    assert cuda_lib.aero_cuda_pages_bounds_bytes(ctypes.byref(d)) == 2 * 10 * 4 * 2 * 128 * 2
    bad = nc.PagesDesc(2, 10, 17, 4, 128, 3, 5, nc.TYPE_F16, 0, 0)
    assert cuda_lib.aero_cuda_pages_bounds_bytes(ctypes.byref(bad)) == -1
    assert cuda_lib.aero_cuda_pages_bounds_bytes(None) == -1
    from aero_b200.pages import plan_bytes
    with_bounds, without = plan_bytes(2, 10, 16, 4, 128, 3, 5, bounds=True), plan_bytes(2, 10, 16, 4, 128, 3, 5)
    assert with_bounds["kv_cache"] - without["kv_cache"] == with_bounds["total"] - without["total"] == 2 * 10 * 4 * 2 * 128 * 2


def test_null_handles(cuda_lib):
    assert cuda_lib.aero_cuda_pages_keep_bounds(None) == -1 and cuda_lib.aero_cuda_pages_bounds(None) is None
    assert cuda_lib.aero_cuda_pages_set_bounds(None, 0, None, 0) == -1
    assert cuda_lib.aero_cuda_pages_select(None, 0, None, 0, 0, 0, 1, None, None, 0, 1, 1, 4, None) == -1
    assert cuda_lib.aero_cuda_pages_attend_blocks(None, 0, None, 0, 0, 0, 1, None, None, 0, None, 1, 1.0, None, 0, 0) == -1


def sample_args(**kw):
    host = kw.pop("host")
    a = dict(logits=host, ld=8, dtype=nc.TYPE_F32, rows=1, vocab=8, u=host, temperature=None, top_k=None, top_p=None, min_p=None,
             tokens=host, logprob=None, stream=None)
    a.update(kw)
    return a.values()


@pytest.mark.parametrize("bad,why", [
    (dict(dtype=8), b"F32"), (dict(rows=-1), b"rows"), (dict(rows=(1 << 20) + 1), b"rows"), (dict(vocab=0), b"vocab"),
    (dict(vocab=(1 << 22) + 1), b"vocab"), (dict(ld=-1), b"ld"), (dict(logits=None), b"device memory"), (dict(), b"device memory")])
def test_sample_refuses(cuda_lib, bad, why):
    host = np.zeros(16, np.float32)
    assert cuda_lib.aero_cuda_logits_sample(*sample_args(host=host.ctypes.data, **bad)) == -1
    assert why in cuda_lib.aero_cuda_moe_last_error(None)


def test_sample_of_no_rows(cuda_lib):
    host = np.zeros(16, np.float32)
    assert cuda_lib.aero_cuda_logits_sample(*sample_args(host=host.ctypes.data, rows=0)) == 0


def test_sample_needs_a_gpu(cuda_lib):
    if nc.gpu_count() > 0:
        pytest.skip("a GPU is visible")
    torch = pytest.importorskip("torch")
    from aero_b200.logits import sample
    with pytest.raises(nc.CudaMoeUnavailable):
        sample(torch.zeros((1, 8)), torch.zeros(1))
