"""The paged cache where its calls meet one another's state and incomplete books: shared pages, lists
that name what is not there, tables with holes, values that are not finite, weights of many small
parts, streams. Tolerances of outputs are those of test_gpu_pages.py, derived there."""

import math

import pytest

from aero_b200 import native_cuda as nc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _gpu(cuda_lib):
    nc.require_gpu()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda").reshape(-1)


# ------------------------------------------------------------------ books
@pytest.mark.parametrize("D,shift", [(64, 0), (64, 1), (128, 0)])
def test_append_leaves_shared_pages_alone(D, shift):
    """Rows for a full page that a fork shares are skipped, with a code; rows for the sequences' own
    pages, in the same call, are written; when the last but one holder is gone, so is the refusal."""
    from aero_b200.pages import PagedCache
    c = PagedCache(2, 12, 8, 2, D, 3, 4, dtype=F16)
    c.k().normal_()
    c.v().normal_()
    c.extend(i32([0]), i32([19]))  # two full pages and three rows of a third
    c.fork(i32([0]), i32([1]))
    c.extend(i32([0, 1]), i32([1, 1]))
    c.check()
    table = c.tables()[0].tolist()
    assert table[0][:2] == table[1][:2] and table[0][2] != table[1][2]
    k, v = (torch.randn((4, 2, D + shift), device="cuda").to(F16)[..., shift:] for _ in range(2))
    seqs, pos = [0, 1, 0, 1], [3, 15, 19, 19]
    want = c.k().clone(), c.v().clone()
    for t in (2, 3):
        for w, x in zip(want, (k, v)):
            w[1, table[seqs[t]][2], :, 3] = x[t]
    c.append(1, k, v, i32(seqs), i32(pos))
    assert c.status() == 8
    assert torch.equal(c.k(), want[0]) and torch.equal(c.v(), want[1])
    c.free(i32([1]))
    c.append(1, k[:1], v[:1], i32([0]), i32([3]))
    c.check()
    assert torch.equal(c.k(1)[table[0][0], :, 3], k[0]) and torch.equal(c.v(1)[table[0][0], :, 3], v[0])
