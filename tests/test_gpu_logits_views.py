"""Adjusted logits of calls on views: histories and masks narrower than the rows they are cut from,
shared by all rows, or overlapping. What such a call gives is what copies of its arguments give, to
the bit: the values and the order of every operation are the same."""

import pytest

from aero_b200 import native_cuda as nc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_lib):
    nc.require_gpu()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def f32(x):
    return torch.tensor(x, dtype=torch.float32, device="cuda")


def penalties(rows):
    return dict(repetition=f32([1.3 + 0.1 * r for r in range(rows)]), frequency=f32([0.25] * rows), presence=f32([0.5] * rows))


@pytest.mark.parametrize("rows,width,first", [(3, 4, 2), (1, 4, 0), (2, 1, 5), (4, 9, 1)])
def test_history_counts_no_tokens_outside_the_view(rows, width, first):
    """n_history larger than the view is wide: the tokens beside the view do not count, in a batch as
    in a row alone."""
    from aero_b200.logits import adjust
    vocab = 200
    x = torch.randn((rows, vocab), device="cuda")
    # (one row more than the view: what lies behind its last row is this test's own)
    wide = torch.arange((rows + 1) * 16, dtype=torch.int32, device="cuda").reshape(rows + 1, 16)
    view = wide[:rows, first:first + width]
    kw = dict(n_history=i32([16] * rows), n_prompt=i32([width // 2] * rows), **penalties(rows))
    got = adjust(x, history=view, **kw)
    assert torch.equal(got, adjust(x, history=view.clone(), **{**kw, "n_history": i32([width] * rows)}))
    changed = (got != x).nonzero().tolist()
    assert changed and all(v in view[r].tolist() for r, v in changed)
    for r in range(rows):
        one = {k: v[r:r + 1] for k, v in kw.items()}
        assert torch.equal(adjust(x[r:r + 1], history=view[r:r + 1], **one), got[r:r + 1])


def test_shared_and_overlapping_rows():
    """One history and one mask for all rows (stride 0), and histories that overlap."""
    from aero_b200.logits import adjust
    rows, vocab = 3, 70
    x = torch.randn((rows, vocab), device="cuda")
    tokens = i32([[5, 6, 7, 8, 5, 69, 64, 31, 32]])
    bits = i32([[0x5A5A5A5A, -0x12345678, 0x3F]])
    kw = dict(n_history=i32([9, 3, 0]), n_prompt=i32([2, 3, 0]), **penalties(rows))
    got = adjust(x, history=tokens.expand(rows, -1), mask=bits.expand(rows, -1), **kw)
    assert torch.equal(got, adjust(x, history=tokens.repeat(rows, 1), mask=bits.repeat(rows, 1), **kw))
    sliding = tokens[0].as_strided((rows, 6), (1, 1))
    assert torch.equal(adjust(x, history=sliding, **kw), adjust(x, history=torch.stack(list(sliding)), **kw))


@pytest.mark.parametrize("start", [[0, 3, 9], [-4, 2, 5], [0, 5, 2**30], [4, 1, 5], [7, 9, 9], [-9, -3, 1], [-2**31, 2**31 - 1, 0]])
def test_bias_offsets_outside_the_list(start):
    """Offsets that begin before the list, end behind it or descend: what lies in the list counts, and
    nothing beside it."""
    from aero_b200.logits import adjust
    rows, vocab, first, n = len(start) - 1, 50, 6, 5
    x = torch.randn((rows, vocab), device="cuda")
    token, value = torch.arange(20, dtype=torch.int32, device="cuda"), torch.full((20,), 8.0, device="cuda")
    got = adjust(x, bias_start=i32(start), bias_token=token[first:first + n], bias_value=value[first:first + n])
    want = x.clone()
    for r in range(rows):
        for i in range(max(start[r], 0), min(start[r + 1], n)):
            want[r, first + i] += 8.0
    assert torch.equal(got, want)
