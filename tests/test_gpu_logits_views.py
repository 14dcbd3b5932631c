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


def long_lists(rows, vocab, per_row, dtype, seed, spread=1):
    """Lists of per_row biases a row, most tokens more than once, with histories and a mask."""
    import numpy as np
    r = np.random.default_rng(seed)
    x = torch.randn((rows, vocab), device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).mul_(4).to(dtype)
    history = r.integers(0, vocab, (rows, 300)).astype(np.int32)
    token = r.integers(-2, vocab // spread + 2, rows * per_row).astype(np.int32)
    value = r.normal(size=rows * per_row).astype(np.float32)
    mask = r.integers(-2**31, 2**31, (rows, (vocab + 31) // 32)).astype(np.int32)
    return x, dict(history=history, n_history=np.full(rows, 300, np.int32), n_prompt=np.full(rows, 100, np.int32),
                   repetition=np.full(rows, 1.25, np.float32), frequency=np.full(rows, 0.25, np.float32),
                   presence=np.full(rows, 0.5, np.float32), bias_start=np.arange(rows + 1, dtype=np.int32) * per_row,
                   bias_token=token, bias_value=value, mask=mask)


@pytest.mark.parametrize("rows,vocab,per_row,dtype,spread", [
    (1, 9000, 513, torch.float32, 8), (2, 9001, 2000, torch.float16, 2), (3, 5003, 12000, torch.float32, 1),
    (2, 40001, 3000, torch.bfloat16, 400), (1, 700, 9000, torch.float32, 1)])
def test_long_bias_lists_match_plain(rows, vocab, per_row, dtype, spread):
    """More biases in a slice than its place in shared memory holds. Tolerance as in test_gpu_logits.py:
    f32 sums of the values met, one rounding an addition, then the type's own."""
    import numpy as np

    from aero_b200.logits import adjust
    from test_gpu_logits import U, plain
    x, kw = long_lists(rows, vocab, per_row, dtype, 3, spread)
    dev = {k: torch.from_numpy(v).cuda() for k, v in kw.items()}
    got = adjust(x, **dev)
    want, mag = plain(x, kw["history"], kw["n_history"], kw["n_prompt"], kw["repetition"], kw["frequency"], kw["presence"],
                      kw["bias_start"], kw["bias_token"], kw["bias_value"], kw["mask"])
    g, off = got.double().cpu().numpy(), np.isinf(want)
    assert np.array_equal(np.isneginf(g), off)
    most = np.bincount(kw["bias_token"][kw["bias_token"] >= 0]).max()
    tol = U[dtype] * np.abs(want[~off]) + 8 * 2.0**-24 * (mag[~off] + 1) * (1 + most)
    assert (np.abs(g[~off] - want[~off]) <= tol).all()
    again = x.clone()
    assert adjust(again, out=again, **dev) is again and torch.equal(again, got)  # in place


def test_dense_biases_take_time_in_proportion():
    """A bias for every token of a vocabulary, against one for every eighth: no more than 16 times as long
    (each token searching the whole list takes 64 times as long)."""
    from aero_b200.logits import adjust
    took = []
    for per_row in (5000, 40000):
        x, kw = long_lists(4, 40000, per_row, torch.float32, 5)
        kw["bias_token"] = torch.arange(40000).repeat(4)[::40000 // per_row].int().numpy()
        dev = {k: torch.from_numpy(v).cuda() for k, v in kw.items()}
        best = 1e9
        for _ in range(4):
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record()
            adjust(x, **dev)
            e1.record()
            torch.cuda.synchronize()
            best = min(best, e0.elapsed_time(e1))
        took.append(best)
    assert took[1] < 16 * took[0] + 0.1
