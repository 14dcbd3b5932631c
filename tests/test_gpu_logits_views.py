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


def exact_adjust(x, kw):
    """The definition in 64 bits on the GPU: the adjusted logits, and the largest values met on the way."""
    rows, vocab = x.shape
    y = x.double()
    at = torch.arange(kw["history"].shape[1], device="cuda")[None, :]
    ids = kw["history"].long()
    inside = (at < kw["n_history"][:, None]) & (ids >= 0) & (ids < vocab)

    def counted(keep):
        return torch.zeros((rows, vocab), dtype=torch.float64, device="cuda").scatter_add_(1, ids.clamp(0, vocab - 1), keep.double())

    there, c = counted(inside) > 0, counted(inside & (at >= kw["n_prompt"][:, None]))
    rep, fr, pr = (kw[n].double()[:, None] for n in ("repetition", "frequency", "presence"))
    mag = y.abs() * torch.maximum(rep, 1 / rep)
    y = torch.where(there, torch.where(y > 0, y / rep, y * rep), y)
    y = torch.where(c > 0, y - fr * c - pr, y)
    mag = mag + fr.abs() * c + pr.abs()
    most = 1
    for r in range(rows):
        t = kw["bias_token"][int(kw["bias_start"][r]):int(kw["bias_start"][r + 1])].long()
        v = kw["bias_value"][int(kw["bias_start"][r]):int(kw["bias_start"][r + 1])].double()
        t, v = t[(t >= 0) & (t < vocab)], v[(t >= 0) & (t < vocab)]
        y[r].scatter_add_(0, t, v)
        mag[r].scatter_add_(0, t, v.abs())
        most = max(most, int(torch.bincount(t).max()) if t.numel() else 0)
    bit = torch.arange(vocab, device="cuda")
    allowed = (kw["mask"][:, bit // 32] >> (bit % 32).int()) & 1
    return torch.where(allowed.bool(), y, torch.full_like(y, -float("inf"))), mag, most


@pytest.mark.parametrize("rows,vocab,width,per_row,dtype", [
    (64, 151937, 300, 8, torch.float32), (64, 151937, 300, 8, torch.bfloat16), (40, 100001, 2000, 64, torch.float16),
    (70, 152064, 40000, 5, torch.float32), (3, 50001, 70000, 600, torch.bfloat16), (1, 33, 33000, 40, torch.float16),
    (2, 262145, 50, 0, torch.float32)])
def test_large_calls_match_plain(rows, vocab, width, per_row, dtype):
    """Slices of several trips with a remainder, vocabularies that are no multiple of a vector, notes of 32
    bits (histories wider than 32767, one token repeated more often than 16 bits count), more rows than
    slices. Tolerance as in test_gpu_logits.py."""
    from aero_b200.logits import adjust
    from test_gpu_logits import U
    g = torch.Generator("cuda").manual_seed(vocab + width)
    x = torch.randn((rows, vocab), device="cuda", generator=g).mul_(4).to(dtype)
    history = torch.randint(-2, vocab + 2, (rows, width), device="cuda", generator=g, dtype=torch.int32)
    if width > 32767:
        history[:, 100:34000] = vocab // 3  # (33900 times)
        history[-1, :200] = vocab - 1
    n = torch.randint(width // 2, width + 1, (rows,), device="cuda", generator=g, dtype=torch.int32)
    n[0] = width
    kw = dict(history=history, n_history=n, n_prompt=torch.div(n, 3, rounding_mode="floor").int(),
              repetition=0.8 + 0.7 * torch.rand(rows, device="cuda", generator=g),
              frequency=torch.rand(rows, device="cuda", generator=g) / 64, presence=torch.rand(rows, device="cuda", generator=g),
              bias_start=torch.arange(rows + 1, device="cuda", dtype=torch.int32) * per_row,
              bias_token=torch.randint(-1, vocab + 1, (rows * per_row,), device="cuda", generator=g, dtype=torch.int32),
              bias_value=torch.randn(rows * per_row, device="cuda", generator=g),
              mask=torch.randint(-2**31, 2**31, (rows, (vocab + 31) // 32), device="cuda", generator=g).int())
    got = adjust(x, **kw)
    want, mag, most = exact_adjust(x, kw)
    off = torch.isinf(want)
    assert torch.equal(torch.isneginf(got), off) and bool(off.any())
    err = (got.double() - want).abs()[~off]
    tol = (U[dtype] * want.abs() + 8 * 2.0**-24 * (mag + 1) * (1 + most))[~off]
    assert (err <= tol).all(), float((err / tol).max())
    again = x.clone()
    assert adjust(again, out=again, **kw) is again and torch.equal(again, got)
