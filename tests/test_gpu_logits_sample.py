"""Tokens drawn from logits against a plain form in 64 bits.

A token is where the running sum of the weights passes u times their sum. The library's weights are multiples of
2^-b of the largest, so each is off by 2^-(b+1) and by some 2^-50 of itself: a sum of V of them by less than
V 2^-(b+1) + 2^-48 S = tol. A drawn token must be one whose interval of running sums holds u S to within 2 tol (u S and
the interval's end each off by tol); the end of what top_p keeps likewise, so where a limit lies
within 2 tol of a border either side of it is taken, and the checks below allow both. logprob: f32's rounding, half a step
2^-24 of the value, and the sum's tol relative to it (at least 1): 2^-24 |v| + 2^-26.
"""

import math

import numpy as np
import pytest

from aero_b200 import native_cuda as nc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_lib):
    nc.require_gpu()


def dev(x, dtype=torch.float32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def check_row(x, u, T, k, p, least, token, logp):
    """x: the row's values in 64 bits."""
    V = len(x)
    tol = V * 2.0 ** -(min(48, 62 - math.ceil(math.log2(max(V, 2)))) + 1) + 2.0**-48 * V
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not len(order):
        assert token == -1 and logp == -math.inf
        return
    if not T > 0:
        assert token == order[0] and logp == 0
        return
    v = x[order]
    with np.errstate(invalid="ignore"):
        log_w = np.where(v == v[0], 0.0, (v - v[0]) / T)
    log_w = np.where(np.isnan(log_w), -np.inf, log_w)
    w = np.exp(log_w)
    n = len(w) if k <= 0 else min(k, len(w))
    run = np.cumsum(w)
    ends = {n}
    if p < 1:
        first = run - w
        ends = {max(1, int(np.searchsorted(first[:n], p * run[n - 1] + d))) for d in (-2 * tol, 0, 2 * tol)}
    if least > 0:
        many = {max(1, int(np.count_nonzero(w >= least * (1 + d)))) for d in (-1e-13, 0, 1e-13)}
        ends = {min(a, b) for a in ends for b in many}
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    j = int(np.nonzero(order == token)[0][0])
    good = False
    for n in ends:
        S = run[n - 1]
        good |= j < n and (run[j] - w[j] <= u * S + 2 * tol) and (run[j] > u * S - 2 * tol or (u >= 1 and w[j] > 0 and run[j] >= S - 2 * tol)) \
            and abs(logp - (log_w[j] - math.log(S))) <= 2.0**-24 * abs(log_w[j] - math.log(S)) + 2.0**-26
    assert good, (j, ends, u, T, k, p, least, token, logp, run[j] - w[j], run[j])


def check(x, u, T=None, k=None, p=None, least=None):
    from aero_b200.logits import sample
    rows = x.shape[0]
    token, logp = sample(x, dev(u), temperature=None if T is None else dev(T), top_k=None if k is None else dev(k, torch.int32),
                         top_p=None if p is None else dev(p), min_p=None if least is None else dev(least), logprob=True)
    token, logp, xs = token.cpu().numpy(), logp.cpu().numpy().astype(np.float64), x.double().cpu().numpy()
    f = np.float32
    for r in range(rows):
        check_row(xs[r], float(f(u[r])), 1.0 if T is None else float(f(T[r])), 0 if k is None else k[r],
                  1.0 if p is None or math.isnan(p[r]) else float(f(p[r])), 0.0 if least is None or math.isnan(least[r]) else float(f(least[r])),
                  token[r], logp[r])
    return token


def logits(rows, vocab, dtype, seed, spread=2.0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.empty((rows, vocab), device="cuda").normal_(std=spread, generator=g)
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 20), device="cuda", generator=g), 12 * torch.rand((rows, 20), device="cuda", generator=g))
    return x.to(dtype)


LIMITS = [dict(), dict(T=0.7), dict(k=40), dict(p=0.9), dict(least=0.05), dict(T=1.3, k=50, p=0.95), dict(k=3000, p=0.8), dict(T=2.0, k=2000, least=0.01),
          dict(p=0.999, least=0.001, T=0.5), dict(k=5, p=0.5, least=0.3), dict(k=2, T=5.0), dict(k=1), dict(p=1e-6), dict(T=3.0, p=0.97)]


@pytest.mark.parametrize("rows,vocab,dtype,seed", [
    (1, 1, torch.float32, 0), (3, 2, torch.float16, 1), (5, 31, torch.bfloat16, 2), (2, 2047, torch.float32, 3),
    (4, 4097, torch.bfloat16, 4), (1, 8193, torch.float32, 5), (7, 32000, torch.float16, 6), (1, 151936, torch.float32, 7),
    (40, 50257, torch.bfloat16, 8), (160, 5003, torch.float32, 9), (3, 151936, torch.bfloat16, 10)])
@pytest.mark.parametrize("limits", LIMITS)
def test_sample_matches_plain(rows, vocab, dtype, seed, limits):
    x = logits(rows, vocab, dtype, seed)
    u = np.random.default_rng(seed).random(rows).astype(np.float32)
    u[0] = 0.0
    u[-1] = np.float32(1 - 2.0**-24)
    check(x, u.tolist(), **{n: [v] * rows for n, v in limits.items()})


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits(dtype):
    """Slices of the row with thousands of equal values: the answer by arithmetic, and the token by number."""
    V = 20011
    us = [0.0, 0.1, 0.5, 0.77, 1 - 2.0**-24]
    g = torch.Generator("cuda").manual_seed(3)
    same = torch.full((5, V), 1.5, device="cuda", dtype=dtype)
    two = torch.where(torch.rand((5, V), device="cuda", generator=g) < 0.3, 2.0, 1.0).to(dtype)
    steps = (torch.randint(0, 5, (5, V), device="cuda", generator=g) / 4 - 3).to(dtype)
    coarse = torch.randn((5, V), device="cuda", generator=g).bfloat16().to(dtype)
    huge = torch.full((5, V), 3e38, device="cuda", dtype=torch.float32)
    huge[:, ::2] = -3e38
    for x in (same, two, steps, coarse, huge):
        for limits in (dict(), dict(k=7777), dict(k=3), dict(p=0.4), dict(p=0.9, k=15000), dict(least=0.5), dict(p=0.3, least=0.9, T=0.1)):
            check(x, us, **{n: [v] * 5 for n, v in limits.items()})
    assert check(same, us) is not None and check(same, [0.0] * 5).tolist() == [0] * 5


@pytest.mark.parametrize("V", [32767, 32768, 40000, 65535, 65536, 65537, 100003, 131072, 151936, 300001, (1 << 20) + 7])
def test_flat_rows_of_many_tokens(V):
    """Sums as large as they can be: all weights the largest, or nearly."""
    u = [0.0, 0.3, 0.71, 1 - 2.0**-24]
    x = torch.full((4, V), 1.5, device="cuda")
    check(x, u)
    check(x, u, p=[0.9, 0.5, 1.0, 0.25], least=[1.0, 0.5, 0.0, 1e-9])
    check(x, u, k=[0, V - 1, 3000, 40000], T=[1e-3, 1.0, 9.0, 1e9])
    x += torch.rand(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(V)) * 1e-3
    check(x.to(torch.bfloat16), u, p=[0.99, 1.0, 0.6, 0.999])
    check(x, u, T=[1.0, 5.0, 0.1, 1e5])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [2500, 30011])
def test_no_numbers_among_tokens_nearly_alike(dtype, V):
    """Slices that hold thousands of tokens, positive and negative ones, of which only the numbers count."""
    T = [1.0, 30.0, 485.0, 1e5, 1e12]
    x = torch.randn((5, V), device="cuda", generator=torch.Generator("cuda").manual_seed(12))
    odd = torch.rand(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(13))
    x[odd < 0.1] = math.nan
    x[odd < 0.05] *= -1
    x[odd > 0.99] = -math.inf
    x = x.to(dtype)
    x.view(torch.int32 if dtype == torch.float32 else torch.int16)[:, 7::50] = -1  # no number, its sign set
    for u in (0.0, 0.5, 1 - 2.0**-24):
        for limits in (dict(), dict(k=1300), dict(k=V * 2 // 3), dict(p=0.7), dict(k=2000, p=0.4), dict(least=0.99)):
            check(x, [u] * 5, T=T, **{n: [v] * 5 for n, v in limits.items()})


def test_values_of_every_kind():
    V = 9001
    x = logits(12, V, torch.float32, 5)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, ::2] = -math.inf
    x[3, ::3] = math.nan
    x[4, 5] = math.inf
    x[5, 100:200] = math.inf
    x[6, ::2] = torch.finfo(torch.float32).min
    x[7] = -math.inf
    x[7, 4000] = -7.0
    x[8] *= 1e30
    x[9] *= 1e-42  # below the normal numbers
    x[10] = 0.0
    x[10, ::2] = -0.0
    x[11, 1:] = torch.finfo(torch.float32).min
    x[11, 0] = torch.finfo(torch.float32).max
    u = [0.3, 0.3, 0.9, 0.5, 0.5, 0.505, 0.99, 0.2, 0.6, 0.7, 0.37, 0.9]
    for limits in (dict(), dict(k=8000), dict(k=30), dict(p=0.7), dict(least=0.1), dict(T=1e9, p=0.9), dict(T=1e-3), dict(T=math.inf, k=4000)):
        got = check(x, u, **{n: [v] * 12 for n, v in limits.items()})
        assert got[0] == -1 and got[1] == -1 and got[4] == 5 and 100 <= got[5] < 200 and got[7] == 4000


def test_limits_of_every_kind_in_one_batch():
    """Each row its own limits, the odd ones of each kind among them."""
    V, inf, nan = 6001, math.inf, math.nan
    rows = [  # u, T, k, p, min_p
        (0.4, 0.0, 0, 1.0, 0.0), (0.4, -1.0, 5, 0.5, 0.1), (0.4, nan, 0, 1.0, 0.0), (0.4, 1e-38, 0, 1.0, 0.0), (0.4, inf, 0, 1.0, 0.0),
        (0.4, 1e30, 0, 0.5, 0.0), (0.4, 1.0, -3, 1.0, 0.0), (0.9, 1.0, 6001, 1.0, 0.0), (0.9, 1.0, 9999, 0.9, 0.0), (0.9, 4.0, 2048, 1.0, 0.0),
        (0.9, 4.0, 2049, 1.0, 0.0), (0.9, 4.0, 2047, 0.9, 0.0), (0.9, 1.0, 0, 0.0, 0.0), (0.9, 1.0, 0, -1.0, 0.0), (0.9, 1.0, 0, nan, 0.0),
        (0.9, 1.0, 0, 2.0, 0.0), (0.9, 1.0, 0, 1.0, 1.0), (0.9, 1.0, 0, 1.0, 5.0), (0.9, 1.0, 0, 1.0, nan), (0.9, 1.0, 0, 1.0, -1.0),
        (nan, 1.0, 0, 1.0, 0.0), (-0.5, 1.0, 0, 1.0, 0.0), (1.0, 1.0, 50, 1.0, 0.0), (7.0, 1.0, 50, 0.9, 0.0), (0.5, 1e-45, 0, 1.0, 0.0)]
    x = logits(len(rows), V, torch.float32, 9, spread=1.0)
    u, T, k, p, least = (list(c) for c in zip(*rows))
    got = check(x, u, T, k, p, least)
    for r in (0, 1, 2, 3, 12, 13, 16, 17, 24):
        assert got[r] == int(x[r].argmax())


def test_views_streams_and_replays():
    from aero_b200.logits import sample
    V = 7013
    wide = logits(6, V + 9, torch.float16, 4)
    x = wide[::2, 3:3 + V]  # rows that begin anywhere, lie apart
    u = [0.2, 0.6, 0.95]
    want = check(x, u, p=[0.9] * 3)
    assert sample(x.contiguous(), dev(u), top_p=dev([0.9] * 3)).tolist() == want.tolist()
    one = sample(x[0].expand(3, V), dev(u), top_p=dev([0.9] * 3))  # one row for all
    check(x[:1].expand(3, V).contiguous(), u, p=[0.9] * 3)
    assert one[0] == want[0]
    out = torch.full((3,), 7, dtype=torch.int32, device="cuda")
    assert sample(x, dev(u), top_p=dev([0.9] * 3), out=out) is out and out.tolist() == want.tolist()
    # on another stream, captured and replayed with other inputs
    xs, us, ps = x.contiguous(), dev(u), dev([0.9] * 3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        first = sample(xs, us, top_p=ps)
    s.synchronize()
    assert first.tolist() == want.tolist()
    with torch.cuda.graph(g, stream=s):
        sample(xs, us, top_p=ps, out=out)
    xs.copy_(logits(3, V, torch.float16, 77))
    us.fill_(0.5)
    g.replay()
    torch.cuda.synchronize()
    assert out.tolist() == check(xs, [0.5] * 3, p=[0.9] * 3).tolist()


def test_refusals():
    from aero_b200.logits import sample
    x, u = torch.zeros((2, 50), device="cuda"), torch.zeros(2, device="cuda")
    for bad in (lambda: sample(x.double(), u), lambda: sample(x[0], u), lambda: sample(x.T, u), lambda: sample(x.cpu(), u.cpu()),
                lambda: sample(x, None), lambda: sample(x, u[:1]), lambda: sample(x, u.double()), lambda: sample(x, u.cpu()),
                lambda: sample(x, u, temperature=u.half()), lambda: sample(x, u, top_k=u), lambda: sample(x, u, top_p=u.cpu()),
                lambda: sample(x, u, min_p=torch.zeros(4, device="cuda")[::2]), lambda: sample(x, u, out=torch.zeros(2, device="cuda")),
                lambda: sample(x[:, :0], u), lambda: sample(x[:1].expand(2, 50)[:, :1].expand(2, (1 << 22) + 1), u)):
        with pytest.raises(ValueError):
            bad()
    assert sample(x[:0], u[:0]).shape == (0,)
    token, logp = sample(x[:0], u[:0], logprob=True)
    assert token.numel() == 0 and logp.numel() == 0
