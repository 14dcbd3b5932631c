"""Adjusted logits against a plain form in 64 bits.

Tolerance, from f32 arithmetic on f32 inputs: one rounding each for the quotient or
product, frequency times count, the two differences and the bias, each at most
2^-24 of the values met on the way; then the output type's own rounding.
"""

import math

import numpy as np
import pytest

from aero_b200 import native_cuda as nc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


@pytest.fixture(autouse=True)
def _gpu(cuda_lib):
    nc.require_gpu()


def plain(x, hist, n, n_prompt, rep, freq, pres, start, tok, val, mask):
    x = x.double().cpu().numpy().copy()
    mag = np.abs(x)
    B, V = x.shape
    for r in range(B):
        for v in sorted(set(int(t) for t in hist[r][:n[r]] if 0 <= t < V)) if hist is not None else []:
            y = x[r, v]
            x[r, v] = y / rep[r] if y > 0 else y * rep[r]
            c = sum(1 for t in hist[r][n_prompt[r]:n[r]] if t == v)
            mag[r, v] = max(mag[r, v], abs(x[r, v])) + (abs(freq[r]) * c + abs(pres[r]) if c else 0)
            if c:
                x[r, v] -= freq[r] * c + pres[r]
        for i in range(start[r], start[r + 1]) if start is not None else []:
            if 0 <= tok[i] < V:
                x[r, tok[i]] += val[i]
                mag[r, tok[i]] += abs(val[i])
        if mask is not None:
            for v in range(V):
                if not (int(mask[r, v // 32]) >> (v % 32)) & 1:
                    x[r, v] = -math.inf
    return x, mag


@pytest.mark.parametrize("rows,vocab,hist,nb,masked,dtype,seed", [
    (1, 1, 1, 1, True, torch.float32, 0), (3, 31, 40, 3, True, torch.float32, 1), (2, 8193, 700, 50, False, torch.float16, 2),
    (5, 1003, 0, 0, True, torch.bfloat16, 3), (4, 20001, 5000, 200, True, torch.float32, 4),
    (2, 16384, 333, 0, False, torch.bfloat16, 5), (1, 300, 2000, 33, True, torch.float16, 6)])
def test_adjust_matches_plain(rows, vocab, hist, nb, masked, dtype, seed):
    from aero_b200.logits import adjust
    r = np.random.default_rng(seed)
    wide = torch.randn((rows, vocab + 5), device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).mul_(4).to(dtype)
    x = wide[:, :vocab] if seed % 2 else wide[:, :vocab].contiguous()
    h = r.integers(-3, vocab + 3, (rows, hist)).astype(np.int32) if hist else None  # ids outside are passed over
    if hist > 10:
        h[:, 3:7] = vocab // 2
    n = r.integers(0, hist + 1, rows).astype(np.int32)
    n_prompt = (n // 2).astype(np.int32)
    rep, freq, pres = (r.uniform(a, b, rows).astype(np.float32) for a, b in ((0.8, 1.5), (-0.5, 0.5), (0, 0.5)))
    start = tok = val = None
    if nb:
        start = np.sort(np.concatenate([[0, nb], r.integers(0, nb + 1, rows - 1)])).astype(np.int32)
        tok = r.integers(-1, min(vocab, 20) + 1, nb).astype(np.int32)  # many twice
        val = r.normal(size=nb).astype(np.float32)
    mask = r.integers(-2**31, 2**31, (rows, (vocab + 31) // 32 + 1)).astype(np.int32) if masked else None
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    kw = dict(history=dev(h), n_history=dev(n) if hist else None, n_prompt=dev(n_prompt) if hist else None,
              repetition=dev(rep), frequency=dev(freq), presence=dev(pres), bias_start=dev(start), bias_token=dev(tok),
              bias_value=dev(val), mask=dev(mask))
    got = adjust(x, **kw)
    want, mag = plain(x, h, n, n_prompt, rep, freq, pres, start, tok, val, mask)
    g = got.double().cpu().numpy()
    off = np.isinf(want)
    assert np.array_equal(np.isneginf(g), off)
    tol = U[dtype] * np.abs(want[~off]) + 8 * 2.0**-24 * (mag[~off] + 1) * (1 + nb)
    assert (np.abs(g[~off] - want[~off]) <= tol).all()
    again = x.clone()
    assert adjust(again, out=again, **kw) is again and torch.equal(again, got)  # in place


def test_adjust_identity_and_special_values():
    from aero_b200.logits import adjust
    x = torch.tensor([[1.0, -math.inf, math.inf, math.nan, 0.0, -2.0]], device="cuda")
    assert torch.equal(adjust(x).nan_to_num(7.5), x.nan_to_num(7.5))
    one = lambda v, t=torch.int32: torch.tensor([v], dtype=t, device="cuda")  # noqa: E731
    y = adjust(x, history=torch.arange(6, dtype=torch.int32, device="cuda")[None], n_history=one(6), n_prompt=one(6),
               repetition=one(2.0, torch.float32), mask=torch.tensor([[0b110111]], dtype=torch.int32, device="cuda"))
    assert y[0, :3].tolist() == [0.5, -math.inf, math.inf] and y[0, 3] == -math.inf and y[0, 4:].tolist() == [0.0, -4.0]


def test_adjust_refusals():
    from aero_b200.logits import adjust
    x = torch.zeros((2, 40), device="cuda")
    h = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    for a, kw in ((x.cpu(), {}), (x.double(), {}), (x[0], {}), (x.t(), {}), (x, dict(history=h)), (x, dict(n_history=n)),
                  (x, dict(history=h.long(), n_history=n)), (x, dict(history=h[:1], n_history=n)),
                  (x, dict(repetition=n)), (x, dict(frequency=torch.zeros(3, device="cuda"))),
                  (x, dict(mask=h[:, :1])), (x, dict(bias_start=n)), (x, dict(out=x[:1]))):
        with pytest.raises(ValueError):
            adjust(a, **kw)
    lib = nc.lib()
    host = np.zeros(8, np.float32)
    none = [None] * 8
    assert lib.aero_cuda_logits_adjust(host.ctypes.data, 8, 0, 1, 8, None, 0, *none, None, 0, host.ctypes.data, 8, None) == -1
    assert "device memory" in nc.last_error()
    assert lib.aero_cuda_logits_adjust(x.data_ptr(), 39, 0, 2, 40, None, 0, *none, None, 0, x.data_ptr(), 40, None) == -1
    assert lib.aero_cuda_logits_adjust(x.data_ptr(), 40, 5, 2, 40, None, 0, *none, None, 0, x.data_ptr(), 40, None) == -1
