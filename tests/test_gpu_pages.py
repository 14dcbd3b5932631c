"""The paged key/value cache: attention over its pages against a plain form in 64 bits, the
books and page moves against a model in Python, and what the calls refuse.

Tolerance of an attention output, from the roundings the kernels make: u|o| for the
output's own rounding (u = 2^-11 in f16, 2^-8 in bf16); u sum w|v| for the
probabilities' rounding before they meet V; 2^-14 sum w|v| for scores, exponentials and
sums in f32 (|score| up to about 30 with an error of some 2^-21 of it); and in f16, whose
smallest step is 2^-24, 2^-25 sum |v| / l for probabilities below 2^-14.
"""

import math
import random

import numpy as np
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


def open_cache(lens, P, HK, D, dtype, *, layers=1, spare=3, seed=0, extra_rows=0):
    """A cache whose pool is NaN but for the rows that the sequences of lengths `lens` hold
    (normal values), their pages scattered. Returns (cache, K, V): lists of (length, HK, D)
    tensors for layer `layers - 1`."""
    from aero_b200.pages import PagedCache
    r = random.Random(seed)
    n = len(lens)
    used = [-(-x // P) for x in lens]
    n_page, width = sum(used) + spare, max([1, *used]) + 1
    c = PagedCache(layers, n_page, P, HK, D, n + extra_rows, width, dtype=dtype)
    c.k().fill_(math.nan)
    c.v().fill_(math.nan)
    order = list(range(n_page))
    r.shuffle(order)
    table = np.full((n + extra_rows, width), -1, np.int32)
    refs = np.zeros(n_page, np.int32)
    for s, u in enumerate(used):
        for i in range(u):
            table[s, i] = order.pop()
            refs[table[s, i]] = 1
    c.set_tables(torch.from_numpy(table).cuda(), i32(list(lens) + [0] * extra_rows), i32(refs))
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 1)
    T = sum(lens)
    k = torch.randn((T, HK, D), device="cuda", generator=g).to(dtype)
    v = torch.randn((T, HK, D), device="cuda", generator=g).to(dtype)
    seqs = i32([s for s, x in enumerate(lens) for _ in range(x)])
    pos = i32([i for x in lens for i in range(x)])
    c.append(layers - 1, k, v, seqs, pos)
    c.check()
    return c, list(k.split(lens)), list(v.split(lens))


def reference(q, K, V, positions, window, sinks, scale):
    """q (t, H, D) at `positions` over one sequence's K, V (n, HK, D), all in 64 bits: the
    output, sum w|v|, and sum |v| / l (see the tolerance)."""
    t, H, D = q.shape
    n, HK = K.shape[0], K.shape[1]
    out = torch.zeros((t, H, D), dtype=torch.float64, device="cuda")
    mag, tiny = torch.zeros_like(out), torch.zeros_like(out)
    for i in range(t):
        p = positions[i]
        see = torch.tensor([j for j in range(n) if j <= p and (not window or j > p - window or j < sinks)], device="cuda",
                           dtype=torch.long)
        if not see.numel():
            continue
        Ks, Vs = K[see].double(), V[see].double()
        for h in range(H):
            s = (Ks[:, h // (H // HK)] @ q[i, h].double()) * scale
            e = torch.exp(s - s.max())
            w = e / e.sum()
            v = Vs[:, h // (H // HK)]
            out[i, h] = w @ v
            mag[i, h] = w @ v.abs()
            tiny[i, h] = v.abs().sum(0) / e.sum()
    return out, mag, tiny


def close(got, ref, dtype):
    out, mag, tiny = ref
    u = 2.0**-11 if dtype == F16 else 2.0**-8
    tol = u * out.abs() + (u + 2.0**-14) * mag + (2.0**-25 * tiny if dtype == F16 else 0) + 2.0**-24
    err = (got.double() - out).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.3f} of the tolerance"


def join(refs):
    return tuple(torch.cat([r[i] for r in refs]) for i in range(3))


# ------------------------------------------------------------------ one token a sequence
DECODE = [
    # lens, page, HK, G, D, dtype, window, sinks
    ([1], 8, 1, 1, 64, F16, 0, 0),
    ([0, 1, 2, 63, 64, 65, 0], 8, 2, 3, 64, BF16, 0, 0),
    ([700, 5, 129], 16, 4, 8, 128, F16, 0, 0),
    ([1000, 999, 128], 64, 1, 16, 128, BF16, 0, 0),
    ([3000], 32, 2, 4, 128, F16, 0, 0),
    ([513, 77, 300], 128, 2, 5, 192, F16, 0, 0),
    ([260, 1, 257, 512], 256, 2, 7, 256, BF16, 0, 0),
    ([1500, 20], 16, 2, 8, 256, F16, 0, 0),
    # windows and first tokens: longer and shorter than the sequence, ends inside a tile
    ([700, 5, 129, 64], 16, 2, 4, 128, F16, 1, 0),
    ([700, 5, 129, 64], 16, 2, 4, 128, BF16, 64, 4),
    ([2000, 100, 333], 8, 2, 2, 64, F16, 100, 1),
    ([2000, 100, 333], 64, 2, 16, 128, F16, 130, 200),
    ([900, 450], 32, 1, 6, 256, BF16, 33, 65),
    ([900, 450], 32, 2, 3, 192, BF16, 4096, 4),
]


@pytest.mark.parametrize("lens,P,HK,G,D,dtype,window,sinks", DECODE)
def test_decode_matches_plain(lens, P, HK, G, D, dtype, window, sinks):
    c, K, V = open_cache(lens, P, HK, D, dtype)
    # keys that no token of the call sees may hold anything
    table = c.tables()[0]
    for s, n in enumerate(lens):
        for j in range(n):
            if window and j <= n - 1 - window and j >= sinks:
                c.k(0)[int(table[s, j // P]), :, j % P] = math.inf
                c.v(0)[int(table[s, j // P]), :, j % P] = math.nan
    q = (2 * torch.randn((len(lens), HK * G, D), device="cuda")).to(dtype)
    seqs = list(range(len(lens)))[::-1]
    out = c.attend(0, q, i32(seqs), window=window, sinks=sinks)
    c.check()
    sc = 1 / math.sqrt(D)
    close(out, join([reference(q[i:i + 1], K[s], V[s], [lens[s] - 1], window, sinks, sc) for i, s in enumerate(seqs)]), dtype)
    for i, s in enumerate(seqs):
        if lens[s] == 0:
            assert (out[i] == 0).all()
    # the same call again: the same bits (what is split is joined in one order)
    assert torch.equal(out, c.attend(0, q, i32(seqs), window=window, sinks=sinks))


def test_decode_listed_twice_and_strides():
    c, K, V = open_cache([300, 70], 16, 2, 128, F16)
    wide = torch.randn((4, 9, 131), device="cuda").to(F16)
    q = wide[:, 1:9, 1:129]  # rows that start on no 16-byte (nor 4-byte) boundary
    out = torch.zeros((4, 8, 130), device="cuda", dtype=F16)[:, :, 1:129]
    seqs = [1, 0, 1, 1]
    c.attend(0, q, i32(seqs), out=out, scale=0.3)
    c.check()
    close(out, join([reference(q[i:i + 1], K[s], V[s], [[300, 70][s] - 1], 0, 0, 0.3) for i, s in enumerate(seqs)]), F16)
    even = torch.randn((8, 4, 128), device="cuda").to(F16).transpose(0, 1)  # heads in front of tokens
    got = c.attend(0, even, i32(seqs))
    assert torch.equal(got, c.attend(0, even.contiguous(), i32(seqs)))


def test_decode_large_scores():
    """Scores far apart: all the weight on one key, none lost to an early maximum."""
    c, K, V = open_cache([500], 16, 1, 64, F16)
    q = (60 * torch.randn((1, 4, 64), device="cuda")).to(F16)
    out = c.attend(0, q, i32([0]))
    o, mag, tiny = reference(q, K[0], V[0], [499], 0, 0, 0.125)
    # scores of some hundreds have an f32 error of about 2^-15, and so have the weights
    close(out, (o, mag * (1 + 2.0**-14 / 2.0**-11), tiny), F16)


def test_decode_many_sequences():
    """More sequences than threads, of all lengths: every CTA begins somewhere in the middle."""
    r = random.Random(5)
    lens = [r.choice([0, 1, 17, 64, 200, 700]) for _ in range(400)]
    c, K, V = open_cache(lens, 16, 2, 64, BF16)
    q = torch.randn((400, 4, 64), device="cuda").to(BF16)
    out = c.attend(0, q, i32(range(400)))
    c.check()
    pick = list(range(0, 400, 13))
    close(out[pick], join([reference(q[s:s + 1], K[s], V[s], [lens[s] - 1], 0, 0, 0.125) for s in pick]), BF16)
    assert all((out[s] == 0).all() for s in range(400) if lens[s] == 0)


# ------------------------------------------------------------------ several tokens a sequence
PROMPT = [
    # lens, new tokens of each (its last ones), page, HK, G, D, dtype, window, sinks
    ([1], [1], 8, 1, 1, 64, F16, 0, 0),
    ([5, 64, 65, 128, 129, 3], [5, 64, 1, 128, 129, 0], 8, 2, 3, 64, BF16, 0, 0),
    ([300, 200], [300, 7], 16, 2, 8, 128, F16, 0, 0),
    ([257, 511, 40], [257, 260, 40], 64, 1, 16, 128, BF16, 0, 0),
    ([600], [130], 128, 2, 1, 128, F16, 0, 0),
    ([300, 90], [200, 90], 32, 2, 5, 192, BF16, 0, 0),
    ([300, 90], [300, 3], 256, 1, 4, 256, F16, 0, 0),
    ([700, 300], [300, 300], 16, 1, 4, 128, F16, 1, 0),
    ([700, 300], [400, 300], 16, 2, 4, 128, BF16, 64, 4),
    ([900, 150], [500, 150], 64, 1, 8, 64, F16, 200, 1),
    ([900, 150], [300, 150], 8, 2, 2, 128, F16, 130, 300),
    ([700, 33], [140, 33], 32, 1, 6, 256, BF16, 100, 129),
    # few rows over long caches: split over CTAs and joined, one with a part that sees nothing
    ([4000], [33], 64, 1, 8, 128, F16, 0, 0),
    ([3000, 200], [40, 5], 16, 2, 3, 64, BF16, 0, 0),
    ([2500, 50], [30, 4], 32, 1, 4, 256, F16, 0, 0),
    ([3000], [260], 16, 1, 1, 192, BF16, 700, 40),
    # few tokens: one by one
    ([700, 90, 64], [9, 20, 1], 8, 2, 8, 128, F16, 0, 0),
    ([700, 90, 64, 5], [2, 1, 1, 0], 16, 1, 4, 192, BF16, 100, 4),
]


@pytest.mark.parametrize("lens,new,P,HK,G,D,dtype,window,sinks", PROMPT)
def test_prompt_matches_plain(lens, new, P, HK, G, D, dtype, window, sinks):
    c, K, V = open_cache(lens, P, HK, D, dtype)
    q = (2 * torch.randn((sum(new), HK * G, D), device="cuda")).to(dtype)
    start = [0]
    for x in new:
        start.append(start[-1] + x)
    out = c.attend(0, q, i32(range(len(lens))), i32(start), window=window, sinks=sinks)
    c.check()
    r = random.Random(1)
    rows, refs = [], []
    for s, (n, x) in enumerate(zip(lens, new)):
        # the first, the last, those at tiles' edges and some others
        pick = sorted(set(t for t in [0, 1, 15, 16, 31, 32, 63, 64, 127, 128, x - 1, *[r.randrange(max(x, 1)) for _ in range(12)]]
                          if 0 <= t < x))
        if pick:
            rows += [start[s] + t for t in pick]
            refs.append(reference(q[[start[s] + t for t in pick]], K[s], V[s], [n - x + t for t in pick], window, sinks,
                                  1 / math.sqrt(D)))
    close(out[rows], join(refs), dtype)
    assert torch.equal(out, c.attend(0, q, i32(range(len(lens))), i32(start), window=window, sinks=sinks))


def test_prompt_masked_places_hold_anything():
    """Rows that a token does not see (later tokens, what left its window) are infinite or
    no numbers; the tokens that do not see them come out as without them."""
    lens, new, P, HK, G, D, window, sinks = [500], [300], 16, 2, 4, 128, 100, 3
    c, K, V = open_cache(lens, P, HK, D, F16)
    q = torch.randn((300, HK * G, D), device="cuda").to(F16)
    want = c.attend(0, q, i32([0]), i32([0, 300]), window=window, sinks=sinks)
    table = c.tables()[0]
    for j, kv in ((50, math.nan), (410, math.nan), (333, math.inf)):
        c.k(0)[int(table[0, j // P]), :, j % P] = kv
        c.v(0)[int(table[0, j // P]), :, j % P] = kv
    got = c.attend(0, q, i32([0]), i32([0, 300]), window=window, sinks=sinks)
    c.check()
    pos = torch.arange(200, 500, device="cuda")
    clean = torch.ones(300, dtype=torch.bool, device="cuda")
    for j in (410, 333):
        clean &= (pos < j) | (pos - j >= window)
    assert int(clean.sum()) == 300 - 90 - 100 + 23
    tol = 2 * (2.0**-11 + 2.0**-14) * float(V[0].abs().max())  # both within their tolerance of the same number
    assert torch.isfinite(got[clean]).all() and (got[clean] - want[clean]).abs().max() <= tol
    assert not torch.isfinite(got[~clean]).any()


@pytest.mark.parametrize("dtype,bad", [(F16, math.nan), (BF16, math.nan), (F16, math.inf), (BF16, -math.inf)])
def test_keys_that_are_no_numbers(dtype, bad):
    """One key at a time not finite, V finite: a token that sees it has no result (infinite
    scores of both signs, or none), the others theirs."""
    c, K, V = open_cache([300], 16, 1, 64, dtype)
    q = (torch.rand((40, 2, 64), device="cuda") + 0.5).to(dtype)  # scores of an infinite key: infinite
    for j in (270, 279, 285, 291):
        row = c.k(0)[int(c.tables()[0][0, j // 16]), :, j % 16]
        keep = row.clone()
        row.fill_(bad)
        many = c.attend(0, q, i32([0]), i32([0, 40]))
        one = c.attend(0, q[39:], i32([0]))
        k = K[0].clone()
        row.copy_(keep)
        want = reference(q[:j - 260], k, V[0], list(range(260, j)), 0, 0, 0.125)
        close(many[:j - 260], want, dtype)
        if bad == -math.inf:  # scores of -inf: a weight of 0
            k = torch.cat([k[:j], k[j + 1:]])
            v = torch.cat([V[0][:j], V[0][j + 1:]])
            close(many[j - 260:], reference(q[j - 260:], k, v, list(range(j - 1, 299)), 0, 0, 0.125), dtype)
            close(one, reference(q[39:], k, v, [298], 0, 0, 0.125), dtype)
        else:
            assert not torch.isfinite(many[j - 260:]).any() and not torch.isfinite(one).any()
    c.check()


@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_prompt_repeats_with_growing_maxima(D):
    """Rows whose maxima grow from tile to tile (O rescaled often), again and again: the same
    result, and no device wait that gives up."""
    for T, n in ((303, 303), (40, 900), (64, 100), (130, 129 + 130)):
        c, K, V = open_cache([n], 64, 1, D, F16)
        c.k().mul_(torch.linspace(0.1, 6, c.n_page * 64, device="cuda").reshape(1, -1, 1, 64, 1).half())
        q = (3 * torch.randn((T, 4, D), device="cuda")).half()
        first = c.attend(0, q, i32([0]), i32([0, T]))
        for _ in range(40):
            again = c.attend(0, q, i32([0]), i32([0, T]))
        c.check()
        assert torch.equal(again, first) and torch.isfinite(first).all()


def test_prompt_strides_and_bad_rows():
    c, K, V = open_cache([150, 60], 16, 2, 64, BF16)
    wide = torch.randn((101, 9, 67), device="cuda").to(BF16)
    q = wide[:, 1:9, 3:67]
    out = torch.zeros((101, 8, 66), device="cuda", dtype=BF16)[:, :, 1:65]
    c.attend(0, q, i32([1, 0]), i32([0, 31, 101]), out=out)
    assert torch.equal(out, c.attend(0, q.contiguous(), i32([1, 0]), i32([0, 31, 101])))
    close(out[[0, 30, 31, 100]], join([reference(q[[0, 30]], K[1], V[1], [29, 59], 0, 0, 0.125),
                                       reference(q[[31, 100]], K[0], V[0], [80, 149], 0, 0, 0.125)]), BF16)
    assert c.status() == 0
    few, table = q[:31].contiguous(), i32([1, 0])
    for start in ([0, 31, 32], [1, 20, 31], [0, 25, 20]):
        c.attend(0, few, table, i32(start))
        assert c.status() == 6, start
    for start in ([0, 90, 101], [0, 40, 30], [5, 31, 101], [0, 31, 100]):  # more tokens than positions; not ascending; ends
        c.attend(0, q, i32([1, 0]), i32(start))
        assert c.status() == 6, start
    c.attend(0, q, i32([1, 9]), i32([0, 31, 101]))
    assert c.status() in (1, 6)  # no such sequence, so no positions either


def test_offsets_past_32_bits():
    """A pool of 5 GB for K alone; the rows read lie at its end."""
    from aero_b200.pages import PagedCache
    P, HK, D = 256, 8, 256
    c = PagedCache(5, 1024, P, HK, D, 1, 4, dtype=F16)
    assert c.k().numel() * 2 > 5 * 10**9
    table = torch.tensor([[1023, 1020, 1022, -1]], dtype=torch.int32, device="cuda")
    refs = torch.zeros(1024, dtype=torch.int32, device="cuda")
    refs[[1023, 1020, 1022]] = 1
    n = 700
    c.set_tables(table, i32([n]), refs)
    k, v = (torch.randn((n, HK, D), device="cuda").to(F16) for _ in range(2))
    c.append(4, k, v, i32([0] * n), i32(range(n)))
    q = torch.randn((1, 16, D), device="cuda").to(F16)
    close(c.attend(4, q, i32([0])), reference(q, k, v, [n - 1], 0, 0, 1 / 16), F16)
    c.copy(i32([1020]), i32([3]))
    c.compact()
    assert c.tables()[0][0, :3].tolist() == [2, 0, 1]
    assert torch.equal(c.attend(4, q, i32([0])), c.attend(4, q, i32([0])))
    close(c.attend(4, q, i32([0])), reference(q, k, v, [n - 1], 0, 0, 1 / 16), F16)
    c.check()


# ------------------------------------------------------------------ the books
class Books:
    """The books as the header defines them, one list operation at a time."""

    def __init__(self, n_seq, max_pages, n_page, P):
        self.P, self.width = P, max_pages
        self.table = [[-1] * max_pages for _ in range(n_seq)]
        self.length, self.refs = [0] * n_seq, [0] * n_page

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def extend(self, seqs, counts):
        need = sum(-(-(self.length[s] + x) // self.P) - -(-self.length[s] // self.P) for s, x in zip(seqs, counts))
        if len(set(seqs)) != len(seqs) or any(not 0 <= s < len(self.length) for s in seqs):
            return 1
        if any(x < 0 or self.length[s] + x > self.width * self.P for s, x in zip(seqs, counts)):
            return 3
        if need > self.refs.count(0):
            return 2
        for s, x in zip(seqs, counts):
            for i in range(-(-self.length[s] // self.P), -(-(self.length[s] + x) // self.P)):
                self.table[s][i] = self.take()
            self.length[s] += x
        return 0

    def fork(self, parents, children):
        if len(set(children)) != len(children) or any(not 0 <= s < len(self.length) for s in parents + children):
            return 1, []
        if any(self.length[s] for s in children):
            return 4, []
        if sum(1 for s in parents if self.length[s] % self.P) > self.refs.count(0):
            return 2, []
        copies, lens = [], [self.length[a] for a in parents]
        for a, b, n in zip(parents, children, lens):
            for i in range(n // self.P):
                self.table[b][i] = self.table[a][i]
                self.refs[self.table[a][i]] += 1
            if n % self.P:
                self.table[b][n // self.P] = self.take()
                copies.append((self.table[a][n // self.P], self.table[b][n // self.P], n % self.P))
            self.length[b] = n
        return 0, copies

    def free(self, seqs):
        for s in seqs:
            for i in range(-(-self.length[s] // self.P)):
                self.refs[self.table[s][i]] -= 1
                self.table[s][i] = -1
            self.length[s] = 0

    def compact(self):
        live = sum(1 for x in self.refs if x)
        holes = [p for p in range(live) if not self.refs[p]]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p]]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in r] for r in self.table]
        return to

    def same(self, cache):
        t, n, r = (x.tolist() for x in cache.tables())
        assert n == self.length
        assert r == self.refs
        assert t == self.table


@pytest.mark.parametrize("P,n_page,n_seq,width,layers,HK,D,seed", [
    (8, 40, 6, 12, 1, 1, 64, 1), (16, 300, 20, 40, 2, 2, 128, 2), (64, 5000, 100, 200, 1, 1, 64, 3),
    (8, 9001, 1500, 30, 1, 1, 64, 4), (128, 33, 5, 9, 3, 3, 192, 5)])
def test_books_follow_the_model(P, n_page, n_seq, width, layers, HK, D, seed):
    """Random calls, refused ones among them: the books, and the pages' contents, after each."""
    from aero_b200.pages import PagedCache
    r = random.Random(seed)
    c = PagedCache(layers, n_page, P, HK, D, n_seq, width, dtype=BF16)
    b = Books(n_seq, width, n_page, P)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c.k().normal_(generator=g)
    c.v().normal_(generator=g)
    k, v = c.k().clone(), c.v().clone()
    codes = set()
    for step in range(60):
        op = r.choice(["extend", "extend", "fork", "free", "compact", "copy"])
        if op == "extend":
            seqs = [r.randrange(n_seq) for _ in range(r.randint(1, min(8, n_seq)))] if r.random() < 0.2 else \
                r.sample(range(n_seq), r.randint(1, n_seq if n_seq < 50 else 40))
            counts = [r.choice([0, 1, P - 1, P, P + 1, r.randint(0, 3 * P)]) for _ in seqs]
            if r.random() < 0.1:
                counts[-1] = r.choice([-1, width * P + 1])
            want = b.extend(seqs, counts)
            c.extend(i32(seqs), i32(counts))
        elif op == "fork":
            full, empty = [s for s in range(n_seq) if b.length[s]], [s for s in range(n_seq) if not b.length[s]]
            if not full or not empty:
                continue
            children = r.sample(empty, r.randint(1, min(len(empty), 5)))
            if r.random() < 0.2:
                children[0] = r.choice([full[0], children[-1], n_seq])
            parents = [r.choice(full) for _ in children]
            want, copies = b.fork(parents, children)
            c.fork(i32(parents), i32(children))
            for x, y, n in copies:
                k[:, y, :, :n], v[:, y, :, :n] = k[:, x, :, :n], v[:, x, :, :n]
        elif op == "free":
            seqs, want = r.sample(range(n_seq), r.randint(1, max(1, n_seq // 3))), 0
            b.free(seqs)
            c.free(i32(seqs))
        elif op == "compact":
            want = 0
            for x, y in b.compact().items():
                k[:, y], v[:, y] = k[:, x], v[:, x]
            c.compact()
        else:
            some = r.sample(range(n_page), 2 * r.randint(1, min(5, n_page // 2)))
            src, dst, want = some[::2], some[1::2], 0
            c.copy(i32(src), i32(dst))
            k[:, dst], v[:, dst] = k[:, src], v[:, src]
        assert c.status() == want, (step, op)
        codes.add(want)
        b.same(c)
        assert torch.equal(c.k(), k) and torch.equal(c.v(), v), (step, op)
    assert 0 in codes and len(codes) > 1


def test_append_rows_and_strides():
    from aero_b200.pages import PagedCache
    c = PagedCache(2, 20, 8, 3, 64, 3, 6, dtype=F16)
    c.extend(i32([0, 2]), i32([20, 9]))
    seqs, pos = [0, 2, 0, 2, 0], [0, 8, 19, 0, 7]
    table = c.tables()[0].tolist()
    for layer, shift in ((0, 0), (1, 1)):  # 16-byte rows, and rows on odd addresses
        wide = torch.randn((5, 4, 70), device="cuda").to(F16)
        k = wide[:, :3, shift:64 + shift] if shift else wide[:, :3, :64].contiguous()
        v = torch.randn((3, 5, 64), device="cuda").to(F16).transpose(0, 1)
        c.append(layer, k, v, i32(seqs), i32(pos))
        for t in range(5):
            page = table[seqs[t]][pos[t] // 8]
            assert torch.equal(c.k(layer)[page, :, pos[t] % 8], k[t])
            assert torch.equal(c.v(layer)[page, :, pos[t] % 8], v[t])
    c.check()
    k = torch.ones((3, 3, 64), device="cuda", dtype=F16)
    before = c.k().clone()
    for seqs, pos, code in (([0, 9, -1], [0, 0, 0], 1), ([0, 0, 1], [20, -1, 0], 5)):
        c.append(0, before[0, table[0][0], :, 0].expand(3, 3, 64).contiguous(), k, i32(seqs), i32(pos))
        assert c.status() == code  # rows at fault are skipped
        assert torch.equal(c.k(), before)


def test_copy_skips_bad_pages():
    from aero_b200.pages import PagedCache
    c = PagedCache(1, 6, 8, 1, 64, 1, 2, dtype=F16)
    c.k().normal_()
    before = c.k().clone()
    c.copy(i32([0, 1, -1]), i32([6, 2, 3]))
    assert c.status() == 5
    before[:, 2] = before[:, 1]
    assert torch.equal(c.k(), before)


def test_streams_and_graph():
    """Work follows torch's current stream; a captured step replays on new data."""
    c, K, V = open_cache([100, 40], 16, 2, 64, F16)
    q = torch.randn((2, 4, 64), device="cuda").to(F16)
    seqs = i32([0, 1])
    want = c.attend(0, q, seqs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.attend(0, q, seqs)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    out = torch.empty_like(q)
    new_k, new_v = torch.randn((2, 2, 64), device="cuda").to(F16), torch.randn((2, 2, 64), device="cuda").to(F16)
    ones, pos = i32([1, 1]), i32([100, 40])
    g = torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.attend(0, q, seqs, out=out)  # on this stream before the capture
        with torch.cuda.graph(g, stream=s):
            c.extend(seqs, ones)
            c.append(0, new_k, new_v, seqs, pos)
            c.attend(0, q, seqs, out=out)
            pos.add_(1)
    torch.cuda.synchronize()
    rows = [[k] for k in K], [[v] for v in V]
    for _ in range(3):
        new_k.normal_()
        new_v.normal_()
        q.normal_()
        for i in (0, 1):
            rows[0][i].append(new_k[i:i + 1].clone())
            rows[1][i].append(new_v[i:i + 1].clone())
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        ks, vs = [torch.cat(x) for x in rows[0]], [torch.cat(x) for x in rows[1]]
        close(out, join([reference(q[i:i + 1], ks[i], vs[i], [ks[i].shape[0] - 1], 0, 0, 0.125) for i in (0, 1)]), F16)
    c.check()


def test_capture_on_a_stream_of_its_own():
    """A capture whose stream the cache has not run on before, then calls on the old stream again."""
    c, K, V = open_cache([100, 40], 16, 2, 64, F16)
    q, seqs = torch.randn((2, 4, 64), device="cuda").to(F16), i32([0, 1])
    want = c.attend(0, q, seqs)
    out = torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.attend(0, q, seqs, out=out)
    g.replay()
    assert torch.equal(out, want) and torch.equal(c.attend(0, q, seqs), want)
    q.mul_(0.5)
    g.replay()
    assert torch.equal(out, c.attend(0, q, seqs))
    c.check()


def test_refusals():
    from aero_b200.pages import PagedCache, plan_bytes
    for bad in (dict(page_size=12), dict(page_size=4), dict(page_size=512), dict(head_dim=96), dict(n_page=0),
                dict(n_page=2**22, page_size=256, n_head_kv=8), dict(max_pages=0), dict(device=99)):
        a = dict(n_layer=1, n_page=4, page_size=16, n_head_kv=2, head_dim=64, n_seq=2, max_pages=2, device=0)
        a.update(bad)
        with pytest.raises(RuntimeError):
            PagedCache(**a)
    with pytest.raises(ValueError):
        PagedCache(1, 4, 16, 2, 64, 2, 2, dtype=torch.float32)
    g = nc.MemoryGuard()
    committed = g.committed()
    c = PagedCache(1, 4, 16, 2, 64, 2, 2, dtype=F16)
    assert g.committed() - committed == plan_bytes(1, 4, 16, 2, 64, 2, 2)["total"]
    q = torch.zeros((1, 4, 64), device="cuda", dtype=F16)
    one = i32([0])
    for call in (lambda: c.attend(1, q, one), lambda: c.attend(-1, q, one), lambda: c.attend(0, q.to(BF16), one),
                 lambda: c.attend(0, q[:, :3], one), lambda: c.attend(0, q.repeat(1, 9, 1), one),
                 lambda: c.attend(0, q, i32([0, 1])), lambda: c.attend(0, q, one.long()),
                 lambda: c.attend(0, q, one.cpu()), lambda: c.attend(0, q[..., :32], one),
                 lambda: c.attend(0, q, one, window=-1), lambda: c.attend(0, q, one, sinks=-1),
                 lambda: c.attend(0, q, one, scale=math.nan), lambda: c.attend(0, q, one, out=q[:, :2]),
                 lambda: c.attend(0, q.transpose(1, 2).contiguous().transpose(1, 2), one),
                 lambda: c.attend(0, q, one, i32([0])),
                 lambda: c.extend(i32([0, 1, 0]), i32([1, 1, 1])), lambda: c.extend(one, i32([1, 1])),
                 lambda: c.copy(i32([0] * 5), i32([1] * 5)), lambda: c.append(0, q, q, one, one),
                 lambda: c.set_tables(one, one, one)):
        with pytest.raises(ValueError):
            call()
    assert c.status() == 0
    lib, L = nc.lib(), c.handle
    host = np.zeros(4, np.int32)
    assert lib.aero_cuda_pages_free(L, host.ctypes.data, 1) == -1 and "device memory" in c.last_error()
    c.attend(0, q, i32([7]))  # a sequence that is none: an empty one, and a code
    assert c.attend(0, q, i32([7])).abs().max() == 0
    c.close()
    with pytest.raises(RuntimeError):
        c.attend(0, q, one)
    assert g.committed() == committed
