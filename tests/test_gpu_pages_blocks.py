"""Attention over selected blocks of the paged cache: the bounds of pages, the choice of blocks and the
attention over a list, each against a plain form in 64 bits, and what the calls refuse.

Bounds and block numbers are exact: minima and maxima of the cache's own values; scores in 64 bits, whose
order two sums of at most 512 products with errors of 2^-53 each can change only where they
agree to 2^-44 (values of a few bits make equal scores equal in both).

Tolerance of an attention output: u|o| for its own rounding (u = 2^-11 in f16, 2^-8 in bf16); (2^-14 +
2^-16) sum w|v| for scores, exponentials and sums in f32 (|score| up to about 30 with an error of some 2^-21
of it) and for probabilities that meet V as two values of the type; 2^-24 where it underflows.
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


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def open_cache(lens, P, HK, D, dtype, *, layers=1, spare=3, seed=0, extra_rows=0, values=None, width=None):
    """A cache with bounds whose pool is NaN but for the sequences' rows, pages scattered, filled by append into
    layer `layers - 1`. Returns (cache, [K of a sequence (n, HK, D)], [V])."""
    from aero_b200.pages import PagedCache
    r = random.Random(seed)
    n, used = len(lens), [-(-x // P) for x in lens]
    n_page, width = sum(used) + spare, width or max([1, *used]) + 1
    c = PagedCache(layers, n_page, P, HK, D, n + extra_rows, width, dtype=dtype, bounds=True)
    c.k().fill_(math.nan)
    c.v().fill_(math.nan)
    order = list(range(n_page))
    r.shuffle(order)
    table, refs = np.full((n + extra_rows, width), -1, np.int32), np.zeros(n_page, np.int32)
    for s, u in enumerate(used):
        for i in range(u):
            table[s, i] = order.pop()
            refs[table[s, i]] = 1
    c.set_tables(torch.from_numpy(table).cuda(), i32(list(lens) + [0] * extra_rows), i32(refs))
    T = sum(lens)
    k = torch.randn((T, HK, D), device="cuda", generator=gen(seed + 1)) if values is None else values
    k, v = k.to(dtype), torch.randn((T, HK, D), device="cuda", generator=gen(seed + 2)).to(dtype)
    c.append(layers - 1, k, v, i32([s for s, x in enumerate(lens) for _ in range(x)]), i32([i for x in lens for i in range(x)]))
    c.check()
    return c, list(k.split(lens)), list(v.split(lens))


def plain_bounds(K, P):
    """(blocks, HK, 2, D) of one sequence's keys (n, HK, D), as values."""
    big = torch.finfo(K.dtype).max
    x = K.double()
    lo = torch.where(x.isnan(), math.inf, x.clamp(-big, big))
    hi = torch.where(x.isnan(), -math.inf, x.clamp(-big, big))
    out = []
    for b in range(0, K.shape[0], P):
        pair = torch.stack([lo[b:b + P].amin(0), hi[b:b + P].amax(0)], 1)
        out.append(torch.where(pair.isinf(), 0.0, pair))
    return torch.stack(out) if out else torch.zeros((0, K.shape[1], 2, K.shape[2]), dtype=torch.float64, device="cuda")


def held_bounds(c, s, n, layer=0):
    table = c.tables()[0]
    return c.bounds(layer)[table[s, :-(-n // c.page_size)].long()].double()


# ------------------------------------------------------------------ bounds
@pytest.mark.parametrize("lens,P,HK,D,dtype", [
    ([1], 8, 1, 64, F16), ([0, 7, 8, 9, 0, 100], 8, 3, 128, BF16), ([64, 65, 300], 64, 2, 192, F16),
    ([255, 256, 257, 1], 256, 2, 256, BF16), ([33] * 40, 16, 1, 128, F16)])
def test_bounds_of_appended_pages(lens, P, HK, D, dtype):
    values = torch.randn((sum(lens), HK, D), device="cuda", generator=gen(5))
    odd = torch.rand(values.shape, device="cuda", generator=gen(6))
    values[odd < 0.02] = math.nan
    values[(odd > 0.02) & (odd < 0.03)] = math.inf
    values[(odd > 0.03) & (odd < 0.04)] = -math.inf
    values[:, :, 0] = math.nan
    values[:, :, 1] = math.inf
    c, K, _ = open_cache(lens, P, HK, D, dtype, layers=2, values=values)
    made = c.bounds().clone()
    for s, n in enumerate(lens):
        assert torch.equal(held_bounds(c, s, n, 1), plain_bounds(K[s], P))
    used = c.tables()[0][c.tables()[0] >= 0].long()
    rest = torch.ones(c.n_page, dtype=torch.bool, device="cuda")
    rest[used] = False
    assert (made[1][rest] == 0).all() and (made[0] == 0).all()
    # the same from the pool, and for listed sequences only
    c.bounds().fill_(7)
    some = [s for s in range(len(lens)) if s % 2 == 0]
    c.set_bounds(1, i32(some))
    c.check()
    assert (c.bounds(0) == 7).all()
    for s, n in enumerate(lens):
        want = plain_bounds(K[s], P)
        assert torch.equal(held_bounds(c, s, n, 1), want if s in some else torch.full_like(want, 7))
    assert (c.bounds(1)[rest] == 7).all()


def test_bounds_move_with_their_pages():
    c, K, _ = open_cache([100, 40, 64], 16, 2, 64, F16, layers=2, extra_rows=2, spare=12)
    c.bounds(0).copy_(torch.randn(c.bounds(0).shape, device="cuda"))
    before = [[held_bounds(c, s, n, layer) for layer in (0, 1)] for s, n in enumerate((100, 40, 64))]
    c.fork(i32([0, 2]), i32([3, 4]))
    for s, n, parent in ((3, 100, 0), (4, 64, 2)):
        for layer in (0, 1):
            assert torch.equal(held_bounds(c, s, n, layer), before[parent][layer])
    # a step of the copies: their last pages are their own
    c.extend(i32([3, 4]), i32([1, 1]))
    k = 9 * torch.ones((2, 2, 64), dtype=F16, device="cuda")
    c.append(1, k, k, i32([3, 4]), i32([100, 64]))
    assert torch.equal(held_bounds(c, 0, 100, 1), before[0][1])
    assert torch.equal(held_bounds(c, 3, 101, 1), plain_bounds(torch.cat([K[0], k[:1]]), 16))
    assert torch.equal(held_bounds(c, 4, 65, 1), plain_bounds(torch.cat([K[2], k[:1]]), 16))
    c.free(i32([1, 0]))
    c.compact()
    c.check()
    assert torch.equal(held_bounds(c, 3, 101, 1), plain_bounds(torch.cat([K[0], k[:1]]), 16))
    assert torch.equal(held_bounds(c, 3, 100, 0), before[0][0])
    assert torch.equal(held_bounds(c, 2, 64, 0), before[2][0])
    a, b = int(c.tables()[0][2, 0]), int((c.tables()[2] == 0).nonzero()[-1])
    c.copy(i32([a]), i32([b]))
    assert torch.equal(c.bounds()[:, a], c.bounds()[:, b])


def test_bounds_step_by_step_and_refused_appends():
    """Single tokens; a later write of an earlier position; rows that an append refuses leave the bounds."""
    from aero_b200.pages import PagedCache
    c = PagedCache(1, 8, 8, 1, 64, 3, 4, bounds=True)
    rows = torch.randn((20, 1, 64), device="cuda", generator=gen(1)).half()
    for i in range(20):
        c.extend(i32([1]), i32([1]))
        c.append(0, rows[i:i + 1], rows[i:i + 1], i32([1]), i32([i]))
        assert torch.equal(held_bounds(c, 1, i + 1), plain_bounds(rows[:i + 1], 8))
    rows[3] = 0
    c.append(0, rows[3:4], rows[3:4], i32([1]), i32([3]))
    assert torch.equal(held_bounds(c, 1, 20), plain_bounds(rows, 8))
    c.check()
    c.fork(i32([1]), i32([0]))
    was = c.bounds().clone()
    c.append(0, rows[:3], rows[:3], i32([1, 5, 1]), i32([0, 0, 20]))  # a shared page, no sequence, past the end
    assert c.status() != 0 and torch.equal(was, c.bounds())


def test_bounds_of_a_page_that_sequences_of_several_lengths_hold():
    """Adopted books may share a page that not all of its sequences fill: its bounds cover it whole, in any order."""
    from aero_b200.pages import PagedCache
    c = PagedCache(1, 9, 64, 2, 64, 3, 2, dtype=BF16, bounds=True)
    rows = torch.randn((9, 2, 64, 64), device="cuda", generator=gen(2)).to(BF16)
    c.k(0).copy_(rows.reshape(c.k(0).shape))
    c.set_tables(i32([4, 7, 4, -1, 4, 2]), i32([70, 9, 128]), i32([0, 0, 1, 0, 3, 0, 0, 1, 0]))

    def whole(page, n=64):
        return plain_bounds(rows[page, :, :n].transpose(0, 1), 64)[0]

    for order in ([0, 1, 2], [2, 1, 0], [1], [0, 2, 1]):
        c.bounds().fill_(7)
        c.set_bounds(0, i32(order))
        c.check()
        assert torch.equal(c.bounds(0)[4].double(), whole(4))
        if 0 in order:
            assert torch.equal(c.bounds(0)[7].double(), whole(7, 6)) and torch.equal(c.bounds(0)[2].double(), whole(2))


# ------------------------------------------------------------------ the choice
def plain_select(q, bounds, n, P, W, first, recent):
    """Block numbers (HK, W) of one token that sees n positions; bounds (blocks, HK, 2, D)."""
    HK = bounds.shape[1]
    nb = -(-n // P)
    b, x = bounds[:nb].cpu().numpy(), q.double().reshape(HK, -1, q.shape[-1]).cpu().numpy()
    out = np.full((HK, W), -1, np.int64)
    number = np.arange(nb)
    always = (number < first) | (number >= nb - recent)
    for h in range(HK):
        with np.errstate(invalid="ignore"):
            s = np.maximum(x[h][None] * b[:, None, h, 0], x[h][None] * b[:, None, h, 1]).sum(-1)
        s = np.where(np.isnan(s), np.inf, s).max(1)
        order = np.argsort(-s, kind="stable")
        got = np.sort(np.concatenate([number[always], order[~always[order]]])[:W])
        out[h, :len(got)] = got
    return out


def few_bits(shape, seed):
    """Values whose products and sums are exact in 64 bits, so that equal scores are equal."""
    return torch.randint(-8, 9, shape, device="cuda", generator=gen(seed)).float() / 4


SELECT = [
    # lens, page, HK, G, D, dtype, n_blocks, first, recent
    ([1], 8, 1, 1, 64, F16, 4, 1, 1),
    ([0, 1, 8, 9, 200, 33], 8, 2, 3, 64, BF16, 4, 0, 1),
    ([300, 777, 40], 16, 4, 8, 128, F16, 8, 1, 2),
    ([700, 64], 8, 1, 16, 128, BF16, 3, 1, 2),     # no room but for those chosen always
    ([700, 641], 16, 2, 5, 192, F16, 40, 2, 1),    # one sequence shorter than the list, one just longer
    ([2000, 100], 8, 2, 12, 256, BF16, 17, 0, 3),
    ([9000], 8, 2, 4, 64, F16, 100, 1, 1),
    ([4000] * 5, 16, 3, 2, 128, BF16, 1, 0, 1),
]


@pytest.mark.parametrize("lens,P,HK,G,D,dtype,W,first,recent", SELECT)
@pytest.mark.parametrize("exact", [True, False])
def test_select_matches_plain(lens, P, HK, G, D, dtype, W, first, recent, exact):
    values = few_bits((sum(lens), HK, D), 3) if exact else None
    c, K, _ = open_cache(lens, P, HK, D, dtype, values=values)
    q = few_bits((len(lens), HK * G, D), 4) if exact else torch.randn((len(lens), HK * G, D), device="cuda", generator=gen(4))
    q = q.to(dtype)
    seqs = list(range(len(lens)))[::-1]
    got = c.select(0, q, i32(seqs), n_blocks=W, first=first, recent=recent).cpu().numpy()
    c.check()
    for i, s in enumerate(seqs):
        want = plain_select(q[i], plain_bounds(K[s], P), lens[s], P, W, first, recent)
        assert (got[i] == want).all(), (s, got[i], want)


def test_select_ties_and_values_that_are_no_numbers():
    """Equal scores go to the lowest blocks; a score that is no number counts as +infinity."""
    P, HK, D, n = 8, 2, 64, 8 * 300
    values = few_bits((8, HK, D), 1).repeat(300, 1, 1)  # every block alike
    values[8 * 41:8 * 42] += 1
    c, K, _ = open_cache([n], P, HK, D, F16, values=values)
    for fill in (0.0, 1.0, math.nan, math.inf):
        q = torch.full((1, 2 * HK, D), fill, dtype=F16, device="cuda")
        got = c.select(0, q, i32([0]), n_blocks=9, first=1, recent=2)[0].cpu().numpy()
        c.check()
        assert (got == plain_select(q[0], plain_bounds(K[0], P), n, P, 9, 1, 2)).all()
        others = [41, 1, 2, 3, 4, 5] if fill == 1.0 else [1, 2, 3, 4, 5, 6]
        assert got[0].tolist() == sorted([0, *others, 298, 299])


@pytest.mark.parametrize("width,G,D", [(700, 4, 64), (7000, 4, 64), (50000, 4, 64), (131072, 4, 64), (131072, 16, 256)])
def test_select_in_caches_of_long_rows(width, G, D):
    """The cluster's size and the keys' place follow from max_pages."""
    lens, P, HK = [8 * 600 + 3, 20], 8, 1
    c, K, _ = open_cache(lens, P, HK, D, BF16, width=width)
    q = torch.randn((2, G, D), device="cuda", generator=gen(7)).to(BF16)
    got = c.select(0, q, i32([0, 1]), n_blocks=31).cpu().numpy()
    for s in (0, 1):
        assert (got[s] == plain_select(q[s], plain_bounds(K[s], P), lens[s], P, 31, 1, 1)).all()


def test_select_several_tokens_a_sequence():
    lens, new, P, HK, G, D = [500, 9, 1200], [5, 9, 3], 16, 2, 4, 128
    c, K, _ = open_cache(lens, P, HK, D, F16)
    q = torch.randn((sum(new) + 4, HK, 2 * G, D), device="cuda", generator=gen(8)).half()
    q = q[4:, :, :G].transpose(1, 2).reshape(sum(new), G * HK, D)  # a copy; then a view with other strides
    wide = torch.empty((sum(new), G * HK, 2 * D), dtype=F16, device="cuda")
    wide[..., 1:1 + D] = q
    view = wide[..., 1:1 + D]
    got = c.select(0, view, i32([0, 1, 2]), i32([0, 5, 14, 17]), n_blocks=8, first=1, recent=2).cpu().numpy()
    c.check()
    t = 0
    for s, x in enumerate(new):
        for i in range(x):
            assert (got[t] == plain_select(q[t], plain_bounds(K[s], P), lens[s] - x + i + 1, P, 8, 1, 2)).all()
            t += 1


# ------------------------------------------------------------------ attention over a list
def reference(q, K, V, n, P, lists, scale):
    """One token q (H, D) that sees n positions; lists: per kv head its blocks, each as often as it is listed."""
    H, D = q.shape
    HK = len(lists)
    out, mag = (torch.zeros((H, D), dtype=torch.float64, device="cuda") for _ in range(2))
    for h in range(HK):
        at = [j for b in lists[h] if b >= 0 for j in range(b * P, min(n, (b + 1) * P))]
        if not at:
            continue
        at = torch.tensor(at, device="cuda")
        s = (q[h * (H // HK):(h + 1) * (H // HK)].double() @ K[at, h].double().T) * scale
        w = torch.softmax(s, 1)
        out[h * (H // HK):(h + 1) * (H // HK)] = w @ V[at, h].double()
        mag[h * (H // HK):(h + 1) * (H // HK)] = w @ V[at, h].double().abs()
    return out, mag


def close(got, refs, dtype):
    out, mag = (torch.stack([r[i] for r in refs]) for i in (0, 1))
    u = 2.0**-11 if dtype == F16 else 2.0**-8
    tol = u * out.abs() + (2.0**-14 + 2.0**-16) * mag + 2.0**-24
    err = (got.double() - out).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.3f} of the tolerance"


BLOCKS = [
    # lens, page, HK, G, D, dtype, width of the lists
    ([1], 8, 1, 1, 64, F16, 1),
    ([0, 1, 7, 8, 9, 200], 8, 2, 3, 64, BF16, 5),
    ([700, 5, 129], 16, 4, 8, 128, F16, 13),
    ([1000, 999, 128], 64, 1, 16, 128, BF16, 3),
    ([3000, 40], 32, 2, 4, 128, F16, 70),
    ([513, 77, 300], 128, 2, 5, 192, F16, 2),
    ([1260, 1, 257, 512], 256, 2, 7, 256, BF16, 3),
    ([1500, 20], 16, 2, 16, 256, F16, 40),
    ([2100], 8, 1, 2, 192, BF16, 262),
]


@pytest.mark.parametrize("lens,P,HK,G,D,dtype,W", BLOCKS)
def test_attend_blocks_matches_plain(lens, P, HK, G, D, dtype, W):
    c, K, V = open_cache(lens, P, HK, D, dtype)
    r = random.Random(W)
    lists, pages = [], c.tables()[0].cpu().numpy()
    for s, n in enumerate(lens):
        nb = -(-n // P)
        rows = []
        for h in range(HK):
            row = r.sample(range(nb), min(nb, r.randint(0, W)))  # any order
            if row and r.random() < 0.3:
                row[-1] = row[0]  # twice
            if r.random() < 0.5:
                row += [nb + r.randint(0, 3)] if len(row) < min(W, nb) else []  # a block that the token does not have
                row.sort(reverse=True)
            row = (row + [r.choice([-1, -7]) for _ in range(W)])[:W]
            rows.append(row)
        lists.append(rows)
        # blocks of this sequence that nobody lists may hold anything
        for b in set(range(nb)) - {x for row in rows for x in row}:
            c.k(0)[int(pages[s, b])] = math.inf
            c.v(0)[int(pages[s, b])] = math.nan
    q = (2 * torch.randn((len(lens), HK * G, D), device="cuda", generator=gen(9))).to(dtype)
    got = c.attend_blocks(0, q, i32(list(range(len(lens)))), i32(lists).reshape(len(lens), HK, W))
    c.check()
    refs = []
    for s, n in enumerate(lens):
        nb = -(-n // P)
        seen = [[b for b in row[:nb] if 0 <= b < nb] for row in lists[s]]
        refs.append(reference(q[s], K[s], V[s], n, P, seen, 1 / math.sqrt(D)))
    close(got, refs, dtype)


def test_attend_blocks_of_every_block_is_attend():
    lens, P, HK, G, D = [300, 17, 64], 16, 2, 4, 128
    c, _, _ = open_cache(lens, P, HK, D, F16)
    q = torch.randn((3, HK * G, D), device="cuda", generator=gen(2)).half()
    lists = torch.arange(19, dtype=torch.int32, device="cuda").expand(3, HK, 19).contiguous()
    assert torch.equal(c.attend_blocks(0, q, i32([0, 1, 2]), lists), c.attend(0, q, i32([0, 1, 2])))


def test_attend_blocks_several_tokens_views_and_scale():
    lens, new, P, HK, G, D = [500, 9, 120], [5, 9, 3], 16, 2, 3, 64
    T, W = sum(new), 6
    c, K, V = open_cache(lens, P, HK, D, BF16, layers=3)
    q = torch.randn((T, HK * G, D), device="cuda", generator=gen(3)).to(BF16)
    wide, out = (torch.zeros((T, HK * G + 1, D + 3), dtype=BF16, device="cuda") for _ in range(2))
    wide[:, 1:, 1:1 + D] = q
    r = random.Random(0)
    lists = [[[r.randrange(40) for _ in range(W)] for _ in range(HK)] for _ in range(T)]
    ret = c.attend_blocks(2, wide[:, 1:, 1:1 + D], i32([0, 1, 2]), i32(lists).reshape(T, HK, W), i32([0, 5, 14, 17]), scale=0.2,
                          out=out[:, 1:, 3:])
    c.check()
    assert ret.data_ptr() == out[:, 1:, 3:].data_ptr() and (out[:, 0] == 0).all() and (out[:, :, :3] == 0).all()
    refs, t = [], 0
    for s, x in enumerate(new):
        for i in range(x):
            n = lens[s] - x + i + 1
            nb = -(-n // P)
            refs.append(reference(q[t], K[s], V[s], n, P, [[b for b in row[:nb] if b < nb] for row in lists[t]], 0.2))
            t += 1
    close(out[:, 1:, 3:], refs, BF16)


def test_many_tokens_of_one_list_and_long_lists():
    """More parts than CTAs, segments that several CTAs share, lists wider than a sequence."""
    lens, P, HK, G, D = [5000] + [3] * 90, 8, 2, 8, 128
    c, K, V = open_cache(lens, P, HK, D, F16)
    q = torch.randn((91, HK * G, D), device="cuda", generator=gen(5)).half()
    lists = torch.arange(1000, dtype=torch.int32, device="cuda").flip(0).expand(91, HK, 1000).contiguous()
    got = c.attend_blocks(0, q, i32(list(range(91))), lists)
    c.check()
    # of the long one's 625 blocks the first 625 entries are looked at: blocks 999 to 375, of which it has those below 625
    refs = [reference(q[0], K[0], V[0], 5000, P, [list(range(375, 625))] * HK, 1 / math.sqrt(D))]
    # a short one has one block, and its list's first entry is not it
    refs += [reference(q[s], K[s], V[s], 3, P, [[]] * HK, 1 / math.sqrt(D)) for s in range(1, 91)]
    close(got, refs, F16)


# ------------------------------------------------------------------ together, captured, refused
def test_a_step_captured_and_replayed():
    """append, select and attend_blocks of a decode step as a graph, replayed with other inputs."""
    lens, P, HK, G, D, W = [130, 64, 15], 16, 2, 4, 64, 4
    c, K, V = open_cache(lens, P, HK, D, F16, spare=6)
    seqs, pos = i32([0, 1, 2]), i32(lens)
    k, v = (torch.zeros((3, HK, D), dtype=F16, device="cuda") for _ in range(2))
    q, out = (torch.zeros((3, HK * G, D), dtype=F16, device="cuda") for _ in range(2))
    lists = torch.zeros((3, HK, W), dtype=torch.int32, device="cuda")
    ones = i32([1, 1, 1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        c.extend(seqs, ones)
        c.append(0, k, v, seqs, pos)
        c.select(0, q, seqs, n_blocks=W, out=lists)
        c.attend_blocks(0, q, seqs, lists, out=out)
        pos.add_(1)
    for step in range(3):
        nk, nv = (torch.randn((3, HK, D), device="cuda", generator=gen(10 + 2 * step + i)).half() for i in (0, 1))
        nq = torch.randn((3, HK * G, D), device="cuda", generator=gen(20 + step)).half()
        k.copy_(nk), v.copy_(nv), q.copy_(nq)
        graph.replay()
        torch.cuda.synchronize()
        refs = []
        for s in range(3):
            K[s], V[s] = torch.cat([K[s], nk[s:s + 1]]), torch.cat([V[s], nv[s:s + 1]])
            n = lens[s] + step + 1
            want = plain_select(nq[s], plain_bounds(K[s], P), n, P, W, 1, 1)
            assert (lists[s].cpu().numpy() == want).all()
            refs.append(reference(nq[s], K[s], V[s], n, P, want.tolist(), 1 / math.sqrt(D)))
        close(out, refs, F16)
    del graph
    c.check()


def test_what_only_the_device_sees():
    c, K, V = open_cache([50, 100], 16, 1, 64, F16)
    q = torch.randn((2, 2, 64), device="cuda", generator=gen(1)).half()
    lists = i32([[0, 1, 2], [1, 3, -1]]).reshape(2, 1, 3)
    good = c.attend_blocks(0, q, i32([0, 1]), lists)
    # sequence numbers outside the cache: no blocks, zeros
    assert (c.select(0, q, i32([0, 9]), n_blocks=3)[1] == -1).all() and c.status() == 1
    got = c.attend_blocks(0, q, i32([-1, 1]), lists)
    assert (got[0] == 0).all() and torch.equal(got[1], good[1]) and c.status() == 1
    c.set_bounds(0, i32([1, 9]))
    assert c.status() == 1
    # a listed block without a page counts as keys and values of zeros
    table, length, refs = (x.clone() for x in c.tables())
    page = int(table[1, 3])
    table[1, 3] = -1
    c.set_tables(table, length, refs)
    got = c.attend_blocks(0, q, i32([0, 1]), lists)
    assert torch.equal(got[0], good[0]) and c.status() == 5
    K0, V0 = K[1].clone(), V[1].clone()
    K0[48:64] = 0
    V0[48:64] = 0
    close(got[1:], [reference(q[1], K0, V0, 100, 16, [[1, 3]], 1 / 8)], F16)
    # and has bounds 0 in a choice
    bounds = plain_bounds(K[1], 16)
    bounds[3] = 0
    got = c.select(0, q[1:], i32([1]), n_blocks=4).cpu().numpy()
    assert c.status() == 5 and (got[0] == plain_select(q[1], bounds, 100, 16, 4, 1, 1)).all()
    assert page >= 0
    # q_start that does not ascend to T
    c.select(0, q, i32([0]), i32([0, 1]), n_blocks=3)
    assert c.status() == 6


def test_refusals():
    from aero_b200.pages import PagedCache, plan_bytes
    c, _, _ = open_cache([50], 16, 2, 64, F16)
    q = torch.zeros((1, 4, 64), dtype=F16, device="cuda")
    one = i32([0])
    lists = i32([0, 0]).reshape(1, 2, 1)
    for kw in (dict(n_blocks=0), dict(n_blocks=1), dict(n_blocks=4, first=-1), dict(n_blocks=4, recent=0),
               dict(n_blocks=1 << 28), dict(n_blocks=4, out=torch.zeros((1, 2, 3), dtype=torch.int32, device="cuda")),
               dict(n_blocks=4, out=torch.zeros((1, 2, 4), device="cuda"))):
        if kw["n_blocks"] == 1 << 28:
            kw["out"] = torch.zeros((1, 2, 1), dtype=torch.int32, device="cuda").expand(1, 2, 1 << 28)
        with pytest.raises(ValueError):
            c.select(0, q, one, **kw)
    for bad in (lambda: c.select(1, q, one, n_blocks=4), lambda: c.select(0, q[:, :3], one, n_blocks=4),
                lambda: c.select(0, q.bfloat16(), one, n_blocks=4), lambda: c.select(0, q, i32([0, 0]), n_blocks=4),
                lambda: c.select(0, q.cpu(), one, n_blocks=4), lambda: c.set_bounds(-1, one),
                lambda: c.set_bounds(0, one.long()), lambda: c.set_bounds(0, i32([0, 0])),
                lambda: c.attend_blocks(0, q, one, lists.long()), lambda: c.attend_blocks(0, q, one, lists[:, :1]),
                lambda: c.attend_blocks(0, q, one, lists[..., :0]), lambda: c.attend_blocks(0, q, one, lists, scale=0.0),
                lambda: c.attend_blocks(0, q, one, lists, scale=math.nan), lambda: c.attend_blocks(0, q, one, lists.cpu()),
                lambda: c.attend_blocks(0, q, one, lists, out=q[:, :2]), lambda: c.attend_blocks(2, q, one, lists)):
        with pytest.raises(ValueError):
            bad()
    plain = PagedCache(1, 4, 16, 2, 64, 1, 4)
    for bad in (plain.bounds, lambda: plain.set_bounds(0, one), lambda: plain.select(0, q, one, n_blocks=4)):
        with pytest.raises(ValueError, match="keeps no bounds"):
            bad()
    assert (plain.attend_blocks(0, q, one, lists) == 0).all()  # (a list is served without bounds)
    plain.check()
    with pytest.raises(ValueError, match="131072"):
        PagedCache(1, 4, 16, 2, 64, 1, 131073, bounds=True).select(0, q, one, n_blocks=4)
    p = plan_bytes(2, 10, 16, 4, 128, 3, 5, bounds=True)
    assert p["kv_cache"] == plan_bytes(2, 10, 16, 4, 128, 3, 5)["kv_cache"] + 2 * 10 * 4 * 2 * 128 * 2
    # no tokens, no sequences
    assert c.select(0, q[:0], one[:0], n_blocks=4).shape == (0, 2, 4)
    assert c.attend_blocks(0, q[:0], one[:0], lists[:0]).shape == (0, 4, 64)
    c.set_bounds(0, one[:0])
    c.check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("alike", [5, 40, 400])
def test_select_scores_next_to_one_another(dtype, alike):
    """Blocks whose scores differ by less than sums in f32 resolve, a few of them, more than a CTA's list, all."""
    P, HK, D, blocks = 8, 1, 256, 600
    values = few_bits((blocks, 1, D), 11) * 4
    values[100:100 + alike] = values[100].abs() + 20  # alike, and high
    step = {F16: 2.0**-10, BF16: 2.0**-7}[dtype]
    which = torch.randperm(alike, generator=torch.Generator().manual_seed(1))
    for i in range(alike):  # then each a few of the last bits of its columns more, in no order
        values[100 + i, 0, :min(D, int(which[i]) % 200)] *= 1 + step
    keys = values.repeat_interleave(P, 0).to(dtype)
    c, K, _ = open_cache([P * blocks], P, HK, D, dtype, values=keys)
    q = torch.rand((1, 8, D), device="cuda", generator=gen(12)).mul_(0.001).add_(1).to(dtype)
    for W in (3, 4, 30, 300):
        got = c.select(0, q, i32([0]), n_blocks=W).cpu().numpy()
        c.check()
        assert (got[0] == plain_select(q[0], plain_bounds(K[0], P), P * blocks, P, W, 1, 1)).all()


@pytest.mark.parametrize("power", [-72, -66, -63, -60, -52, 55])
def test_select_of_the_smallest_and_largest_values(power):
    """Products around and below what f32 holds without loss, and sums near its largest."""
    lens, P, HK, G, D = [4000, 640], 8, 2, 4, 128
    values = torch.randn((sum(lens), HK, D), device="cuda", generator=gen(21)) * 2.0**power
    c, K, _ = open_cache(lens, P, HK, D, BF16, values=values)
    q = (torch.randn((2, HK * G, D), device="cuda", generator=gen(22)) * 2.0**power).to(BF16)
    got = c.select(0, q, i32([0, 1]), n_blocks=30).cpu().numpy()
    c.check()
    for s, n in enumerate(lens):
        assert (got[s] == plain_select(q[s], plain_bounds(K[s], P), n, P, 30, 1, 1)).all()


def test_select_of_wide_rows_of_queries():
    """A batch with rows of zeros and of infinities beside ordinary ones, long and short sequences, over 16 query heads."""
    lens, P, HK, G, D = [3000, 5, 1111, 2048, 3000], 8, 2, 16, 192
    c, K, _ = open_cache(lens, P, HK, D, F16)
    q = torch.randn((5, HK * G, D), device="cuda", generator=gen(13)).half()
    q[0] = 0
    q[3, 5] = math.inf
    q[4] *= 1e-4
    got = c.select(0, q, i32([0, 1, 2, 3, 4]), n_blocks=20, first=2, recent=3).cpu().numpy()
    for s, n in enumerate(lens):
        assert (got[s] == plain_select(q[s], plain_bounds(K[s], P), n, P, 20, 2, 3)).all()


def test_memory_is_charged_and_given_back():
    import gc
    from aero_b200.pages import PagedCache, plan_bytes
    gc.collect()
    lib = nc.lib()
    before = [lib.aero_cuda_guard_committed(i) for i in range(5)]
    c = PagedCache(2, 40, 16, 2, 128, 3, 9, bounds=True)
    held = sum(lib.aero_cuda_guard_committed(i) for i in range(5)) - sum(before)
    assert held == plan_bytes(2, 40, 16, 2, 128, 3, 9, bounds=True)["total"]
    assert lib.aero_cuda_pages_keep_bounds(c.handle) == 0  # again: nothing more
    assert sum(lib.aero_cuda_guard_committed(i) for i in range(5)) - sum(before) == held
    c.close()
    assert [lib.aero_cuda_guard_committed(i) for i in range(5)] == before


def test_calls_on_other_streams_and_a_set_stream():
    """The cache follows torch's current stream; what one stream wrote the next call on another waits for."""
    c, K, V = open_cache([300, 90], 16, 2, 64, F16)
    q = torch.randn((2, 8, 64), device="cuda", generator=gen(3)).half()
    lists = c.select(0, q, i32([0, 1]), n_blocks=3)
    want = c.attend_blocks(0, q, i32([0, 1]), lists)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    seqs, out = i32([0, 1]), torch.empty_like(lists)
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(20000000)
        c.select(0, q, seqs, n_blocks=3, out=out)
    with torch.cuda.stream(b):  # the cache's calls run one after another
        got = c.attend_blocks(0, q, seqs, out)
    torch.cuda.synchronize()
    assert torch.equal(out, lists) and torch.equal(got, want)
    c.set_stream(a)
    got = c.attend_blocks(0, q, seqs, out)
    a.synchronize()
    assert torch.equal(got, want)
    c.check()
