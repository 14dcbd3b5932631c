"""Attention over listed blocks: every entry of a list counts, wherever it stands and however long the list is.

Lists with -1 in front and between, with blocks that the token does not see in front of others, with blocks listed again,
longer than the sequence has blocks. Against the plain form and with the tolerance of test_gpu_pages_blocks.py (an output's
own rounding, f32 scores and sums, two values of the type for a probability; a block listed twice weighs twice in both).
"""

import math
import random

import pytest

from aero_b200 import native_cuda as nc
from test_gpu_pages_blocks import close, gen, i32, open_cache, reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _gpu(cuda_lib):
    nc.require_gpu()


def seen(row, nb):
    return [b for b in row if 0 <= b < nb]


def check(c, K, V, lens, lists, q, P, dtype, q_start=None, row_seq=None, row_len=None):
    """lists[t][h]: token t's entries for kv head h."""
    T, HK, W = len(lists), len(lists[0]), len(lists[0][0])
    row_seq, row_len = row_seq or list(range(T)), row_len or list(lens)
    got = c.attend_blocks(0, q, i32(sorted(set(row_seq))), i32(lists).reshape(T, HK, W), None if q_start is None else i32(q_start))
    c.check()
    close(got, [reference(q[t], K[s], V[s], n, P, [seen(row, -(-n // P)) for row in lists[t]], 1 / math.sqrt(q.shape[-1]))
                for t, (s, n) in enumerate(zip(row_seq, row_len))], dtype)
    return got


CASES = [
    # lens, page, HK, G, D, dtype, width of the lists
    ([1], 8, 1, 1, 64, F16, 2),
    ([1, 8, 9, 40, 0], 8, 2, 3, 64, BF16, 19),
    ([6 * 16], 16, 1, 8, 128, F16, 8),
    ([700, 5, 129], 16, 4, 8, 128, BF16, 71),
    ([3000, 40, 33, 1], 32, 2, 4, 128, F16, 300),
    ([1000, 64, 65], 64, 1, 16, 128, F16, 40),
    ([513, 77, 128], 128, 2, 5, 192, F16, 25),
    ([1260, 1, 257, 512], 256, 2, 7, 256, BF16, 33),
    ([1500, 20], 16, 2, 16, 256, F16, 530),
]


@pytest.mark.parametrize("lens,P,HK,G,D,dtype,W", CASES)
@pytest.mark.parametrize("holes", [0.0, 0.5, 0.97])
def test_entries_anywhere(lens, P, HK, G, D, dtype, W, holes):
    c, K, V = open_cache(lens, P, HK, D, dtype)
    r = random.Random(W)
    lists, pages = [], c.tables()[0].cpu().numpy()
    for s, n in enumerate(lens):
        nb = -(-n // P)

        def entry():
            if r.random() < holes:
                return r.choice([-1, -1, -7, -(1 << 31), nb, nb + 1, (1 << 31) - 1])
            return r.randrange(nb) if nb else 0
        rows = [[entry() for _ in range(W)] for _ in range(HK)]
        rows[0][-1] = max(0, nb - 1)  # the token's own block, last
        lists.append(rows)
        for b in set(range(nb)) - {x for row in rows for x in row}:
            c.k(0)[int(pages[s, b])] = math.inf
            c.v(0)[int(pages[s, b])] = math.nan
    q = (2 * torch.randn((len(lens), HK * G, D), device="cuda", generator=gen(9))).to(dtype)
    check(c, K, V, lens, lists, q, P, dtype)


@pytest.mark.parametrize("pad", [1, 3, 31, 32, 255, 256, 257, 1000])
@pytest.mark.parametrize("P,D", [(8, 128), (64, 64), (256, 256)])
def test_lists_filled_in_front(pad, P, D):
    """-1 in front: a short sequence's blocks are no fewer for it."""
    lens = [P, 5 * P + 3, 1]
    c, K, V = open_cache(lens, P, 1, D, BF16)
    q = torch.randn((3, 4, D), device="cuda", generator=gen(4)).to(BF16)
    lists = [[[-1] * pad + row] for row in ([0] + [-1] * 5, [5, 0, 3, 1, 2, 4], [-1] * 5 + [0])]
    check(c, K, V, lens, lists, q, P, BF16)


def test_six_blocks_in_a_list_of_eight():
    c, K, V = open_cache([6 * 16], 16, 1, 128, F16)
    q = torch.randn((1, 8, 128), device="cuda", generator=gen(4)).half()
    check(c, K, V, [96], [[[-1, -1, -1, 0, 1, 2, 3, 5]]], q, 16, F16)


def test_drafts_that_share_a_falling_list():
    """The list of a sequence's last token for each of them: the first ones do not see what it begins with."""
    lens, new, P, HK, G, D = [40, 9, 400], [9, 9, 9], 8, 2, 4, 128
    c, K, V = open_cache(lens, P, HK, D, F16)
    row_seq = [s for s, x in enumerate(new) for _ in range(x)]
    row_len = [n - x + i + 1 for n, x in zip(lens, new) for i in range(x)]
    q = torch.randn((27, HK * G, D), device="cuda", generator=gen(6)).half()
    lists = [[list(range(-(-lens[s] // P) - 1, -1, -1))[:5] + [0] * max(0, 5 - -(-lens[s] // P))] * HK for s in row_seq]
    check(c, K, V, lens, lists, q, P, F16, [0, 9, 18, 27], row_seq, row_len)


def test_long_lists_of_blocks_that_short_sequences_lack():
    """1000 entries that fall to 0, of a sequence of 625 blocks and of 90 of one."""
    lens, P, HK, G, D = [5000] + [3] * 90, 8, 2, 8, 128
    c, K, V = open_cache(lens, P, HK, D, F16)
    q = torch.randn((91, HK * G, D), device="cuda", generator=gen(5)).half()
    check(c, K, V, lens, [[list(range(999, -1, -1))] * HK] * 91, q, P, F16)


def test_every_block_three_times_over_many_ctas():
    lens, P, HK, G, D = [20000, 64], 16, 1, 8, 128
    c, K, V = open_cache(lens, P, HK, D, BF16)
    q = torch.randn((2, G, D), device="cuda", generator=gen(5)).to(BF16)
    lists = [[list(range(1250)) * 3], [list(range(4)) * 937 + [-1, 3]]]
    check(c, K, V, lens, lists, q, P, BF16)


def test_captured_and_replayed_with_other_lists():
    lens, P, HK, G, D, W = [130, 64, 15], 16, 2, 4, 64, 40
    c, K, V = open_cache(lens, P, HK, D, F16)
    seqs, lists = i32([0, 1, 2]), torch.full((3, HK, W), -1, dtype=torch.int32, device="cuda")
    q = torch.randn((3, HK * G, D), device="cuda", generator=gen(3)).half()
    out = torch.zeros_like(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        c.attend_blocks(0, q, seqs, lists, out=out)
    r = random.Random(3)
    for _ in range(4):
        rows = [[[r.choice([-1, -1, -1, *range(10)]) for _ in range(W)] for _ in range(HK)] for _ in lens]
        lists.copy_(i32(rows).reshape(3, HK, W))
        graph.replay()
        torch.cuda.synchronize()
        close(out, [reference(q[s], K[s], V[s], n, P, [seen(row, -(-n // P)) for row in rows[s]], 1 / math.sqrt(D))
                    for s, n in enumerate(lens)], F16)
    del graph
    c.check()
