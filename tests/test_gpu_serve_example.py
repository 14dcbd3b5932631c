"""The serving example: its parts together, against the same tokens without them."""

import pytest

from aero_b200 import native_cuda as nc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_lib):
    nc.require_gpu()


def test_example_runs_and_books_close():
    from aero_b200.serve_example import serve
    r = serve(steps=40, samples=2)
    assert r["compacted"] >= 1 and len(r["live"]) <= 5
    assert r["highest"] == r["pages"] - 1  # compacted: the live pages are the pool's first
    for row in r["live"]:
        n, s = r["n"][row], (row - 3) // r["samples"]
        assert n == len(r["prompts"][s]) + 40 and int(r["length"][row]) == n - 1
        answer = r["history"][row, len(r["prompts"][s]) + 1:n].tolist()
        assert set(answer) <= set(r["allowed"])  # the mask held from the first adjusted token on
        # samples of one prompt share its tokens and differ after it
    a, b = [row for row in (3, 4)]
    n = len(r["prompts"][0])
    assert r["history"][a, :n].tolist() == r["history"][b, :n].tolist() == r["prompts"][0]
    assert r["history"][a, n] != r["history"][b, n]


def test_steps_agree_with_one_prompt():
    """Tokens taken one a step (forked after the prompt, pages moved on the way) give the logits of
    the same tokens taken as one prompt: the two forms of attention, the fork and the compaction
    change nothing but roundings (f16 cache rows and weights, 2^-11 each, over two layers: 1%)."""
    from aero_b200.pages import PagedCache
    from aero_b200.serve_example import PagedDecoder, i32
    c = PagedCache(2, 64, 16, 2, 64, 6, 16)
    net = PagedDecoder(c, 8, 256, 500, window=32, sinks=4, seed=3)
    tokens = [(11 * j + 5) % 500 for j in range(90)]
    with torch.cuda.stream(net.stream):
        def prompt(s, toks):
            c.extend(i32([s]), i32([len(toks)]))
            return net.forward(i32(toks), i32([s] * len(toks)), i32(range(len(toks))), i32([s]), i32([0, len(toks)]))
        prompt(5, tokens[:40])  # in the way of the pages, until it is freed
        prompt(0, tokens[:50])
        c.fork(i32([0]), i32([1]))
        for j in range(50, 90):
            c.extend(i32([1]), i32([1]))
            got = net.forward(i32([tokens[j]]), i32([1]), i32([j]), i32([1]))
            if j == 60:
                c.free(i32([5, 0]))
                c.compact()
        want = prompt(2, tokens)
        c.check()
        torch.cuda.synchronize()
    rms = want.pow(2).mean().sqrt()
    assert (got - want).abs().max() <= 0.05 * rms and (got - want).pow(2).mean().sqrt() <= 0.01 * rms
    net.close()
