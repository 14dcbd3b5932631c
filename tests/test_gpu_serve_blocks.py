"""The serving example with tokens drawn by temperature and with attention over selected blocks."""

import pytest

from aero_b200 import native_cuda as nc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_lib):
    nc.require_gpu()


def check_shape(r):
    for s in r["live"]:
        assert int(r["length"][s]) == r["n"][s] - 1
        prompt = r["prompts"][(s - len(r["prompts"])) // r["samples"]]
        tokens = r["history"][s, :r["n"][s]].tolist()
        assert tokens[:len(prompt)] == prompt and all(t in r["allowed"] for t in tokens[len(prompt) + 1:])


def test_every_block_is_what_attention_without_blocks_gives():
    from aero_b200.serve_example import serve
    dense, blocks = serve(steps=20, seed=3), serve(steps=20, seed=3, blocks=16)  # more blocks than any sequence has
    assert torch.equal(dense["history"], blocks["history"]) and dense["n"] == blocks["n"]


def test_few_blocks():
    from aero_b200.serve_example import serve
    r = serve(steps=24, seed=1, blocks=2)
    check_shape(r)
    again = serve(steps=24, seed=1, blocks=2)
    assert torch.equal(r["history"], again["history"])


def test_tokens_drawn():
    from aero_b200.serve_example import serve
    greedy, one = serve(steps=16, seed=2), serve(steps=16, seed=2, temperature=0.9, top_k=1)
    assert torch.equal(greedy["history"], one["history"])  # of one token the first is drawn
    a, b = (serve(steps=16, seed=2, temperature=1.0, top_k=50, top_p=0.9, min_p=0.02, blocks=3) for _ in range(2))
    check_shape(a)
    assert torch.equal(a["history"], b["history"]) and not torch.equal(a["history"], greedy["history"])


def test_main(capsys, monkeypatch):
    from aero_b200 import serve_example
    monkeypatch.setattr("sys.argv", ["serve_example", "--steps", "6", "--temperature", "0.8", "--top-p", "0.9", "--blocks", "2"])
    serve_example.main()
    assert "sequences live" in capsys.readouterr().out
