"""bench.py's reference arm without the reference: it says so, and times nothing in its place."""

import json
import os
import sys
from types import SimpleNamespace

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("workload", ["c1", "c5"])
def test_no_reference_no_figure(monkeypatch, capsys, workload):
    monkeypatch.syspath_prepend(ROOT)
    import bench
    import oracle as O
    from aero_b200 import synth
    assert "oracle" in sys.modules
    monkeypatch.setattr(O, "ref_available", lambda: False)

    def never(*_a, **_k):
        raise AssertionError("timed something all the same")

    for name in ("moe_block", "ref_block"):
        monkeypatch.setattr(O, name, never)
    monkeypatch.setattr(synth, "make_layer", never)
    bench.run_reference(SimpleNamespace(steps=2, warmup=3), 1, synth.CONFIGS[workload])
    lines = capsys.readouterr().out.strip().splitlines()
    assert len(lines) == 1
    line = json.loads(lines[0])
    assert line["impl"] == "reference" and line["unavailable"] and "value" not in line
