"""pytest setup: the `gpu` marker, repo imports, and the golden fixtures."""

import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "oracle"))

GOLDEN = os.path.join(ROOT, "tests", "golden", "golden.npz")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200); run with -m gpu")


@pytest.fixture(scope="session")
def golden():
    return dict(np.load(GOLDEN, allow_pickle=False))


@pytest.fixture(scope="session")
def cuda_lib():
    """The built CUDA library (builds it if missing); GPU tests fail loudly without it."""
    from aero_b200 import build, native_cuda
    build.build()
    return native_cuda.lib()


# Tests that expect what the interface rules out. They stay as they were and run, and have to fail.
WRONG_VALUES = {
    "test_gpu_pages_blocks.py::test_many_tokens_of_one_list_and_long_lists":
        "expects a list's entries past as many as the token has blocks to be left out; every entry counts "
        "(the same call with the right values: test_gpu_pages_lists.py)",
}


def pytest_collection_modifyitems(items):
    for item in items:
        why = WRONG_VALUES.get(f"{item.path.name}::{item.name}")
        if why:
            item.add_marker(pytest.mark.xfail(reason=why, strict=True))
