import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "oracle"), os.path.join(ROOT, "ferrum-cpu_amd")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs the HIP path through the C ABI)")


# Tests that hold a value that has been shown to be wrong: they run as they are and are expected to fail.
HOLD_WRONG_VALUES = {
    "test_gpu_tree_accept.py::test_rows_outside_beyond_and_in_place":
        "its third call wants 4 rows accepted behind 30 in a cache of 33 (a length of 34, rows 33 and 34 never "
        "stored); test_gpu_tree_accept_bounds.py has what is right, and this test's other calls",
    "test_gpu_gqa_uses.py::test_single_tokens_behind_an_accepted_tree":
        "it wants self.pos one past the position that forward_one fed over an f32 cache, where a program that steps "
        "by self.pos has always found that position; test_gpu_llama_places.py has the rest of it",
}


def pytest_collection_modifyitems(items):
    for item in items:
        reason = HOLD_WRONG_VALUES.get(item.nodeid.split("/")[-1])
        if reason:
            item.add_marker(pytest.mark.xfail(reason=reason, strict=True))


@pytest.fixture(scope="session")
def orc():
    import oracle

    oracle.build()
    return oracle


@pytest.fixture(scope="session")
def fh():
    """The product library on cuda:0, through its C ABI."""
    import ferrum_hip

    ctx = ferrum_hip.Context(0)
    yield ctx
    ctx.close()
