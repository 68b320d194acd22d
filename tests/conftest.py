import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a HIP GPU (MI355X); run with -m gpu")
    config.addinivalue_line("markers", "slow: longer CPU oracle runs")


# Tests that hold a wrong value. By packed_plan's definition row i of a sequence is its token k_lens - q_lens + i; these
# expect k_out - cu_q[s + 1] + r, formed from the cut key count and the cut offset, where a sequence's rows pass the row
# buffer or its tokens the cache: q_lens [3, 4, 5], k_lens [10, 10, 10] in 8 rows give row 7, the first of five new
# ones, token 9 instead of 5; 2 new rows of 100 tokens in a cache of 50 give tokens 98 and 99 the slots of 48 and 49.
# The right values, written out, are in test_gpu_packed_limits.py.
_PLAN = "tests/test_gpu_packed.py::test_plan"
WRONG_VALUES = {
    f"{_PLAN}[q_lens4-k_lens4-9]", f"{_PLAN}[q_lens6-k_lens6-8]", f"{_PLAN}[q_lens8-k_lens8-4]", f"{_PLAN}_saturates",
    *(f"{_PLAN}_many_sequences[{s}]" for s in (1, 2, 63, 64, 65, 255, 256, 257, 1000, 4096)),
}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid in WRONG_VALUES:
            item.add_marker(pytest.mark.xfail(raises=AssertionError, strict=True,
                                              reason="expects the token of the cut lengths, not the row's own"))


@pytest.fixture(scope="session")
def dev():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    from appcorr_amd import _lib

    _lib.verify_runtime(0)
    return torch.device("cuda", 0)
