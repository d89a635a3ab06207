import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs the HIP kernels)")


@pytest.fixture(scope="session")
def orc():
    import oracle

    return oracle


# Tests that expect what is now known to be wrong.  They run as they are and have to
# fail at that value; the tests named beside them hold the right one.
_WRONG_VALUE = {
    "test_gpu_beam.py::test_select_masked_rows":
        "its form adds a row's log-sum to a maximum at the type's lowest or largest value, where the sum and the beam's "
        "score vanish: 0 for -19 + log_softmax = -25.9 (test_gpu_beam_scores.py::test_masked_rows)",
    "test_gpu_beam.py::test_select_flat_and_peaked_rows":
        "the same, in its last rows of about 1e38 (test_gpu_beam_scores.py::test_flat_and_peaked_rows)",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, reason in _WRONG_VALUE.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.xfail(raises=AssertionError, strict=True, reason=reason))
