import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


# Tests that hold a wrong value.  They stay as they were written and run; tests/test_gpu_paged_bounds.py holds the right one.
WRONG = {
    "test_gpu_paged.py::test_write_bounds_what_the_device_arrays_say":
        "wants the tokens of positions 897 to 899, for which its table of 16 positions has no page, in the rows of positions 13 to 15, over "
        "the keys that belong there",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, why in WRONG.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.xfail(reason=why, strict=True))


@pytest.fixture(scope="session")
def golden_dir():
    return os.path.join(ROOT, "tests", "golden")
