import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
HERE = os.path.dirname(os.path.abspath(__file__))
if HERE not in sys.path:
    sys.path.insert(0, HERE)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200); run with -m gpu")


# Tests of what is refused before a device is touched: they call the library with addresses of nothing.  What it does not refuse ends, without a
# device, in that error; with one the addresses would be read.
WITHOUT_A_DEVICE = {"test_cabi.py", "test_paged_overlap.py", "test_paged_refusals.py", "test_tree_overlap.py", "test_tree_refusals.py"}


def pytest_collection_modifyitems(items):
    mine = [i for i in items if os.path.basename(str(i.fspath)) in WITHOUT_A_DEVICE and i.get_closest_marker("gpu") is None]
    if mine:
        import torch
        if torch.cuda.is_available():
            for i in mine:
                i.add_marker(pytest.mark.skip(reason="calls the library with addresses of nothing: for machines without a device"))


@pytest.fixture(scope="session")
def golden_dir():
    return os.path.join(ROOT, "tests", "golden")
