import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


# Tests whose expected value is wrong: they run, and have to fail in the way that is said here.
EXPECTED_FAILURES = {
    "test_long_context_training_gpu.py::test_loss_and_gradients[True-a larger base, a SiLU gate]":
        (ValueError, "takes one set of dynamic frequencies, the row's, for documents of 50, 46, 31, 65 and 96 tokens: the ones of 46 and 31 are below the original length of 48 and alone not stretched at all"),
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, (error, reason) in EXPECTED_FAILURES.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.xfail(raises=error, reason=reason, strict=True))


@pytest.fixture(scope="session")
def gpu_device():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    return torch.device("cuda:0")
