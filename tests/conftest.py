import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a ROCm GPU (MI355X); run with -m gpu")


def pytest_collection_modifyitems(items):
    """Cases that hold a value that has been shown to be wrong.  They stay as they are, and run."""
    reason = ("the expected loss gives a label outside the vocabulary the gradient of -logsumexp, where the log-probability that the operator "
              "returns, and that the same case checks, is the constant 0; test_adapters_labels_gpu.py has these sizes with that value's gradient")
    for item in items:
        if item.name.startswith("test_training_against_64_bits[") and item.path.name == "test_adapters_gpu.py" and item.callspec.params["T"] > 4:
            item.add_marker(pytest.mark.xfail(reason=reason, raises=AssertionError, strict=True))


@pytest.fixture(scope="session")
def cuda_device():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("a test marked gpu was run without a GPU")
    return torch.device("cuda:0")
