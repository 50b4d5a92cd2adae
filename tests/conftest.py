import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200, sm_100a)")


# Tests that pin a value which is not the operator's, each with the test that holds the right one.
_PINS_A_WRONG_VALUE = {
    "test_losses_gpu.py::test_masked_logits":
        "expects log-probability 0 of a label in a row whose logits are all alike (the type's lowest or highest value); log softmax "
        "is -log(vocab) there: tests/test_losses_values_gpu.py::test_masked_rows, test_rows_of_one_value",
}


def pytest_collection_modifyitems(items):
    for item in items:
        reason = _PINS_A_WRONG_VALUE.get(item.nodeid.split("/")[-1].split("[")[0])
        if reason:
            item.add_marker(pytest.mark.xfail(reason=reason, raises=AssertionError, strict=True))


@pytest.fixture(scope="session")
def golden():
    import torch
    return torch.load(os.path.join(ROOT, "tests", "golden", "golden_quant.pt"))
