import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (run with -m gpu on the GPU box)")


# Tests whose expected value is wrong, and why.  They run as they are and have to fail.
WRONG_VALUES = {
    "test_gpu_mxfp4_linear.py::test_fp32_master_weight_and_bias_with_bf16_activations": (
        "expects the fp32 bias rounded to bf16 before the sum, two roundings where the layer makes one: a product of -1 and a bias "
        "of 1 + 2**-12 give 2**-12, and 0 that way; test_gpu_mxfp4_bias_types.py::test_fp32_master_weight_and_bias has the unrounded one"
    ),
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, reason in WRONG_VALUES.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.xfail(reason=reason, strict=True, raises=AssertionError))


@pytest.fixture(scope="session")
def device():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    return torch.device("cuda:0")


@pytest.fixture(scope="session")
def golden():
    import json

    with open(os.path.join(ROOT, "tests", "golden", "reference_known_answers.json")) as fh:
        return json.load(fh)
