import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (REPO, os.path.join(REPO, "oracle")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200, sm_100a)")


@pytest.fixture(scope="session")
def oracle_mod():
    import oracle as o

    o.lib()
    return o


# Two cases compare the loss with a value that is none: their plain form adds an id's entries one by one,
# sum p (log p - log q), so two equal entries of an id that the model is sure of give -ln 2 where the divergence
# is 0.  They stay as they were; test_gpu_divergence.py has the same lists with the divergence of distinct ids.
WRONG_VALUE = ("test_gpu_logits.py::test_distill_lists[False]", "test_gpu_logits.py::test_distill_lists[True]")


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.endswith(WRONG_VALUE):
            item.add_marker(pytest.mark.xfail(strict=True, reason="adds up the entries of an id one by one"))
