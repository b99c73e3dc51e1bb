import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a HIP GPU (MI355X); parity tests proper")
    config.addinivalue_line("markers", "slow: long-running")


# A test whose expected values are wrong, kept as it was written: fifty logits of the
# type's lowest value are a uniform row, whose loss is log 50 and whose p is 1 / 50
# (torch.nn.functional.cross_entropy's too); it expects 0 and 1.
WRONG = {"test_logits_all_at_the_lowest_value":
         "expects loss 0 and p = 1 of a uniform row of 50; they are log 50 and 1 / 50"}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.name in WRONG:
            item.add_marker(pytest.mark.xfail(reason=WRONG[item.name], strict=True))
