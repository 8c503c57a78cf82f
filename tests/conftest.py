import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on the B200 box)")


# Tests whose expected value is wrong, and why.  They stand as they are and have to fail.
WRONG_VALUE = {
    "test_compact_does_not_write_into_a_page_that_others_share":
        "expects a row of 64 positions to have 63 after a move that was refused, while no byte of its page may change: its position "
        "62 would then hold draft 2, which was not accepted (the accepted ones are 0, 1 and 3). The row stays at 64: "
        "test_pages_compact_refused.py",
}


def pytest_collection_modifyitems(config, items):
    for it in items:
        if it.name in WRONG_VALUE:
            it.add_marker(pytest.mark.xfail(reason=WRONG_VALUE[it.name], strict=True))
    try:
        import torch
        has_gpu = torch.cuda.is_available()
    except Exception:
        has_gpu = False
    if has_gpu:
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for it in items:
        if "gpu" in it.keywords:
            it.add_marker(skip)
