import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200, sm_100a)")
    config.addinivalue_line("markers", "slow: long CPU-side oracle runs")


@pytest.hookimpl(hookwrapper=True)
def pytest_runtest_call(item):
    """A test that calls the reference's own build where there is none is skipped, as those are that ask
    for it first."""
    outcome = yield
    from oracle import ref
    if outcome.excinfo and issubclass(outcome.excinfo[0], ref.NotBuilt):
        outcome.force_exception(pytest.skip.Exception("oracle/_ref not built"))


@pytest.fixture(scope="session")
def golden():
    import numpy as np
    return np.load(os.path.join(ROOT, "tests", "golden", "attention_sync_oracle.npz"))
