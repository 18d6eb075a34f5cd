import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200); run with -m gpu")


@pytest.hookimpl(wrapper=True)
def pytest_runtest_call(item):
    """A test that reaches for the reference's own code where it is not built (oracle/_ref) is skipped with that
    reason, as the tests that ask for it beforehand are."""
    import oracle

    try:
        return (yield)
    except oracle.ReferenceMissing as missing:
        pytest.skip(str(missing))
