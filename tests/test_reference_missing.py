"""What the oracle does where the reference's own code is not built."""
from __future__ import annotations

import numpy as np
import pytest

import oracle


@pytest.mark.parametrize("path,call", [
    ("REF_ONBOARD_PATH", lambda: oracle.onboard_reference(np.zeros((1, 4148), np.float32), np.zeros((1, 10), np.float32))),
    ("REF_ONBOARD_CR_PATH", lambda: oracle.onboard_reference_cr(np.zeros((1, 4148), np.float32),
                                                                np.zeros((1, 10), np.float32))),
    ("REF_TRAINING_PATH", lambda: oracle.ref_training()),
])
def test_a_missing_build_has_an_error_of_its_own(monkeypatch, path, call):
    monkeypatch.setattr(oracle, path, "/nowhere/lib.so")
    for loaded in ("_ref_training", "_ref_onboard", "_ref_onboard_cr"):
        monkeypatch.setattr(oracle, loaded, None)
    with pytest.raises(oracle.ReferenceMissing, match="reference build not available"):
        call()


def test_a_test_that_meets_it_is_skipped(request):
    """conftest.py turns it, and no other error, into a skip with its reason."""
    class Reached(Exception):
        pass

    hook = next(p for p in request.config.pluginmanager.get_plugins()
                if getattr(p, "__file__", "") == __file__.replace("test_reference_missing", "conftest"))
    run = hook.pytest_runtest_call(request.node)
    next(run)
    with pytest.raises(pytest.skip.Exception, match="not available"):
        run.throw(oracle.ReferenceMissing("it is not available"))
    run = hook.pytest_runtest_call(request.node)
    next(run)
    with pytest.raises(Reached):
        run.throw(Reached())
