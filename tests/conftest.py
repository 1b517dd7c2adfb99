import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on a B200)")


# A row of 20000 logits that are all the type's lowest number (bf16 and fp32: -3.4e38) has log-probabilities of -log 20000 = -9.9.  The definition there,
# x - logsumexp(x) in 64 bits, gives 0: beside 3.4e38 the 9.9 are less than half a unit of the last place (2^127 * 2^-53 = 2^74).  The test runs as it is and has
# to fail; test_gpu_beam_edges.py runs the same rows with the logarithm kept apart from the maximum.
_LOSES_THE_LOGARITHM = {"test_gpu_beams.py::test_masks_and_numbers_that_are_none[kind%d]" % i for i in (1, 2)}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.split("/")[-1] in _LOSES_THE_LOGARITHM:
            item.add_marker(pytest.mark.xfail(strict=True, raises=AssertionError, reason="its definition gives 0 for -log V beside logits of -3.4e38"))


@pytest.fixture(scope="session")
def cuda():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from kvmix_b200 import _lib
    _lib.lib()          # fail loudly if the library is not built
    return torch.device("cuda:0")


def pytest_terminal_summary(terminalreporter):
    """List the rounding-dominated rows admitted by the attention parity checks (tests/util.py)."""
    try:
        import util
    except Exception:
        return
    if util.ROUNDING_DOMINATED:
        terminalreporter.write_line("rounding-dominated rows admitted beyond 2e-3 (test, rows, worst error, upstream's own narrowing noise):")
        for rec in util.ROUNDING_DOMINATED:
            terminalreporter.write_line("  %s: %d row(s), %.3e (noise %.3e)" % rec)
