import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


# The oracle of this test rounds a second moment below 2^-14 of its block's scale twice, stochastically and then to nearest: 2
# units of 2^-16 that decay by 0.1 % a step come out as 2 units whatever the random bits, which is what it is rounded
# stochastically to avoid.  The cases whose values reach that far down are expected to differ from the kernel;
# test_gpu_adamw_rounding.py has the oracle that rounds once.
_ROUNDED_TWICE = ["test_gpu_adamw.py::test_8_bit_moments[%s]" % k for k in
                  ("3x257", "1x2048", "5x8191", "6x4096", "1x100003", "63x5", "64x7", "65x9", "200x37", "3x1048576")]


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.endswith(tuple(_ROUNDED_TWICE)):
            item.add_marker(pytest.mark.xfail(reason="the oracle rounds small second moments twice", strict=True))


@pytest.fixture(scope="session")
def orc():
    import oracle
    oracle.lib()
    oracle.set_threads(min(16, oracle.max_threads()))
    return oracle


@pytest.fixture(scope="session")
def hip():
    """numpy-level facade over the C-ABI of libsliced_hip.so on device 0."""
    from sliced_amd import numpy_api
    numpy_api.init(0)
    return numpy_api


# Direct GPU-versus-oracle deviations that the full-size parity tests record, printed as one table
# at the end of the run (and asserted against their ceilings where they are recorded).
_DEVIATIONS = []


@pytest.fixture(scope="session")
def deviations():
    def record(config, what, value, ceiling):
        _DEVIATIONS.append((config, what, float(value), float(ceiling)))
        print("deviation  %-34s %-44s %.3e  (ceiling %.1e)" % (config, what, value, ceiling), flush=True)
        assert value <= ceiling, (config, what, value, ceiling)
    return record


def pytest_terminal_summary(terminalreporter):
    if not _DEVIATIONS:
        return
    terminalreporter.write_line("direct GPU-vs-oracle deviations (worst element per case)")
    for config, what, value, ceiling in _DEVIATIONS:
        terminalreporter.write_line("  %-34s %-44s %.3e  (ceiling %.1e)" % (config, what, value, ceiling))
