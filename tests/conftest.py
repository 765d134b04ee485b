import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")
    # The library is built in-tree ahead of the tests (`__graft_entry__.build()`); it is git-ignored, so a fresh
    # checkout has none.  Build it once then, rather than fail every test that imports `lcm` (a no-op otherwise).
    lib = os.environ.get("LCMHIP_LIB") or os.path.join(ROOT, "chimera-llm_amd", "lcm", "liblcm_hip.so")
    if not os.path.exists(lib) and os.path.exists("/opt/rocm/bin/hipcc"):
        import __graft_entry__
        __graft_entry__.build()


# Kept as it is and run, but expected to fail: its last part holds that a sequence of 2^31 - 1 positions stores its two newest rows
# at positions 14 and 15 of a cache of 16.  They are positions 2^31 - 3 and 2^31 - 2, which that cache does not have, and the rows
# stored there before are lost.  The rest of it, and the right expectation, is test_gpu_paged_edges.py::test_bad_places_are_skipped.
WRONG_VALUE = "test_gpu_paged.py::test_paged_append_skips"


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.endswith(WRONG_VALUE):
            item.add_marker(pytest.mark.xfail(raises=AssertionError, strict=True, reason="expects rows without a place to be stored over older ones"))


@pytest.fixture(scope="session")
def normalizer():
    import oracle
    return oracle.load_dummy_normalizer()
