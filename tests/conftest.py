import ctypes
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "oracle"), os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs through libnship on the device)")


@pytest.fixture(autouse=True)
def moe_split_least(request, monkeypatch):
    """NSHIP_MOE_SPLIT_MIN in a test's environment, the least slots an expert for
    which a layer takes two fp16 pieces.  The library does not read the environment:
    it is told before every call that these tests make of it."""
    if request.module.__name__ not in ("test_moe_topk_gpu", "test_newton_schulz_gpu"):
        yield
        return
    from neuralscript_amd import runtime
    plain = runtime.lib

    def lib():
        L = plain()
        L.nsh_test_moe_split_least(ctypes.c_int64(int(os.environ.get("NSHIP_MOE_SPLIT_MIN", "0"))))
        return L

    monkeypatch.setattr(runtime, "lib", lib)
    yield
    plain().nsh_test_moe_split_least(ctypes.c_int64(0))
