"""Loading a library that does not have every call of the binding."""
import ctypes

import pytest

from vmonarch_b200 import _native as N


def test_a_library_without_a_call_is_told_to_be_rebuilt(monkeypatch):
    class Old:
        class Entry:
            def __call__(self, *a):
                return N.ABI_VERSION

        def __init__(self, *_):
            self.vmb_abi_version = Old.Entry()

    monkeypatch.setattr(ctypes, "CDLL", Old)
    with pytest.raises(ImportError, match="rebuild it"):
        N._load()
