"""A library of another ABI version is refused by its version, whatever names it lacks."""

import pytest

from tattn import _lib


class Older:
    """As ctypes shows a library of version 2 that has none of the entry points added since."""

    def tattn_abi_version(self):
        return 2

    def __getattr__(self, name):
        raise AttributeError(f"undefined symbol: {name}")


def test_an_older_library_is_refused_by_its_version(monkeypatch):
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib.ctypes, "CDLL", lambda path: Older())
    with pytest.raises(RuntimeError, match=f"ABI version 2, expected {_lib.ABI_VERSION}"):
        _lib.load()
    assert _lib._lib is None


def test_entry_points_added_since_version_2_have_a_version_of_their_own():
    assert _lib.ABI_VERSION > 2 and _lib.load().tattn_abi_version() == _lib.ABI_VERSION
