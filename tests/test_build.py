"""`build()` of a tree whose tests are other ones, or none: every kernel that is not a test's own is still built."""
import sys

import pytest

import __graft_entry__ as entry
from trainkernel_b200 import runtime


def prebuilt(monkeypatch, tmp_path):
    """How many kernels `build()` would compile, without compiling them."""
    built = []
    monkeypatch.setattr(runtime, "CACHE_DIR", tmp_path)
    monkeypatch.setattr(runtime, "build_cubin", built.append)
    count = entry._prebuild_kernels()
    assert count == len(built)
    return count


def without(monkeypatch, *names):
    import tests
    for name in names:
        monkeypatch.delattr(tests, name, raising=False)
        monkeypatch.setitem(sys.modules, f"tests.{name}", None)


@pytest.mark.parametrize("absent", [("operator_cases",), ("operator_cases", "dp_check", "cases")])
def test_kernels_are_built_without_the_tests_modules(monkeypatch, tmp_path, absent):
    without(monkeypatch, *absent)
    assert prebuilt(monkeypatch, tmp_path) > 10                # the steps of the package and of the bench


def test_kernels_are_built_without_a_tests_package(monkeypatch, tmp_path):
    for name in [name for name in sys.modules if name == "tests" or name.startswith("tests.")]:
        monkeypatch.delitem(sys.modules, name)
    monkeypatch.setitem(sys.modules, "tests", None)
    assert prebuilt(monkeypatch, tmp_path) > 10
