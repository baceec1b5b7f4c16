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


# -- without the operators' compiled host path -------------------------------------------------------------------

def no_host_path(*_, **__):
    raise RuntimeError("trainkernel: building the operators' host path failed:\nno headers")


def test_build_goes_on_without_the_host_path(monkeypatch, capsys):
    from trainkernel_b200 import noalloc, operators
    for module, name in ((runtime, "build_library"), (runtime, "library"), (noalloc, "build_library"), (operators, "build_library")):
        monkeypatch.setattr(module, name, lambda **_: None)
    monkeypatch.setattr(operators, "build_host", no_host_path)
    monkeypatch.setattr(entry, "_prebuild_kernels", lambda: 7)
    entry.build()
    said = capsys.readouterr().out
    assert "host path skipped" in said and "7 sm_100a kernels" in said


def test_operators_run_without_the_host_path(monkeypatch):
    import torch
    from trainkernel_b200 import operators
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda index: (10, 0))
    monkeypatch.setattr(operators, "_usable", {})
    monkeypatch.setattr(operators, "fast", None)
    monkeypatch.setattr(operators, "_host", None)
    monkeypatch.setattr(operators, "build_host", no_host_path)
    with pytest.warns(RuntimeWarning, match="without their compiled host path"):
        assert operators.require_device(torch.device("cuda", 0)) == 0
    assert operators.fast is None and operators.require_device(torch.device("cuda", 0)) == 0      # said once
