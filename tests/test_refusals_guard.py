"""Calls in order on memory that is not there are made only where no GPU is: every
test of refusals is skipped where the driver's device exists."""

from __future__ import annotations

import inspect

import pytest

import conftest
import test_drafting_args
import test_serving8_args


class Item:
    def __init__(self, name, fn, module):
        self.name, self.fixturenames, self.module, self.marks = name, list(inspect.signature(fn).parameters), module, []

    def add_marker(self, mark):
        self.marks.append(mark)


def items(module):
    return [Item(n, f, module) for n, f in vars(module).items() if n.startswith("test_") and inspect.isfunction(f) and f.__module__ == module.__name__]


@pytest.mark.parametrize("module", [test_serving8_args, test_drafting_args])
@pytest.mark.parametrize("there", [True, False])
def test_refusals_are_skipped_where_a_gpu_is(there, module, tmp_path, monkeypatch):
    monkeypatch.setattr(conftest, "KFD", tmp_path if there else tmp_path / "none")
    found = items(module)
    conftest.pytest_collection_modifyitems(found)
    assert sum("lib" in i.fixturenames for i in found) >= 4
    for item in found:
        assert [m.name for m in item.marks] == (["skip"] if there and "lib" in item.fixturenames else []), item.name


def test_others_are_not_skipped(tmp_path, monkeypatch):
    """A library of that name that is asked nothing on memory that is not there."""
    monkeypatch.setattr(conftest, "KFD", tmp_path)
    item = Item("test_other", lambda lib: None, conftest)
    conftest.pytest_collection_modifyitems([item])
    assert item.fixturenames == ["lib"] and not item.marks


@pytest.mark.parametrize("module", [test_serving8_args, test_drafting_args])
def test_every_test_that_calls_the_library_takes_it_as_lib(module):
    """The tests that use Lib are those that the rule above finds."""
    for name, fn in vars(module).items():
        if name.startswith("test_") and inspect.isfunction(fn) and fn.__module__ == module.__name__:
            code = inspect.getsource(fn)
            assert "lib" in inspect.signature(fn).parameters or not ("Lib(" in code or ".code(" in code or "check(lib" in code), name
