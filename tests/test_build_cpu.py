"""When the library and the extension module are built: the module fits one torch and
one Python, and the library needs neither."""
import importlib.util
import os

import pytest

from rustorch_b200 import build as b


@pytest.fixture(scope="module", autouse=True)
def built():
    b.build()


def test_up_to_date_after_a_build():
    """Also where the newest file is the one with the compiler's flags: objects
    older than it are compiled again, and the next build finds nothing to do."""
    assert not b.needs_build() and not b.ops_stale()


def test_objects_are_as_new_as_the_flags():
    flags = os.path.getmtime(b.__file__)
    assert all(os.path.getmtime(b._obj(s)) >= flags for s in b._sources() if os.path.exists(b._obj(s)))


def test_another_torch_makes_the_module_stale(monkeypatch):
    """What `python -m rustorch_b200.build` is advised for when the module no
    longer loads."""
    called = []
    monkeypatch.setattr(b, "_build_ops", lambda: called.append(1))
    monkeypatch.setattr(b, "_torch_tag", lambda: "another torch")
    assert b.ops_stale()
    b.build()
    assert called == [1]


def test_a_module_without_its_stamp_is_stale(monkeypatch, tmp_path):
    monkeypatch.setattr(b, "OPS_STAMP", str(tmp_path / "none"))
    assert b.ops_stale()


def test_the_library_builds_without_torch(monkeypatch, capsys):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec",
                        lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setattr(b, "_build_ops", lambda: pytest.fail("needs torch"))
    assert b._torch_tag() is None
    assert b.build() == b.LIB and os.path.exists(b.LIB)
    assert "torch" in capsys.readouterr().err
