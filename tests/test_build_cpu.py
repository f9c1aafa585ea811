"""What makes build.py build again."""
import importlib
import importlib.metadata
import importlib.util
import os

import pytest

import bpt


@pytest.fixture
def build():
    path = os.path.join(os.path.dirname(os.path.dirname(bpt.__file__)), "build.py")
    spec = importlib.util.spec_from_file_location("bpt_build", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_binding_is_stale_after_another_torch(build, monkeypatch, tmp_path):
    """The binding is tied to torch's C++ ABI: another version makes it out of date, whatever the
    files' times, and so does not knowing which version it was built with."""
    out, stamp = tmp_path / "_bind.so", tmp_path / "bind.torch"
    out.write_bytes(b"")
    monkeypatch.setattr(build, "BIND_OUT", str(out))
    monkeypatch.setattr(build, "BIND_STAMP", str(stamp))
    assert not build.bind_up_to_date()
    stamp.write_text(build.bind_built_for())
    assert build.bind_up_to_date()
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0.1")
    assert not build.bind_up_to_date()


@pytest.mark.parametrize("error,message", [
    (ImportError("undefined symbol: _ZN3c10"), "does not load .undefined symbol.*rebuild"),
    (ModuleNotFoundError("No module named 'bpt._bind'"), "is not built")])
def test_binding_that_does_not_load_says_why(monkeypatch, error, message):
    """A module built for another torch is not reported as missing."""
    from bpt import evict
    real = importlib.import_module

    def fake(name, package=None):
        if name == "._bind":
            raise error
        return real(name, package)
    monkeypatch.setattr(evict, "_BIND", None)
    monkeypatch.setattr(importlib, "import_module", fake)
    with pytest.raises(ImportError, match=message):
        evict._bind()
