"""When the build command builds: file times, and what the binding was built against."""
import types

import pytest
import torch

from muon_sr_b200 import _lib
from muon_sr_b200 import build as B


class Compiles(Exception):
    pass


@pytest.fixture
def built(tmp_path, monkeypatch):
    """A library and a binding newer than every source; compiling raises instead."""
    def run(*args, **kwargs):
        raise Compiles(args)
    for name in ("LIB", "BINDING"):
        path = tmp_path / name
        path.write_text("")
        monkeypatch.setattr(B, name, str(path))
    monkeypatch.setattr(B, "BINDING_FOR", str(tmp_path / "for"), raising=False)
    monkeypatch.setattr(B.subprocess, "run", run)
    if hasattr(_lib, "built_for"):
        (tmp_path / "for").write_text(_lib.built_for())
    return tmp_path


def test_current_build_is_kept(built):
    assert B.build() == B.LIB
    with pytest.raises(Compiles):
        B.build(force=True)


def test_another_torch_builds_the_binding_again(built, monkeypatch):
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    with pytest.raises(Compiles):
        B.build()


def test_a_binding_of_unknown_origin_is_built_again(built):
    (built / "for").unlink()
    with pytest.raises(Compiles):
        B.build()


def test_binding_of_another_torch_is_refused(monkeypatch):
    """It could load all the same and read the tensors' fields where that torch keeps them."""
    other = types.SimpleNamespace(built_for="torch 9.9.9+other")
    import muon_sr_b200
    monkeypatch.setattr(_lib, "_native_module", None, raising=False)
    monkeypatch.setattr(muon_sr_b200, "_native", other, raising=False)
    with pytest.raises(RuntimeError, match="built for torch 9.9.9.*python -m muon_sr_b200.build"):
        _lib.native()


def test_binding_names_this_torch():
    assert _lib.native().built_for == _lib.built_for()
