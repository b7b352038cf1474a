"""Which parts a build makes, and what each needs, with the compilers replaced."""

from __future__ import annotations

import pytest

from robustgemq_b200 import _lib, build


@pytest.fixture
def made(monkeypatch):
    """Everything stale; the library's compile is noted instead of run."""
    done = []
    monkeypatch.setattr(build, "_stale", lambda: True)
    monkeypatch.setattr(build, "_ext_stale", lambda: done.append("asked for the binding") or True)
    monkeypatch.setattr(build, "_build_lib", lambda verbose, jobs: done.append("library"))
    return done


def test_the_library_is_built_where_the_binding_cannot_be(monkeypatch, made):
    def no_compiler(obj):
        raise FileNotFoundError("g++")

    monkeypatch.setattr(build, "_ext_commands", no_compiler)
    with pytest.raises(Exception, match="g\\+\\+"):
        build.build()
    assert "library" in made


def test_loading_the_library_leaves_the_binding_alone(monkeypatch, made):
    whole = _lib._lib
    monkeypatch.setattr(_lib, "_lib", None)
    lib = _lib.load()
    assert made == ["library"] and lib.gemq_version() == (whole or lib).gemq_version()


def test_a_binding_of_another_torch_is_stale(monkeypatch, tmp_path):
    ext = tmp_path / "ext.so"
    ext.write_bytes(b"")
    stamp = tmp_path / "stamp"
    monkeypatch.setattr(build, "EXT", ext)
    monkeypatch.setattr(build, "EXT_STAMP", stamp)
    assert not build._ext_stale()  # a binding without a stamp goes by its sources
    stamp.write_text(build._torch_version())
    assert not build._ext_stale()
    stamp.write_text("0.0.1")
    assert build._ext_stale()
