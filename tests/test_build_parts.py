"""The library is built whatever becomes of the extension modules around it; no compiler runs here."""
import os

import pytest
import torch

from arcagi2_flashnext_dots3_amd import build


@pytest.fixture
def commands(tmp_path, monkeypatch):
    """Commands as build() would run them, each leaving an empty file at its output."""
    ran = []

    def run(cmd):
        ran.append(cmd)
        if any("py_tensors.cpp" in c for c in cmd) and run.broken:
            raise RuntimeError("build failed: torch headers that do not compile")
        open(cmd[cmd.index("-o") + 1], "w").close()
        return ""
    run.broken = False
    monkeypatch.setattr(build, "_run", run)
    monkeypatch.setattr(build, "REPO", str(tmp_path))
    for name in ("LIB", "NATIVE", "TENSORS"):
        monkeypatch.setattr(build, name, str(tmp_path / (name + ".so")))
    return ran, run


def test_all_parts(commands):
    assert build.build() == build.LIB and all(os.path.exists(p) for p in (build.LIB, build.NATIVE, build.TENSORS))


def test_without_torchs_headers(commands, tmp_path, monkeypatch):
    """A stale module goes, as _native's does without Python's headers."""
    open(build.TENSORS, "w").close()
    monkeypatch.setattr(torch, "__file__", str(tmp_path / "torch" / "__init__.py"))
    assert build.build() == build.LIB and os.path.exists(build.LIB) and os.path.exists(build.NATIVE)
    assert not os.path.exists(build.TENSORS) and not any("py_tensors.cpp" in c for cmd in commands[0] for c in cmd)


def test_without_torch(commands, monkeypatch):
    import sys
    monkeypatch.setitem(sys.modules, "torch", None)            # import torch raises ImportError
    assert build.build() == build.LIB and os.path.exists(build.LIB) and not os.path.exists(build.TENSORS)


def test_with_headers_that_do_not_compile(commands):
    commands[1].broken = True
    with pytest.raises(RuntimeError, match="do not compile"):
        build.build()
    assert os.path.exists(build.LIB) and os.path.exists(build.NATIVE) and not os.path.exists(build.TENSORS)
