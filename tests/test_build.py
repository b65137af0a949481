"""The build's order and what makes it run again (no compiler is called)."""
import os
import subprocess

import pytest
import torch

from flashprefill_b200 import _lib, build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Built files in a folder of their own; compilers that write an empty file, or fail where `broken` names them."""
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "EXT", str(tmp_path / "ext.so"))
    monkeypatch.setattr(build, "EXT_TAG", str(tmp_path / "ext.so.built_for"))
    monkeypatch.setattr(build, "nvcc_path", lambda: "/usr/local/cuda/bin/nvcc")
    calls, broken = [], set()

    def run(cmd, **kw):
        name = os.path.basename(cmd[0])
        calls.append(name)
        if name not in broken:
            open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, int(name in broken), "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    return calls, broken


def test_the_library_does_not_wait_for_the_binding(tree):
    calls, broken = tree
    broken.add("g++")
    with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
        build.build()
    assert calls == ["nvcc", "g++"] and os.path.exists(build.LIB) and not os.path.exists(build.EXT)


def test_the_binding_is_built_again_for_another_torch(tree, monkeypatch):
    calls, _ = tree
    build.build()
    build.build()
    assert calls == ["nvcc", "g++"]
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build()
    assert calls == ["nvcc", "g++", "g++"]
    os.remove(build.EXT_TAG)  # one built before it was recorded
    build.build()
    assert calls == ["nvcc", "g++", "g++", "g++"]


def test_a_binding_for_another_torch_is_refused(monkeypatch):
    if not os.path.exists(_lib.EXT_PATH):
        build.build()
    monkeypatch.setattr(_lib, "_ext", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    with pytest.raises(ImportError, match="built for torch .*, this is 0.0.1"):
        _lib.ext()
    assert _lib._ext is None
