"""When the C++ binding is built again, and how its file gets into place."""
import subprocess
from pathlib import Path

import pytest
import torch

from dflash_mlx_b200.csrc import build


@pytest.fixture
def place(tmp_path, monkeypatch):
    """The files in a folder of their own and a compiler that only writes its output; returns the outputs it was asked for."""
    monkeypatch.setattr(build, "BINDING", tmp_path / "_native.so")
    monkeypatch.setattr(build, "BINDING_STAMP", tmp_path / "build" / "_native.torch")
    asked = []

    def run(cmd, **_):
        out = Path(cmd[cmd.index("-o") + 1])
        asked.append(out)
        # nobody may find this file under the binding's name before it is whole
        assert out != build.BINDING
        out.write_text("half")
        if run.fails:
            return subprocess.CompletedProcess(cmd, 1, "", "error")
        out.write_text("whole")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    run.fails = False
    monkeypatch.setattr(build.subprocess, "run", run)
    asked.append(run)
    return asked


def test_built_once_and_again_for_another_torch(place, monkeypatch):
    assert not build.binding_fits()
    build.build_binding()
    assert build.BINDING.read_text() == "whole" and build.binding_fits() and len(place) == 2
    build.build_binding()
    assert len(place) == 2                                # nothing is newer
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    assert not build.binding_fits()
    build.build_binding()
    assert len(place) == 3 and build.binding_fits()
    build.BINDING_STAMP.unlink()                          # a binding that came without its stamp is trusted
    assert build.binding_fits()


def test_a_failed_build_leaves_the_old_file(place, monkeypatch):
    build.build_binding()
    place[0].fails = True
    with pytest.raises(RuntimeError):
        build.build_binding(force=True)
    assert build.BINDING.read_text() == "whole"
    assert [p.name for p in build.BINDING.parent.iterdir() if p.is_file()] == ["_native.so"]
