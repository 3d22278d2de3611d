"""The in-tree build: every source and header the library is compiled from triggers a rebuild
(an edit to a header that the dependency list missed once left a stale library in place)."""
import os
import subprocess

import pytest

from invision_b200 import build


def test_every_source_is_a_build_dependency():
    csrc = os.path.join(os.path.dirname(build.__file__), "csrc")
    deps = set(build.deps())
    for f in os.listdir(csrc):
        if f.endswith((".cu", ".cuh", ".hpp", ".h")):
            assert os.path.join(csrc, f) in deps, f
    assert os.path.join(build.INCLUDE, "envgemm.h") in deps


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    """build() with its outputs in a folder of the test's; the commands it runs are listed, not run."""
    commands = []
    monkeypatch.setattr(build, "OUT", str(tmp_path / "libenvgemm.so"))
    monkeypatch.setattr(build, "VIEWS", str(tmp_path / "_views.so"))
    monkeypatch.setattr(build.subprocess, "check_call", lambda cmd: commands.append(cmd) or open(cmd[-1], "w").close())
    return commands


@pytest.mark.parametrize("fault", ["compiler", "no compiler", "no torch"])
def test_the_library_is_built_where_the_torch_extension_cannot_be(elsewhere, monkeypatch, capsys, fault):
    def run(cmd):
        elsewhere.append(cmd)
        if cmd[0] == "g++":
            if fault == "no compiler":
                raise FileNotFoundError(cmd[0])
            raise subprocess.CalledProcessError(1, cmd)
        open(cmd[-1], "w").close()

    monkeypatch.setattr(build.subprocess, "check_call", run)
    if fault == "no torch":
        monkeypatch.setitem(__import__("sys").modules, "torch", None)
    open(build.VIEWS, "w").close()  # one of an earlier build
    assert build.build(verbose=False) == build.OUT and os.path.exists(build.OUT)
    assert elsewhere[0][0] == build.NVCC
    assert not os.path.exists(build.VIEWS) and "warning" in capsys.readouterr().err


def test_the_torch_extension_is_rebuilt_for_another_torch_or_source(elsewhere, monkeypatch):
    pytest.importorskip("torch")

    def run(cmd):
        elsewhere.append(cmd)
        with open(cmd[-1], "w") as f:
            f.write("..".join(cmd))

    monkeypatch.setattr(build.subprocess, "check_call", run)
    for want in (1, 1):
        build.build_views(verbose=False)
        assert len(elsewhere) == want
    now = build.views_stamp()
    monkeypatch.setattr(build, "views_stamp", lambda: now.replace("torch ", "torch 9"))
    build.build_views(verbose=False)
    build.build_views(verbose=False)
    assert len(elsewhere) == 2


def test_the_binding_loads_no_extension_of_another_build(monkeypatch):
    torch = pytest.importorskip("torch")
    from invision_b200 import envg

    if not os.path.exists(build.VIEWS):
        pytest.skip("the torch extension was not built")
    for name, value in (("_torch", torch), ("_views", None), ("_Tensor", None)):
        monkeypatch.setattr(envg, name, value)
    now = build.views_stamp()
    monkeypatch.setattr(build, "views_stamp", lambda: now + " of another build")
    envg._load_views()
    assert envg._views is None and envg._Tensor is None
    monkeypatch.setattr(build, "views_stamp", lambda: now)
    envg._load_views()
    assert envg._views.stamp == now and envg._Tensor is torch.Tensor
