"""What the build needs and when it builds the torch binding again."""
import importlib.util
import os
import sysconfig
import types

import pytest

from rustgears_b200 import build


def test_library_builds_without_torch(monkeypatch, tmp_path):
    """The C ABI needs nvcc and NCCL only; the binding is left out."""
    build.build()
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setattr(build, "BIND", str(tmp_path / "_serving_bind.so"))
    assert build.build() == build.LIB
    assert not os.path.exists(build.BIND)


@pytest.fixture
def fake_torch(monkeypatch, tmp_path):
    """A torch folder of its own, and a compiler that only writes its output."""
    torch = tmp_path / "torch"
    (torch / "lib").mkdir(parents=True)
    (torch / "lib" / "libtorch_cuda.so").touch()
    (torch / "version.py").write_text("__version__ = '9.9.1+cu1'\n")
    monkeypatch.setattr(build, "BIND", str(tmp_path / "_serving_bind.so"))
    monkeypatch.setattr(build, "OBJ", str(tmp_path / "obj"))
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: types.SimpleNamespace(
        submodule_search_locations=[str(torch)]) if name == "torch" else find(name, *a))
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build.subprocess, "run", run)
    return torch, runs


def test_binding_follows_torch_and_python(fake_torch, monkeypatch):
    torch, runs = fake_torch
    for _ in range(2):
        assert build.build_binding() == build.BIND
    assert len(runs) == 1
    (torch / "version.py").write_text("__version__ = '9.9.2+cu1'\n")
    build.build_binding()
    build.build_binding()
    assert len(runs) == 2 and any("9.9.2+cu1" in a for a in runs[1])
    var = sysconfig.get_config_var
    monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "cpython-399" if name == "SOABI" else var(name))
    build.build_binding()
    build.build_binding()
    assert len(runs) == 3


def test_no_binding_for_a_torch_without_cuda(fake_torch):
    torch, runs = fake_torch
    (torch / "lib" / "libtorch_cuda.so").unlink()
    assert build.build_binding() is None and not runs


def test_binding_names_its_torch(monkeypatch):
    torch = pytest.importorskip("torch")
    from rustgears_b200 import serving
    assert serving._bind.torch_version == torch.__version__
    monkeypatch.setattr(torch, "__version__", "0.0")
    spec = importlib.util.spec_from_file_location("rustgears_b200._serving_again", serving.__file__)
    with pytest.raises(ImportError, match="built for torch"):
        spec.loader.exec_module(importlib.util.module_from_spec(spec))
