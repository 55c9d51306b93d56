"""CPU: the build recipe where the installed PyTorch has no HIP, where there is none, and where the library of the
PyTorch ops' plain calls does not compile: everything else is built all the same."""
import importlib.machinery
import importlib.util
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def build(monkeypatch, tmp_path):
    spec = importlib.util.spec_from_file_location("build_for_test", ROOT / "voltattn_amd" / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    monkeypatch.setattr(mod, "PKG", tmp_path)
    monkeypatch.setattr(mod, "hipcc", lambda: "/opt/rocm/bin/hipcc")
    return mod


def _no_run(*a, **kw):
    raise AssertionError("nothing is to be compiled")


@pytest.mark.parametrize("found", [False, True])
def test_pytorch_without_hip(build, monkeypatch, tmp_path, found):
    spec = importlib.machinery.ModuleSpec("torch", None, origin=str(tmp_path / "torch" / "__init__.py")) if found else None
    (tmp_path / "torch" / "lib").mkdir(parents=True)
    (tmp_path / "torch" / "lib" / "libc10.so").touch()
    stale = tmp_path / "libvoltattn_torch.so"
    stale.touch()
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: spec)
    monkeypatch.setattr(build, "_run", _no_run)
    assert build.build_torch() is None
    assert not stale.exists()                                # an earlier PyTorch's


def test_the_rest_is_built_first(build, monkeypatch):
    done = []

    def broken():
        raise RuntimeError("no such header")

    monkeypatch.setattr(build, "build_torch", broken)
    for name in ("build_library", "build_oracle", "build_cli"):
        monkeypatch.setattr(build, name, lambda *a, name=name, **kw: done.append(name))
    with pytest.raises(RuntimeError, match="no such header"):
        build.build_all()
    assert done == ["build_library", "build_oracle", "build_cli"]
