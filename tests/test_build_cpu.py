"""What build_native builds and when, with the compilers replaced by a fake that writes down its calls."""
import subprocess
from pathlib import Path

import pytest

import build_native


@pytest.fixture
def fake(monkeypatch, tmp_path):
    """Builds into tmp_path; `fake.fails` names the compilers that fail."""
    class Fake:
        fails, calls = (), []

        def run(self, cmd, check=True):
            name = Path(cmd[0]).name
            self.calls.append((name, Path(cmd[cmd.index("-o") + 1]).name.removesuffix(".tmp")))
            if name in self.fails:
                raise subprocess.CalledProcessError(1, cmd)
            Path(cmd[cmd.index("-o") + 1]).write_text("built")

        def built(self):
            out, self.calls = {n for _, n in self.calls if n.endswith(".so")}, []
            return out

    f = Fake()
    f.calls = []
    monkeypatch.setattr(build_native.subprocess, "run", f.run)
    monkeypatch.setattr(build_native, "HERE", tmp_path)
    monkeypatch.setattr(build_native, "LIB", tmp_path / "libw4a8.so")
    monkeypatch.setattr(build_native, "BINDING", tmp_path / "_w4a8_torch.so")
    return f


def test_the_library_does_not_need_the_torch_module(fake):
    """It is linked where the torch module cannot be compiled, which is an error of its own."""
    fake.fails = ("g++",)
    with pytest.raises(RuntimeError, match="libw4a8.so is built.*_w4a8_torch"):
        build_native.build()
    assert build_native.LIB.exists() and not build_native.BINDING.exists()
    fake.built()
    assert build_native.build(torch_module=False) == build_native.LIB and not fake.built()  # nothing to do
    fake.fails = ()
    assert build_native.build() == build_native.LIB
    assert fake.built() == {"_w4a8_torch.so"}  # what was missing


def test_a_library_that_fails_is_reported_as_itself(fake):
    fake.fails = ("nvcc",)
    with pytest.raises(subprocess.CalledProcessError):
        build_native.build()
    assert not build_native.LIB.exists()


def test_another_torch_or_python_rebuilds_the_module(fake, monkeypatch):
    """The module fits one version of each; file times do not show that."""
    build_native.build()
    assert fake.built() == {"libw4a8.so", "_w4a8_torch.so"}
    build_native.build()
    assert fake.built() == set()
    import torch

    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "99.0")
        build_native.build()
        assert fake.built() == {"_w4a8_torch.so"}
        build_native.build()
        assert fake.built() == set()
    build_native.build()
    assert fake.built() == {"_w4a8_torch.so"}
    monkeypatch.setattr(build_native.sysconfig, "get_config_var", lambda name: "cpython-399")
    build_native.build()
    assert fake.built() == {"_w4a8_torch.so"}


def test_a_module_that_does_not_fit_is_named_with_its_error(monkeypatch):
    import sys

    import int4_int8_ext as ext

    class Finder:
        def find_spec(self, name, path=None, target=None):
            if name == "_w4a8_torch":
                raise ImportError("undefined symbol: of another torch")

    build_native.build()
    monkeypatch.delitem(sys.modules, "_w4a8_torch", raising=False)
    monkeypatch.setattr(sys, "meta_path", [Finder(), *sys.meta_path])
    with pytest.raises(RuntimeError, match="undefined symbol: of another torch.*build_native.py"):
        ext._load_binding()
