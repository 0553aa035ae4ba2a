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
