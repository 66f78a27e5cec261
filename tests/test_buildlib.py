"""buildlib.build(): the library alone where torch or a compiler is missing, and when _serving.so is compiled anew."""
import os
import subprocess
import sys

import pytest

from tmac_zynq_fpga_b200 import buildlib


@pytest.fixture
def fresh(monkeypatch, tmp_path):
    """A package folder without _serving.so, whose library is built; the commands that are run."""
    ran = []

    def run(cmd, check):
        ran.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("module")

    monkeypatch.setattr(buildlib, "build_library", lambda *a, **k: buildlib.OUT)
    monkeypatch.setattr(buildlib, "BINDING_OUT", str(tmp_path / "_serving.so"))
    monkeypatch.setattr(buildlib, "HERE", str(tmp_path))
    os.makedirs(tmp_path.parent / "include", exist_ok=True)
    (tmp_path.parent / "include" / "tmac_cuda.h").write_text("")
    monkeypatch.setattr(subprocess, "run", run)
    return ran


def test_the_library_is_built_without_torch(fresh, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert buildlib.build() == buildlib.OUT
    assert not fresh and "torch is not installed" in capsys.readouterr().err


def test_the_library_is_built_without_cuda_in_torch(fresh, monkeypatch, capsys):
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch.version, "cuda", None)
    assert buildlib.build() == buildlib.OUT
    assert not fresh and "without CUDA" in capsys.readouterr().err


def test_the_library_is_built_without_a_compiler(fresh, monkeypatch, capsys):
    pytest.importorskip("torch")
    monkeypatch.setattr(buildlib, "CXX", "no-such-compiler")
    assert buildlib.build() == buildlib.OUT
    assert not fresh and "no-such-compiler" in capsys.readouterr().err


def test_a_compiler_error_is_raised(fresh, monkeypatch):
    pytest.importorskip("torch")
    monkeypatch.setattr(subprocess, "run", lambda cmd, check: (_ for _ in ()).throw(subprocess.CalledProcessError(1, cmd)))
    with pytest.raises(subprocess.CalledProcessError):
        buildlib.build()


def test_the_module_is_compiled_once_for_a_torch_and_anew_for_another(fresh, monkeypatch):
    torch = pytest.importorskip("torch")
    buildlib.build()
    buildlib.build()
    assert len(fresh) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.0+other")
    buildlib.build()
    buildlib.build()
    assert len(fresh) == 2


def test_operators_without_the_module_say_so():
    """A process in which _serving cannot be imported: the package works, its operators raise TmacError."""
    pytest.importorskip("torch")
    code = ("import sys, torch; sys.modules['tmac_zynq_fpga_b200._serving'] = None; import tmac_zynq_fpga_b200 as tm; tm.lib()\n"
            "try: tm.sample(torch.zeros(2, 10), torch.zeros(2))\nexcept tm.TmacError as e: assert 'build' in str(e); print('refused')")
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(buildlib.HERE), capture_output=True, text=True)
    assert r.stdout == "refused\n", r.stderr
