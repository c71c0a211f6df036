"""What the build makes where parts of the tool chain are missing, with the compilers' runs faked."""
import os
import sysconfig

import pytest

from grouped_gemm_gpu_kernel_b200 import build as gbuild


class Compilers:
    """Stands in for build._run: a run makes its output, and compiling the module needs Python.h."""

    def __init__(self, monkeypatch, tmp_path, headers=True, cxx=True):
        self.include = tmp_path / "include"
        self.include.mkdir()
        if headers:
            (self.include / "Python.h").write_text("")
        self.nvcc, self.cxx, self.broken = 0, 0, False
        self.lib, self.module = str(tmp_path / "lib.so"), str(tmp_path / "_moe_native.so")
        monkeypatch.setattr(gbuild, "LIB_PATH", self.lib)
        monkeypatch.setattr(gbuild, "CALLS_PATH", self.module)
        monkeypatch.setattr(gbuild, "BUILD_DIR", str(tmp_path / "build"))
        monkeypatch.setattr(gbuild, "nvcc", lambda: "nvcc")
        monkeypatch.setattr(gbuild.shutil, "which", lambda name: f"/usr/bin/{name}" if cxx else None)
        paths = dict(sysconfig.get_paths(), include=str(self.include))
        monkeypatch.setattr(gbuild.sysconfig, "get_paths", lambda: paths)
        monkeypatch.setattr(gbuild, "_run", self.run)
        self.has_cxx = cxx

    def run(self, cmd, verbose):
        if cmd[0] == "nvcc":
            self.nvcc += 1
        else:
            self.cxx += 1
            if not self.has_cxx or self.broken or not (self.include / "Python.h").exists():
                raise RuntimeError("command failed")
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass
        return type("Done", (), {"stderr": "", "stdout": ""})()


def test_everything_is_made_once(monkeypatch, tmp_path):
    c = Compilers(monkeypatch, tmp_path)
    assert gbuild.build() == c.lib
    assert os.path.exists(c.lib) and os.path.exists(c.module)
    runs = c.nvcc
    assert runs == len(gbuild.SOURCES) + 1 and c.cxx == 1
    gbuild.build()
    assert c.nvcc == runs and c.cxx == 1
    os.remove(c.module)
    gbuild.build()  # the module alone
    assert c.nvcc == runs and c.cxx == 2 and os.path.exists(c.module)


@pytest.mark.parametrize("missing", ["headers", "cxx"])
def test_the_library_is_made_without_python_headers_or_a_host_compiler(monkeypatch, tmp_path, missing):
    c = Compilers(monkeypatch, tmp_path, **{missing: False})
    with pytest.warns(UserWarning, match="_moe_native"):
        assert gbuild.build() == c.lib
    assert os.path.exists(c.lib) and not os.path.exists(c.module)
    runs = c.nvcc
    with pytest.warns(UserWarning):
        gbuild.build()  # and stays as it is
    assert c.nvcc == runs


def test_a_module_of_older_sources_does_not_stay(monkeypatch, tmp_path):
    """Where it cannot be made again, a module older than its sources goes: it would call another library."""
    c = Compilers(monkeypatch, tmp_path, headers=False)
    with open(c.module, "w"):
        pass
    os.utime(c.module, (1, 1))
    with pytest.warns(UserWarning):
        gbuild.build()
    assert not os.path.exists(c.module)


def test_an_error_in_the_module_is_raised(monkeypatch, tmp_path):
    c = Compilers(monkeypatch, tmp_path)
    c.broken = True
    with pytest.raises(RuntimeError):
        gbuild.build()


def test_the_module_carries_its_python():
    """Named for the interpreter that it was made with, so that another one beside it makes its own and
    never loads this."""
    assert os.path.basename(gbuild.CALLS_PATH) == "_moe_native" + sysconfig.get_config_var("EXT_SUFFIX")
    assert sysconfig.get_config_var("SOABI") in gbuild.CALLS_PATH
