"""build.py: what it builds, and when again.  The compilers are fakes that write their outputs."""
import importlib.util
import os
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hy-nomas-rs_b200")


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py with its outputs under tmp_path; .ran lists the outputs that a compiler wrote."""
    spec = importlib.util.spec_from_file_location("nkv_build_under_test", os.path.join(PKG, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    monkeypatch.setattr(mod, "BUILD", str(tmp_path / "_build"))
    monkeypatch.setattr(mod, "LIB", str(tmp_path / "libnomas_kv.so"))
    monkeypatch.setattr(mod, "BINDING", str(tmp_path / "_block_binding.so"))
    mod.ran, mod.refuse = [], lambda cmd: None

    def run(cmd, **kw):
        bad = mod.refuse(cmd)
        if isinstance(bad, Exception):
            raise bad
        if bad:
            return subprocess.CompletedProcess(cmd, 1, "", bad)
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write(" ".join(cmd))
        mod.ran.append(os.path.basename(out))
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(mod.subprocess, "run", run)
    return mod


def _is_binding(cmd):
    return cmd[-1] == "-lc10"


def test_builds_once(build):
    build.build()
    assert {"libnomas_kv.so", "_block_binding.so", "kernels_packed.cu.o"} <= set(build.ran)
    build.ran.clear()
    build.build()
    assert build.ran == []


@pytest.mark.parametrize("bad", ["no Python.h", FileNotFoundError("g++")])
def test_the_c_library_does_not_wait_for_the_binding(build, bad):
    """Where the extension cannot be compiled, the library is linked all the same, and the error says what is missing."""
    build.refuse = lambda cmd: bad if _is_binding(cmd) else None
    with pytest.raises(RuntimeError, match="binding"):
        build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.BINDING)


def test_without_torch_there_is_the_c_library(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.BINDING)
    assert "not built" in capsys.readouterr().err
