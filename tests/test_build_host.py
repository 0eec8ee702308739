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


@pytest.mark.parametrize("change", ["torch", "python", "compiler"])
def test_the_binding_is_compiled_anew_for_another_torch_or_python(build, monkeypatch, change):
    import importlib.metadata
    build.build()
    build.ran.clear()
    if change == "torch":
        real = importlib.metadata.version
        monkeypatch.setattr(importlib.metadata, "version", lambda n: "0.0.0+other" if n == "torch" else real(n))
    elif change == "python":
        monkeypatch.setattr(sys, "version", "3.99 (another)")
    else:
        monkeypatch.setenv("CXX", "another-c++")
    build.build()
    assert build.ran == ["_block_binding.so"]
    build.ran.clear()
    build.build()
    assert build.ran == []


def test_torch_without_package_metadata(build, monkeypatch):
    """A source build on the path: its version file stands for the version."""
    import importlib.metadata

    def version(name):
        raise importlib.metadata.PackageNotFoundError(name)

    monkeypatch.setattr(importlib.metadata, "version", version)
    build.build()
    assert os.path.exists(build.BINDING)
    build.ran.clear()
    build.build()
    assert build.ran == []


def test_a_folder_named_torch_is_not_torch(build, monkeypatch, tmp_path):
    import importlib.util
    from importlib.machinery import ModuleSpec
    real = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec",
                        lambda n, *a: ModuleSpec(n, None, is_package=True) if n == "torch" else real(n, *a))
    build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.BINDING)


def test_a_stale_binding_does_not_outlive_a_failed_compile(build, monkeypatch):
    build.build()
    monkeypatch.setattr(sys, "version", "3.99 (another)")
    build.refuse = lambda cmd: "no" if _is_binding(cmd) else None
    with pytest.raises(RuntimeError):
        build.build()
    assert not os.path.exists(build.BINDING)


def test_a_failed_compile_is_tried_again(build):
    build.refuse = lambda cmd: "no" if _is_binding(cmd) else None
    for _ in range(2):
        with pytest.raises(RuntimeError):
            build.build()
    build.refuse = lambda cmd: None
    build.ran.clear()
    build.build()
    assert build.ran == ["_block_binding.so"]


def test_clean_builds_everything_again(build):
    build.build()
    first = sorted(build.ran)
    build.ran.clear()
    build.build(clean=True)
    assert sorted(build.ran) == first
