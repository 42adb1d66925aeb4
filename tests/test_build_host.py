"""The build of the torch binding: what makes it stale, compilers of either kind, and builds without torch."""
import importlib.util
import os
import stat
import sys
import sysconfig

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "morph-orchestrates-recursive-pruned-hierarchies_b200")


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py with its outputs under a temporary folder and a compiler that only writes down how it was called."""
    spec = importlib.util.spec_from_file_location("_build_under_test", os.path.join(PKG, "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "NATIVE", str(tmp_path / "_mortar_native.so"))
    monkeypatch.setattr(module, "OBJ", str(tmp_path))
    log = tmp_path / "calls"

    def compiler(rejects=""):
        path = tmp_path / "cxx"
        path.write_text(f"""#!/bin/sh
out=
for a in "$@"; do
  [ "$a" = "{rejects or 'none'}" ] && {{ echo "unrecognized option $a" >&2; exit 1; }}
  [ "$last" = -o ] && out="$a"
  last="$a"
done
case "$*" in *torch_binding.cpp*) echo "$@" >> {log}; : > "$out";; esac
""")
        path.chmod(path.stat().st_mode | stat.S_IXUSR)
        monkeypatch.setenv("CXX", str(path))
    compiler()
    module.calls = lambda: log.read_text().splitlines() if log.exists() else []
    module.compiler = compiler
    return module


def test_binding_is_built_again_when_what_it_was_built_with_changes(build, monkeypatch):
    assert build.build_binding() == build.NATIVE and len(build.calls()) == 1
    build.build_binding()
    assert len(build.calls()) == 1                                   # nothing changed
    build.build_binding(force=True)
    assert len(build.calls()) == 2
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    build.build_binding()
    assert len(build.calls()) == 3
    real = sysconfig.get_config_var
    monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "other" if name == "SOABI" else real(name))
    build.build_binding()
    build.build_binding()
    assert len(build.calls()) == 4
    monkeypatch.setattr(build, "BINDING_FLAGS", [*build.BINDING_FLAGS, "-DOTHER"])
    build.build_binding()
    build.build_binding()
    assert len(build.calls()) == 5
    os.remove(build.NATIVE)
    build.build_binding()
    assert len(build.calls()) == 6


def test_binding_builds_with_a_compiler_that_lacks_a_flag(build):
    build.build_binding()
    build.compiler(rejects="-nostdlib++")
    build.build_binding(force=True)
    first, second = build.calls()
    assert "-nostdlib++" in first and "-nostdlib++" not in second and "-l:libstdc++.so.6" in second


def test_library_builds_where_there_is_no_torch(build, monkeypatch, capsys):
    """A user of the C ABI needs neither torch nor Python's headers: the binding is left out with a message."""
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build_binding() is None
    assert "torch" in capsys.readouterr().err
    monkeypatch.undo()


def test_library_builds_where_python_has_no_headers(build, monkeypatch, tmp_path, capsys):
    real = sysconfig.get_paths
    monkeypatch.setattr(sysconfig, "get_paths", lambda *a, **k: {**real(*a, **k), "include": str(tmp_path / "nowhere")})
    assert build.build_binding() is None and not build.calls()
    assert "Python.h" in capsys.readouterr().err


def test_a_failing_compiler_is_an_error(build):
    build.compiler(rejects="-shared")
    with pytest.raises(RuntimeError, match="failed"):
        build.build_binding()
    build.compiler()
    build.build_binding()
    assert len(build.calls()) == 1                                   # the failure left no record of a build
