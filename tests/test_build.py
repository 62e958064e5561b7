"""What the build needs and which binding is loaded.  No GPU, and nothing is compiled."""
import importlib.util
import os

import pytest
import torch

from k2b import _native


def load():
    package = os.path.dirname(os.path.dirname(os.path.abspath(_native.__file__)))
    spec = importlib.util.spec_from_file_location("_k2b_build_test", os.path.join(package, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_binding_of_another_environment_is_not_taken(monkeypatch):
    """Another torch, Python or C++ ABI has a file of its own."""
    build = load()
    here = _native.bind_path()
    assert build.bind_path() == here
    names = {here}
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    names.add(_native.bind_path())
    assert not build.bind_up_to_date()
    import sysconfig

    monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "cpython-00")
    names.add(_native.bind_path())
    assert len(names) == 3 and all(os.path.dirname(n) == os.path.dirname(_native.LIB_PATH) for n in names)


def test_bind_builds_and_loads_the_file_of_this_environment(monkeypatch):
    """A missing file is built, by the function that builds it alone."""
    asked = []
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    monkeypatch.setattr(_native, "_bind", None)
    monkeypatch.setattr(_native, "lib", lambda: None)
    monkeypatch.setattr(_native, "_build", lambda what, path: asked.append((what, path)))
    with pytest.raises(ImportError):  # nothing was built
        _native.bind()
    assert asked == [("build_bind", _native.bind_path())]


def test_library_is_built_alone(monkeypatch):
    asked = []

    def stop(what, path):
        asked.append(what)
        raise _native.K2BError("stop")

    monkeypatch.setattr(_native, "_lib", None)
    monkeypatch.setattr(_native, "LIB_PATH", os.path.join(os.sep, "nonexistent", "libk2b.so"))
    monkeypatch.setattr(_native, "_build", stop)
    with pytest.raises(_native.K2BError):
        _native.lib()
    assert asked == ["build_lib"]


@pytest.mark.parametrize("missing", ["torch", "headers", "compiler"])
def test_build_without_the_bindings_needs(monkeypatch, capsys, missing):
    """A host without torch, Python's headers or g++ still builds libk2b."""
    build = load()
    done = []
    monkeypatch.setattr(build, "build_lib", lambda *a: done.append("lib"))
    monkeypatch.setattr(build, "build_bind", lambda *a: done.append("bind"))
    if missing == "torch":
        find = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    elif missing == "headers":
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": os.path.join(os.sep, "nonexistent")})
    else:
        which = build.shutil.which
        monkeypatch.setattr(build.shutil, "which", lambda name: None if name == "g++" else which(name))
    assert build.build() == build.OUT
    assert done == ["lib"] and "binding not built" in capsys.readouterr().err


def test_cuda_headers_of_a_bare_compiler_name(monkeypatch, tmp_path):
    """NVCC=nvcc is looked up, so that the headers beside it are found."""
    (tmp_path / "bin").mkdir()
    tool = tmp_path / "bin" / "nvcc"
    tool.write_text("#!/bin/sh\n")
    tool.chmod(0o755)
    monkeypatch.setenv("PATH", f"{tool.parent}{os.pathsep}{os.environ['PATH']}")
    monkeypatch.setenv("NVCC", "nvcc")
    build = load()
    assert build.NVCC == str(tool) and build.CUDA_INCLUDE == str(tmp_path / "include")
