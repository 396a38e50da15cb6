"""When the torch binding is compiled again: a change of its sources, of torch or of Python, a missing file."""

import importlib.util
import os
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("gsa_build_test", ROOT / "gated-sparse-attention_b200" / "csrc" / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    compiled = []

    def compile_native():
        compiled.append(1)
        mod.NATIVE.write_bytes(b"built")

    for name in ("NATIVE", "LIB"):
        monkeypatch.setattr(mod, name, tmp_path / (name.lower() + ".so"))
    monkeypatch.setattr(mod, "OBJ_DIR", tmp_path / "obj")
    monkeypatch.setattr(mod, "SOURCES", [])
    monkeypatch.setattr(mod, "_compile_native", compile_native)
    monkeypatch.setattr(mod, "_nvcc", lambda: "nvcc")
    mod.LIB.write_bytes(b"")
    mod.compiled = compiled
    return mod


def test_the_binding_is_built_once(build):
    build.build()
    assert len(build.compiled) == 1
    build.build()
    assert len(build.compiled) == 1
    build.build(force=True)
    assert len(build.compiled) == 2
    build.NATIVE.unlink()
    build.build()
    assert len(build.compiled) == 3
    old = build.NATIVE_SRC.stat().st_mtime - 10
    os.utime(build.NATIVE, (old, old))
    build.build()
    assert len(build.compiled) == 4


@pytest.mark.parametrize("what", ["torch", "python"])
def test_the_binding_follows_torch_and_python(build, monkeypatch, what):
    """Against another torch's or Python's headers a binding of the same sources is another."""
    import sysconfig

    import torch

    build.build()
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    else:
        config = sysconfig.get_config_var
        monkeypatch.setattr(sysconfig, "get_config_var", lambda n: "cpython-399-other" if n == "SOABI" else config(n))
    build.build()
    assert len(build.compiled) == 2
    build.build()
    assert len(build.compiled) == 2


def test_a_failed_build_is_tried_again(build, monkeypatch):
    good = build._compile_native

    def fails():
        raise RuntimeError("g++ failed")

    monkeypatch.setattr(build, "_compile_native", fails)
    with pytest.raises(RuntimeError, match="g.. failed"):
        build.build()
    build.NATIVE.write_bytes(b"left from before")
    monkeypatch.setattr(build, "_compile_native", good)
    build.build()
    assert len(build.compiled) == 1
