"""What is built and imported without a torch that has CUDA, and without the native half of the Python package."""
import os
import shutil
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "o1.c_b200")


def python(code, **env):
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], cwd=ROOT, env={**os.environ, **env}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout + r.stderr


@pytest.mark.parametrize("torch", ["none", "without CUDA"])
def test_the_library_is_built_without_the_binding(tmp_path, torch):
    """No torch, or one without CUDA: the library is built all the same, and the message says what is not."""
    os.makedirs(tmp_path / "torch" / "lib")
    out = python(f"""
        import importlib.util, os, sys, types
        if {torch == "none"}:
            sys.modules["torch"] = None
        else:
            sys.modules["torch"] = types.SimpleNamespace(__file__={str(tmp_path / "torch" / "__init__.py")!r}, __version__="9.9+cpu", _C=types.SimpleNamespace(_GLIBCXX_USE_CXX11_ABI=True))
        spec = importlib.util.spec_from_file_location("b", os.path.join("o1.c_b200", "build.py"))
        b = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(b)
        b.BINDING = {str(tmp_path / "_binding.so")!r}
        assert b.build() == b.LIB and os.path.exists(b.LIB) and not os.path.exists(b.BINDING)
        """)
    assert "_binding.so is not built" in out and ("no torch" if torch == "none" else "without CUDA") in out


def test_the_package_is_imported_without_the_binding(tmp_path):
    """All of it but the calls that need the binding, which say so."""
    for f in os.listdir(PKG):
        if f.endswith(".py"):
            shutil.copy(os.path.join(PKG, f), tmp_path / f)
    os.symlink(os.path.join(PKG, "libo1b200.so"), tmp_path / "libo1b200.so")
    python(f"""
        import importlib.util, sys
        spec = importlib.util.spec_from_file_location("p", {str(tmp_path / "__init__.py")!r}, submodule_search_locations=[{str(tmp_path)!r}])
        p = sys.modules["p"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(p)
        assert p.Engine and p.Weights and p.lib.o1_kv_attention_workspace_bytes(32, 8) > 0
        for name in ("KvCache", "Decoder", "residual_norm"):
            try:
                getattr(p, name)
            except ImportError as e:
                assert "_binding.so is missing" in str(e)
            else:
                raise SystemExit(name)
        """)


def test_a_binding_of_another_torch_is_refused():
    python("""
        import torch
        from __graft_entry__ import load_package
        p = load_package()
        torch.__version__ = "1.2.3"
        try:
            p.KvCache
        except ImportError as e:
            assert "is of torch" in str(e) and "build.py" in str(e)
        else:
            raise SystemExit("imported")
        """)
