"""CPU tests of how the C++-registered torch ops are found: a libq3torch.so that is missing or cannot be loaded costs its own ops and
nothing else, neither at import nor in the build."""
import importlib.util
import os
import shutil
import subprocess
import sys

import pytest
from conftest import PKG

import q3attn
from q3attn import _lib

HEAD = """
import shutil, sys
sys.path.insert(0, {where!r})
import torch
import q3attn
def call(device='cpu'):
    return torch.ops.q3attn.paged_read_fp8(*q3attn.fp8_cache(2, device=device), torch.zeros(3, dtype=torch.int64, device=device))
def refused(*words):
    try:
        q3attn.paged_read_fp8(*q3attn.fp8_cache(2, device='cpu'), torch.zeros(3, dtype=torch.int64))
    except RuntimeError as e:
        assert all(w in str(e) for w in words), e
    else:
        raise AssertionError('not refused')
"""


def _run(where, code):
    """code in a process of its own, with the package from ``where``."""
    r = subprocess.run([sys.executable, "-c", HEAD.format(where=str(where)) + code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


@pytest.fixture
def package(tmp_path):
    """A copy of the package, its libraries among it."""
    q3attn.lib()
    shutil.copytree(os.path.join(PKG, "q3attn"), tmp_path / "q3attn", ignore=shutil.ignore_patterns("__pycache__"))
    return tmp_path


def test_a_binding_that_cannot_be_loaded(package):
    (package / "q3attn" / "libq3torch.so").write_bytes(b"no library")
    _run(package, "q3attn.lib(); q3attn.PagePool; refused('libq3torch.so', 'cannot be loaded')")


def test_a_library_of_another_abi(package):
    at = package / "q3attn" / "_lib.py"
    at.write_text(at.read_text().replace(f"ABI_VERSION = {_lib.ABI_VERSION}", f"ABI_VERSION = {_lib.ABI_VERSION + 1}"))
    _run(package, "refused('ABI', 'rebuild')")


def test_built_after_the_import(package):
    away = package / "away"
    away.mkdir()
    for name in ("libq3attn.so", "libq3torch.so"):
        shutil.move(package / "q3attn" / name, away / name)
    _run(package, f"""
refused('not found')
for name in ('libq3attn.so', 'libq3torch.so'):
    shutil.copy({str(away)!r} + '/' + name, {str(package / "q3attn")!r} + '/' + name)
refused('must be on a GPU')
k, v = call('meta')
assert k.shape == v.shape == (3, 8, 128) and k.dtype == torch.bfloat16
""")


def _build_module(tmp_path, monkeypatch):
    """build.py with its outputs under tmp_path, the HIP compiler's part left out."""
    spec = importlib.util.spec_from_file_location("q3attn_build_under_test", os.path.join(PKG, "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    for name, file in (("OUT", "libq3attn.so"), ("PROBE_OUT", "libq3probe.so"), ("TORCH_OUT", "libq3torch.so"), ("BUILD", "_build")):
        monkeypatch.setattr(b, name, str(tmp_path / file))
    monkeypatch.setattr(b, "_compile", lambda src: src + ".o")
    run = b._run

    def link_only(cmd, what):
        if what != "link":
            return run(cmd, what)
        with open(cmd[-1], "w") as f:
            f.write("linked")

    monkeypatch.setattr(b, "_run", link_only)
    return b


def test_a_build_without_a_host_compiler_keeps_the_hip_libraries(tmp_path, monkeypatch):
    b = _build_module(tmp_path, monkeypatch)
    (tmp_path / "libq3torch.so").write_text("of an earlier build")
    monkeypatch.setattr(b, "CXX", str(tmp_path / "no-compiler"))
    with pytest.raises(RuntimeError, match="no-compiler"):
        b.build()
    assert (tmp_path / "libq3attn.so").read_text() == (tmp_path / "libq3probe.so").read_text() == "linked"
    assert not (tmp_path / "libq3torch.so").exists()
