"""The in-tree build's decisions (nothing is compiled here)."""

import sys

import pytest

from hcp_vllm_plugin_b200 import build as B


@pytest.fixture
def compiled(monkeypatch, tmp_path):
    """What would have been compiled; artefacts go to a folder of their own."""
    calls = []

    def compile_(cmd, target, verbose):
        calls.append(target)
        marks = [c.split("=", 1)[1].strip('"') for c in cmd if c.startswith("-DHCP_BUILT_FOR=")]
        open(target, "wb").write(b"\0" + "".join(marks).encode() + b"\0")

    monkeypatch.setattr(B, "_compile", compile_)
    monkeypatch.setattr(B, "LIB", str(tmp_path / "libhcp_ring.so"))
    monkeypatch.setattr(B, "FRONT", str(tmp_path / "_hcp_front.so"))
    return calls


def test_the_library_is_built_without_torch(compiled, monkeypatch, capsys):
    """The C library needs no torch: without it the library is built and the torch front end left out."""
    monkeypatch.setitem(sys.modules, "torch", None)
    assert B.build(force=True) == B.LIB
    assert compiled == [B.LIB]
    assert "_hcp_front.so" in capsys.readouterr().err


def test_the_front_end_is_built_anew_for_another_torch(compiled, monkeypatch):
    """Times of files do not tell which torch and Python a module was built for."""
    import os

    import torch
    B.build_front()
    assert compiled == [B.FRONT]
    later = os.path.getmtime(B.FRONT_SOURCE) + 1e6
    os.utime(B.FRONT, (later, later))
    B.build_front()
    assert compiled == [B.FRONT]               # up to date
    monkeypatch.setattr(torch, "__version__", "0.0.1+other")
    B.build_front()
    assert compiled == [B.FRONT] * 2           # not for this torch
    B.build_front()
    assert compiled == [B.FRONT] * 2


def test_a_front_end_built_for_another_torch_is_refused(monkeypatch):
    from hcp_vllm_plugin_b200 import _capi
    _capi.front()
    monkeypatch.setattr(_capi, "_front", None)
    monkeypatch.setattr(B, "front_target", lambda: "torch 0.0.1, another Python")
    with pytest.raises(_capi.HcpError, match="built for torch"):
        _capi.front()


def test_an_installed_package_without_sources_loads_its_modules(tmp_path):
    """Loading asks the build what the module has to be for; that needs no source files."""
    import os
    import shutil
    import subprocess
    home = tmp_path / "hcp_vllm_plugin_b200"
    shutil.copytree(os.path.dirname(B.__file__), home, ignore=shutil.ignore_patterns("csrc", "__pycache__", "*.tmp"))
    r = subprocess.run([sys.executable, "-c", "from hcp_vllm_plugin_b200 import _capi; print(_capi.front().__name__)"],
                       cwd=tmp_path, env={**os.environ, "PYTHONPATH": str(tmp_path)}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "_hcp_front" in r.stdout, r.stderr[-800:]
