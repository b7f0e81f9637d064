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
