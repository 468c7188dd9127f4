"""build.py: the library needs no torch, so nothing that the operators' compiled entry lacks keeps it from
being built."""

import types

import pytest
import torch

import build as B


@pytest.fixture
def steps(monkeypatch, tmp_path):
    """Compilers that only write their output file; returns the outputs in order. `steps.fail`: names that fail."""
    made = types.SimpleNamespace(order=[], fail=())

    def run(cmd, **kw):
        from pathlib import Path

        out = Path(cmd[cmd.index("-o") + 1])
        made.order.append(out.name.split(".")[0])
        if made.order[-1] in made.fail:
            return types.SimpleNamespace(returncode=1, stdout="", stderr="no such library\n")
        out.write_bytes(b"")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(B.subprocess, "run", run)
    monkeypatch.setattr(B, "OUT", tmp_path / "libkvs_b200.so")
    monkeypatch.setattr(B, "fastcall_path", lambda: tmp_path / "_fastcall.so")
    monkeypatch.setattr(B, "opcall_path", lambda: tmp_path / "_opcall.so")
    return made


def test_all_parts_are_built(steps):
    B.build()
    assert sorted(steps.order) == ["_fastcall", "_opcall", "libkvs_b200"] and B.OUT.exists() and B.opcall_path().exists()


def test_library_is_built_where_the_compiled_entry_is_not(steps):
    steps.fail = ("_opcall",)
    with pytest.raises(RuntimeError, match="_opcall"):
        B.build()
    assert B.OUT.exists()


@pytest.mark.parametrize("lacks", ["version", "library"])
def test_torch_without_cuda_has_no_compiled_entry(steps, monkeypatch, tmp_path, lacks):
    if lacks == "version":
        monkeypatch.setattr(torch.version, "cuda", None)
    else:
        monkeypatch.setattr(torch, "__file__", str(tmp_path / "__init__.py"))
    B.build()
    assert steps.order and "_opcall" not in steps.order and B.OUT.exists() and not B.opcall_path().exists()
