"""The build of the library and of the module of Python calls beside it: one does not take the other along, and a module
built for another torch is not used."""

from __future__ import annotations

import pytest
import torch

import build
from minisgl_amd.kernel import lib


def test_the_library_is_built_without_the_module(monkeypatch, tmp_path):
    linked = []

    def fails():
        raise RuntimeError("no torch headers")

    monkeypatch.setattr(build, "BUILD", str(tmp_path))
    monkeypatch.setattr(build, "_build_binding", fails)
    monkeypatch.setattr(build, "_compile", lambda src: src)
    monkeypatch.setattr(build, "_link", lambda objs, out: linked.append(out))
    with pytest.raises(RuntimeError, match="no torch headers"):
        build.build(verbose=False)
    assert linked == [build.OUT, build.PEAKS_OUT]


def test_the_module_needs_no_compiler_of_its_own(monkeypatch, tmp_path):
    ran = []

    class Done:
        returncode, stderr = 1, "stopped"

    monkeypatch.setattr(build, "BINDING_OUT", str(tmp_path / "_mla_torch.so"))
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: ran.append(cmd[0]) or Done)
    with pytest.raises(RuntimeError, match="stopped"):
        build._build_binding()
    assert ran == [build.HIPCC]


def test_a_module_of_another_torch_is_refused(monkeypatch):
    assert lib.load_binding.__wrapped__().built_for.startswith(f"torch {torch.__version__}, Python 3.")
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    with pytest.raises(lib.MLAKernelError, match="was built for torch .*, this is torch 0.0.1"):
        lib.load_binding.__wrapped__()
