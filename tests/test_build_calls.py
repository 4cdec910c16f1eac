"""The native calls of mtpx.ops are built where their headers are; elsewhere the
library's build is whole without them, and says so."""
import importlib.util
import os
import sysconfig
from types import SimpleNamespace

import pytest
import torch

from mtpx import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(monkeypatch, tmp_path):
    spec = importlib.util.spec_from_file_location("mtpx_build", os.path.join(ROOT, "imr-mlp_amd", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "CALLS", str(tmp_path / "_calls.so"))
    return module


def test_without_pythons_headers(build, monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    build.build_calls()
    assert not os.path.exists(build.CALLS) and "Python.h" in capsys.readouterr().out


def test_without_torchs_headers(build, monkeypatch, tmp_path, capsys):
    class Spec:
        submodule_search_locations = [str(tmp_path)]

    monkeypatch.setattr(importlib.util, "find_spec", lambda name: Spec)
    build.build_calls()
    assert not os.path.exists(build.CALLS) and "ATen.h" in capsys.readouterr().out


def test_without_torch(build, monkeypatch, capsys):
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: None)
    build.build_calls()
    assert not os.path.exists(build.CALLS) and capsys.readouterr().out == ""


def test_a_compiler_that_fails_raises(build, monkeypatch):
    monkeypatch.setattr(build, "CXX", "false")
    with pytest.raises(Exception):
        build.build_calls()


def test_recording_without_the_native_calls(monkeypatch):
    """The earlier operators' gradients do not need them."""
    def missing():
        raise RuntimeError("not built")

    monkeypatch.setattr(ops, "_calls", missing)
    monkeypatch.setattr(ops, "_stream", lambda ctx: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    end = SimpleNamespace(metadata={}, variable=SimpleNamespace(is_cuda=True))
    monkeypatch.setattr(ops, "_Leaf", type(end))
    ops._same_streams(SimpleNamespace(ctx=None, next_functions=((end, 0),)))
