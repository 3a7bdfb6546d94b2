"""CPU: the kernel sources behind yolov5m_amd/act8.py and group_norm.py executed lane by lane (tests/emu) by the functions of
tests/test_gpu_act8.py and tests/test_gpu_group_norm.py; and the package's refusal of host tensors without the executor."""
import importlib
import inspect
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
from emu.run_gpu_tests import expand  # noqa: E402

have_clang = os.path.exists(os.environ.get("Y5M_EMU_CXX", "/opt/rocm/lib/llvm/bin/clang++"))


def _collect():
    items = []
    for modname in ("test_gpu_act8", "test_gpu_group_norm"):
        mod = importlib.import_module(modname)
        for name in sorted(n for n in dir(mod) if n.startswith("test_")):
            for i, kw in enumerate(expand(getattr(mod, name))):
                items.append(pytest.param(modname, name, kw, id=f"{modname[9:]}::{name[5:]}[{i}]"))
    return items


@pytest.mark.skipif(torch.cuda.is_available(), reason="CPU-only check")
def test_host_tensors_are_refused():
    from yolov5m_amd import GroupNormAct, act8_store, group_norm_act
    from yolov5m_amd._lib import Y5MError
    x = torch.zeros(1, 2, 2, 16).movedim(-1, 1)
    for call in (lambda: act8_store(x), lambda: group_norm_act(x, 4), lambda: GroupNormAct(4, 16)(x)):
        with pytest.raises(Y5MError, match="no CPU fallback"):
            call()


@pytest.fixture(scope="module")
def emu():
    from emu.harness import emulated
    with emulated() as L:
        yield L


@pytest.mark.skipif(not have_clang, reason="host clang of the ROCm image not present")
@pytest.mark.parametrize("modname,name,kw", _collect())
def test_on_cpu_executor(emu, monkeypatch, modname, name, kw):
    for m in ("test_gpu_act8", "test_gpu_group_norm"):
        monkeypatch.setattr(importlib.import_module(m), "DEV", "cpu")
    fn = getattr(importlib.import_module(modname), name)
    if "monkeypatch" in inspect.signature(fn).parameters:
        kw = dict(kw, monkeypatch=monkeypatch)
    fn(**kw)
