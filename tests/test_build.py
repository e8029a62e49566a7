"""The build recipe where torch, or the Python headers, are missing: everything but the PyTorch binding is
built, as C, C++ and ctypes users need it."""
import importlib.util
import sysconfig

import pytest

import __graft_entry__
from grouped_gemm_gpu_kernel_amd import build

OTHERS = ["build_library", "build_oracle", "build_cpp_tests", "build_bench_driver", "build_vendor_baseline"]


@pytest.fixture
def made(monkeypatch):
    """The steps that were run; none of them compiles anything."""
    steps = []
    for name in OTHERS:
        monkeypatch.setattr(build, name, lambda name=name: steps.append(name))
    monkeypatch.setattr(build, "_run", lambda *a, **k: pytest.fail(f"compiles {a}"))
    return steps


@pytest.fixture(params=["torch", "headers"])
def missing(request, monkeypatch, tmp_path):
    if request.param == "torch":
        found = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else found(name, *a))
    else:
        paths = {**sysconfig.get_paths(), "include": str(tmp_path)}
        monkeypatch.setattr(sysconfig, "get_paths", lambda *a, **k: paths)
    return request.param


def test_everything_else_is_built(made, missing, capsys):
    assert build.main([]) == 0
    assert made == OTHERS
    made.clear()
    __graft_entry__.build()
    assert made == OTHERS
    out = capsys.readouterr().out
    assert out.count("gg_torch.so is not built") == 2
    assert ("torch is not installed" if missing == "torch" else "no Python.h") in out


def test_no_torch_asks_for_nothing(made, missing, capsys):
    assert build.main(["--no-torch"]) == 0
    assert made == OTHERS and "gg_torch.so" not in capsys.readouterr().out
    made.clear()
    assert build.main(["--no-torch", "--no-oracle", "--no-tests"]) == 0
    assert made == [s for s in OTHERS if s not in ("build_oracle", "build_cpp_tests")]


def test_here_both_are_there():
    assert build.torch_binding_lacks() is None
