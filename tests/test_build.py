"""The build recipe where torch, or the Python headers, are missing: everything but the PyTorch binding is
built, as C, C++ and ctypes users need it.  A binding that was built for another torch is refused."""
import importlib.machinery
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


@pytest.fixture(params=["torch", "folder", "headers"])
def missing(request, monkeypatch, tmp_path):
    if request.param != "headers":
        found = importlib.util.find_spec
        torch = None if request.param == "torch" else importlib.machinery.ModuleSpec("torch", None, is_package=True)
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: torch if name == "torch" else found(name, *a))
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
    assert ("no Python.h" if missing == "headers" else "torch is not installed") in out


def test_no_torch_asks_for_nothing(made, missing, capsys):
    assert build.main(["--no-torch"]) == 0
    assert made == OTHERS and "gg_torch.so" not in capsys.readouterr().out
    made.clear()
    assert build.main(["--no-torch", "--no-oracle", "--no-tests"]) == 0
    assert made == [s for s in OTHERS if s not in ("build_oracle", "build_cpp_tests")]


def test_here_both_are_there():
    assert build.torch_binding_lacks() is None


def test_a_binding_of_another_torch_is_refused(monkeypatch):
    """Built, then torch was exchanged: nothing in the old binary is called."""
    import torch

    from grouped_gemm_gpu_kernel_amd import torch_ops

    assert torch_ops._binding().torch_version == torch.__version__
    monkeypatch.setattr(torch_ops, "_gg_torch", None)
    with monkeypatch.context() as other:
        other.setattr(torch, "__version__", "2.9.1+rocm6.4")
        with pytest.raises(RuntimeError, match="was built for torch .* this is 2.9.1.*build it again"):
            torch_ops.moe_route(torch.zeros(3, 4), 2)
    assert torch_ops._binding() is not None


def test_a_binding_that_does_not_load_says_so(monkeypatch, tmp_path):
    from grouped_gemm_gpu_kernel_amd import _lib, torch_ops

    (tmp_path / "gg_torch.so").write_bytes(b"no library")
    monkeypatch.setattr(torch_ops, "_gg_torch", None)
    monkeypatch.setattr(_lib, "TORCH_PATH", tmp_path / "gg_torch.so")
    with pytest.raises(RuntimeError, match="does not fit this torch.*build it again"):
        torch_ops._binding()
