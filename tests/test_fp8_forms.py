"""Every form of the 8-bit products' kernels that a call can take is run by a call here, against 64 bits.

Which form a call takes is asked of the library on the host (ggk_fp8_form).  The calls of CASES together take every form that any
of a sweep over the sizes takes, and those are all the kernels that are built."""
import ctypes
import itertools
import random

import pytest
import torch

from grouped_gemm_gpu_kernel_amd import _lib, torch_ops
from test_fp8 import (BASE, blocks, check_gated, check_moe, check_moe_gated, check_product, matrix_of, matrix_values, routing, row_values,
                      rows_of)
from test_fp8_workspace import gated_args, multiply, wanted
from test_kernel_resources import _scratch

F32, BF16 = torch.float32, torch.bfloat16


def arguments(rows, k, n, experts=0, fan=1, gate=0, fast=False, out=BF16, workspace=False):
    b, r = blocks, rows * fan
    args = _lib.GGKFp8Args(
        rows=r, x_rows=rows, n=n, k=k, experts=experts, gate=gate, x=0x1000, ldx=k, x_scales=0x1000, ldxs=b(k), w=0x1000, ldw=k,
        stride_w=n * k, w_scales=0x1000, ldws=b(k), stride_ws=b(n) * b(k), y=0x1000, ldy=n, fast=int(fast),
        y_type=_lib.GGK_TYPE_F32 if out == F32 else _lib.GGK_TYPE_BF16, counts=0x1000, order=0x1000)
    if gate:
        args.up, args.ldu, args.stride_u, args.up_scales, args.ldus, args.stride_us = 0x1000, k, n * k, 0x1000, b(k), b(n) * b(k)
        args.y_scales, args.ldys = 0x1000, b(n)
        if workspace:
            args.workspace, args.workspace_floats = 0x1000, wanted(args)
    return args


def form(**case):
    text = ctypes.create_string_buffer(100)
    assert _lib.lib().ggk_fp8_form(ctypes.byref(arguments(**case)), text, 100) == 0
    return text.value.decode()


# rows, k, n and what else the call has.  Sizes are small where the form's rule allows it, ragged in rows, columns and K.
CASES = [dict(zip(("rows", "k", "n"), c[:3]), **c[3]) for c in [
    (1, 400, 130, {}), (7, 4096, 14335, {}), (13, 400, 1000, {}), (9, 400, 8193, {}), (16, 1040, 8200, {"out": F32}),
    (29, 1168, 393, {}), (29, 1168, 393, {"fast": True}), (40, 272, 14000, {"fast": True}), (70, 400, 5000, {}),
    (70, 400, 5000, {"fast": True}), (33, 400, 14335, {}), (61, 1168, 14300, {"out": F32}), (64, 144, 14400, {"fast": True}),
    (45, 1040, 14335, {"fast": True}), (700, 1168, 8200, {}), (700, 1168, 8200, {"fast": True}), (9000, 400, 1000, {"fast": True}),
    (9000, 400, 1000, {"out": F32}),
    (5, 400, 700, {"gate": 1}), (20, 400, 1000, {"gate": 1}), (64, 1040, 14335, {"gate": 2}), (64, 4096, 14336, {"gate": 1}),
    (9000, 272, 1000, {"gate": 1}),
    (3, 4096, 700, {"gate": 1, "workspace": True}), (11, 4096, 700, {"gate": 2, "workspace": True}),
    (12, 4096, 4200, {"gate": 1, "workspace": True}), (30, 4096, 390, {"gate": 1, "workspace": True}),
    (40, 4096, 7200, {"gate": 1, "workspace": True}), (60, 4096, 2000, {"gate": 1, "workspace": True}), (200, 2064, 1300, {"gate": 2, "workspace": True}),
    (1, 400, 1792, {"experts": 8, "fan": 2}), (60, 400, 300, {"experts": 16, "fan": 3, "out": F32}),
    (60, 400, 300, {"experts": 4, "fan": 2}), (60, 400, 300, {"experts": 4, "fan": 2, "fast": True}),
    (1, 1168, 14336, {"experts": 8, "fan": 2}), (1, 1168, 14336, {"experts": 8, "fan": 2, "fast": True}),
    (3000, 1040, 2100, {"experts": 6, "fan": 2}), (3000, 1040, 2100, {"experts": 6, "fan": 2, "fast": True}),
    (1500, 2064, 700, {"experts": 4, "fan": 2, "fast": True}),
    (60, 400, 300, {"experts": 4, "fan": 2, "gate": 1}), (3000, 1040, 1100, {"experts": 6, "fan": 2, "gate": 2}),
    (1, 4096, 1792, {"experts": 8, "fan": 2, "gate": 1, "workspace": True}),
    (200, 400, 270, {"experts": 280, "fan": 2, "gate": 1, "workspace": True}),
    (60, 4096, 200, {"experts": 5, "fan": 2, "gate": 2, "workspace": True})]]


def sweep():
    rng = random.Random(1)
    sizes = lambda lo, hi: int(lo * (hi / lo) ** rng.random())
    for _ in range(40000):
        case = dict(rows=sizes(1, 40000), k=16 * sizes(1, 1800), n=sizes(1, 30000))
        if rng.random() < 0.5:
            case.update(experts=sizes(1, 1024), fan=rng.randint(1, 4))
        kind = rng.randrange(4)
        if kind == 0:
            case["out"] = F32
        elif kind == 1:
            case["fast"] = True
        elif kind == 2:
            case.update(gate=rng.randint(1, 2), workspace=rng.random() < 0.7)
        yield case


# ---------------------------------------------------------------- CPU

def test_every_form_is_run_here(tmp_path):
    found = {form(**case) for case in sweep()}
    run = {form(**case) for case in CASES}
    assert run == found, (found - run, run - found)
    # No kernel is built that no call reaches: a stream form is a kernel, tiles of either height are one.
    kernels = [k for k in _scratch("gg_fp8.o", tmp_path) if "fp8_stream_kernel" in k]
    assert len(kernels) == len({f for f in found if f.startswith("stream")})
    kernels = [k for k in _scratch("gg_fp8_tiles.o", tmp_path) if "fp8_tile_kernel" in k]
    assert len(kernels) == len({tuple(f.split()[2:]) for f in found if f.startswith("tiles")})


@pytest.mark.parametrize("fast", [False, True])
def test_64_rows_at_once_where_a_cu_would_get_a_fourth_workgroup(fast):
    for rows in (33, 64):
        assert form(rows=rows, k=4096, n=12288, fast=fast).startswith("stream rows=32 columns=32 ")
        assert form(rows=rows, k=4096, n=12289, fast=fast).startswith("stream rows=64 columns=64 ")
    assert form(rows=40, k=4096, n=6145, gate=1, workspace=True) == "stream rows=64 columns=64 k=4 float pair one"


def test_experts_of_few_slots_by_k_and_slots():
    assert form(rows=384, k=2048, n=300, experts=64, fan=2) == "stream rows=16 columns=256 k=1 float plain experts"
    assert form(rows=384, k=2064, n=300, experts=64, fan=2) == "stream rows=32 columns=128 k=2 float plain experts"
    assert form(rows=385, k=2048, n=300, experts=64, fan=2) == "stream rows=32 columns=128 k=2 float plain experts"


def test_form_of_refused_and_empty_calls():
    text = ctypes.create_string_buffer(b"x" * 20, 20)
    ask = _lib.lib().ggk_fp8_form
    assert ask(None, text, 20) == 1 and ask(ctypes.byref(_lib.GGKFp8Args(**BASE)), None, 20) == 1
    assert ask(ctypes.byref(_lib.GGKFp8Args(**BASE)), text, 0) == 1
    assert ask(ctypes.byref(_lib.GGKFp8Args(**{**BASE, "k": 264})), text, 20) == 1 and text.raw == b"x" * 20
    assert ask(ctypes.byref(_lib.GGKFp8Args(**{**BASE, "n": 0})), text, 20) == 0 and text.value == b""
    assert ask(ctypes.byref(_lib.GGKFp8Args(**BASE)), text, 8) == 0 and text.value == b"stream "


# ---------------------------------------------------------------- GPU

@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace("torch.", ""))
def test_form(torch_cuda, case):
    rows, k, n, experts, fan = case["rows"], case["k"], case["n"], case.get("experts", 0), case.get("fan", 1)
    gate, out, fast = case.get("gate", 0), case.get("out", BF16), case.get("fast", False)
    lead = (experts,) if experts else ()
    x, w = rows_of(rows, k, rows + n), matrix_of(lead, n, k, 7 * k + n)
    if experts:
        ids, counts, order = routing(rows, experts, fan, 4, 0.1 if rows > 1 else 0.0)
    if gate:
        up, activation = matrix_of(lead, n, k, 9 * k + n), ("silu", "gelu")[gate - 1]
        y, scales = torch.zeros(rows * fan, n, dtype=torch.uint8, device="cuda"), torch.zeros(rows * fan, blocks(n), device="cuda")
        args = gated_args(x, w, up, y, scales, activation)
        if experts:
            args.rows, args.experts, args.counts, args.order = rows * fan, experts, counts.data_ptr(), order.data_ptr()
            args.stride_w = args.stride_u = n * k
            args.stride_ws = args.stride_us = blocks(n) * blocks(k)
        if case.get("workspace"):
            room = torch.empty(wanted(args), device="cuda")
            args.workspace, args.workspace_floats = room.data_ptr(), room.numel()
        assert multiply(args) == 0
        got = torch_ops.Fp8Rows(y.view(torch.float8_e4m3fn), scales)
        if experts:
            check_moe_gated(got, *x, w, up, ids, activation)
        else:
            check_gated(got, row_values(*x), matrix_values(*w), matrix_values(*up), activation)
    elif experts:
        weights = torch.rand(rows * fan, device="cuda")
        y = torch_ops.moe_fp8_matmul(*x, *w, counts, order, row_weights=weights, out_dtype=out, fast=fast)
        check_moe(y, *x, *w, ids, not fast, weights)
    else:
        check_product(torch_ops.fp8_matmul(*x, *w, out_dtype=out, fast=fast), row_values(*x), matrix_values(*w), not fast)
