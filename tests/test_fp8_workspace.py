"""The workspace of gated 8-bit products in the C-ABI: its size is stated, a smaller one is refused, none or one of no stated size
is done without; nothing past it is written."""
import ctypes
import math

import pytest
import torch

from grouped_gemm_gpu_kernel_amd import _lib, torch_ops
from test_fp8 import (BASE, FP8, GATE, MOE, blocks, check_gated, check_moe_gated, matrix_of, matrix_values, routing, row_values,
                      rows_of)

PAIR = {**GATE, "k": 4096, "ldx": 4096, "ldw": 4096, "ldu": 4096, "ldxs": 32, "ldws": 32, "ldus": 32}  # 4 rows by 200: two launches


def check(over):
    return _lib.lib().ggk_fp8_check(ctypes.byref(_lib.GGKFp8Args(**{**BASE, **over})))


# ---------------------------------------------------------------- CPU

@pytest.mark.parametrize("over,status", [
    ({}, 0), ({"workspace": 0x1000}, 0), ({"workspace": 0x1000, "workspace_floats": 1600}, 0),
    ({"workspace": 0x1000, "workspace_floats": 1 << 40}, 0), ({"workspace": 0x1000, "workspace_floats": 1599}, 1),
    ({"workspace": 0x1000, "workspace_floats": 1}, 1), ({"workspace": 0x1000, "workspace_floats": -1}, 1),
    ({"workspace_floats": -1}, 1), ({"workspace_floats": 1}, 0), ({"workspace": 0x1008, "workspace_floats": 1600}, 1)])
def test_a_workspace_that_is_too_small_is_refused(over, status):
    args = _lib.GGKFp8Args(**{**BASE, **PAIR, **over})
    assert _lib.lib().ggk_fp8_check(ctypes.byref(args)) == status
    if status:  # before anything is launched
        assert _lib.lib().ggk_fp8_multiply(ctypes.byref(args), None) == status


def test_sizes_of_other_calls_are_not_enough():
    """What another batch was told is looked at, and the question itself does not read it."""
    floats = ctypes.c_longlong(-1)
    for n in (1, 100, 199, 200):
        args = _lib.GGKFp8Args(**{**BASE, **PAIR, "n": n, "workspace": 0x1000, "workspace_floats": 1})
        assert _lib.lib().ggk_fp8_workspace(ctypes.byref(args), ctypes.byref(floats)) == 0
        assert floats.value == 2 * 4 * ((n + 3) // 4 * 4)
        for have in (floats.value, floats.value - 1):
            args.workspace_floats = have
            assert _lib.lib().ggk_fp8_check(ctypes.byref(args)) == (0 if have == floats.value else 1)
    # Calls that make no use of one take any size: plain products, gated ones of many rows.
    assert check({"workspace": 0x1000, "workspace_floats": 1}) == 0
    assert check({**GATE, "rows": 4000, "x_rows": 4000, "workspace": 0x1000, "workspace_floats": 1}) == 0


# ---------------------------------------------------------------- GPU

def gated_args(x, gate, up, y, scales, activation):
    m, k, n = x[0].shape[0], x[0].shape[1], gate[0].shape[-2]
    return _lib.GGKFp8Args(
        rows=m, x_rows=m, n=n, k=k, gate=1 if activation == "silu" else 2, x=x[0].data_ptr(), ldx=k, x_scales=x[1].data_ptr(),
        ldxs=blocks(k), w=gate[0].data_ptr(), ldw=k, w_scales=gate[1].data_ptr(), ldws=blocks(k), up=up[0].data_ptr(), ldu=k,
        up_scales=up[1].data_ptr(), ldus=blocks(k), y=y.data_ptr(), ldy=n, y_scales=scales.data_ptr(), ldys=blocks(n))


def wanted(args):
    floats = ctypes.c_longlong(-1)
    assert _lib.lib().ggk_fp8_workspace(ctypes.byref(args), ctypes.byref(floats)) == 0
    return floats.value


def multiply(args):
    return _lib.lib().ggk_fp8_multiply(ctypes.byref(args), torch.cuda.current_stream().cuda_stream)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,n", [(1, 4096, 520), (7, 8192, 129), (13, 2080, 300), (50, 4096, 257), (200, 2064, 389), (12, 4096, 4200),
                                   (40, 4096, 7200)])
def test_gated_rows_from_a_workspace(torch_cuda, m, k, n, activation):
    x, gate, up = rows_of(m, k, m + n), matrix_of((), n, k, 7 * k + n), matrix_of((), n, k, 9 * k + n)
    values = row_values(*x), matrix_values(*gate), matrix_values(*up)
    y, scales = torch.zeros(m, n, dtype=torch.uint8, device="cuda"), torch.zeros(m, blocks(n), device="cuda")
    args = gated_args(x, gate, up, y, scales, activation)
    floats = wanted(args)
    assert floats == 2 * m * ((n + 3) // 4 * 4)
    workspace = torch.full((floats + 64,), 77.0, device="cuda")
    args.workspace = workspace.data_ptr()
    args.workspace_floats = floats - 1
    assert multiply(args) == 1
    torch.cuda.synchronize()
    assert (workspace == 77).all() and not y.any() and not scales.any()
    args.workspace_floats = floats
    assert multiply(args) == 0
    check_gated(torch_ops.Fp8Rows(y.view(FP8), scales), *values, activation)
    assert (workspace[floats:] == 77).all() and not (workspace[:floats] == 77).all()
    workspace.fill_(77)
    args.workspace_floats = 0  # not known: done without
    y.zero_()
    assert multiply(args) == 0
    check_gated(torch_ops.Fp8Rows(y.view(FP8), scales), *values, activation)
    assert (workspace == 77).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,n", [(5, 139), (60, 139)])
def test_slots_from_a_workspace_with_an_order_that_is_not_trusted(torch_cuda, tokens, n):
    experts, top_k, k = 4, 2, 4096
    rows, in_n, in_k = tokens * top_k, blocks(n), blocks(k)
    x, w, up = rows_of(tokens, k, 1), matrix_of((experts,), n, k, 2), matrix_of((experts,), n, k, 3)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(3)).int().cuda()
    order[5], order[9] = -3, rows + 7  # two slots that nothing names
    lost = sorted(set(range(rows)) - set(order.tolist()))
    counts = torch.tensor([rows // 2, -5, 1 << 30, 1 << 30], dtype=torch.int32, device="cuda")
    y, scales = torch.full((rows, n), 0x55, dtype=torch.uint8, device="cuda"), torch.full((rows, in_n), 77.0, device="cuda")
    args = gated_args(x, w, up, y, scales, "silu")
    args.rows, args.experts, args.counts, args.order = rows, experts, counts.data_ptr(), order.data_ptr()
    args.stride_w = args.stride_u = n * k
    args.stride_ws = args.stride_us = in_n * in_k
    floats = wanted(args)
    assert floats == 2 * rows * ((n + 3) // 4 * 4)
    workspace = torch.full((floats + 64,), math.nan, device="cuda")
    args.workspace, args.workspace_floats = workspace.data_ptr(), floats
    assert multiply(args) == 0
    assert (y[lost] == 0x55).all() and (scales[lost] == 77).all() and workspace[floats:].isnan().all()
    ids = torch.full((rows,), -2)
    for place, slot in enumerate(order.tolist()):
        if 0 <= slot < rows:
            ids[slot] = 0 if place < rows // 2 else 2
    ids = ids.cuda()
    for e in (0, 2):
        at = (ids == e).nonzero()[:, 0]
        check_gated(torch_ops.Fp8Rows(y[at].view(FP8), scales[at]), row_values(*x)[at // top_k], matrix_values(w[0][e], w[1][e]),
                    matrix_values(up[0][e], up[1][e]))


@pytest.mark.gpu
def test_calls_through_torch_use_one(torch_cuda):
    """The binding states the size it allocated: the rows are those of the C-ABI's call with a workspace, bit for bit."""
    x, gate, up = rows_of(3, 4096, 1), matrix_of((), 700, 4096, 2), matrix_of((), 700, 4096, 3)
    y, scales = torch.zeros(3, 700, dtype=torch.uint8, device="cuda"), torch.zeros(3, 6, device="cuda")
    args = gated_args(x, gate, up, y, scales, "silu")
    workspace = torch.empty(wanted(args), device="cuda")
    args.workspace, args.workspace_floats = workspace.data_ptr(), workspace.numel()
    assert multiply(args) == 0
    rows = torch_ops.fp8_gated(*x, *gate, *up)
    assert torch.equal(rows.q.view(torch.uint8), y) and torch.equal(rows.scales, scales)
    ids, counts, order = routing(4, 6, 2, 1)
    w = matrix_of((6,), 139, 4096, 4)
    check_moe_gated(torch_ops.moe_fp8_gated(*rows_of(4, 4096, 5), *w, *w, counts, order), *rows_of(4, 4096, 5), w, w, ids)
