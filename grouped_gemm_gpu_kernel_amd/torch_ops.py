"""PyTorch binding: the grouped GEMM on lists of torch tensors.

    d_i = alpha_i * a_i @ b_i + beta_i * c_i      for every i, in one persistent launch

a_i: float16 [m_i, k_i], b_i: float16 [k_i, n_i], c_i: float32 [m_i, n_i] or None, d_i: float32
[m_i, n_i]; products accumulate in float32 (the contract of the reference's ProblemDesc,
include/grouped_gemm/grouped_gemm.cuh:18-35).  Rows may be padded (a row stride above the row
length, e.g. a column slice of a wider tensor); elements inside a row must be contiguous.

Two forms:
* run_grouped_gemm(a, b, c, alpha, beta, ...) -- one call, the reference's run_grouped_gemm_once
  (src/grouped_gemm.cu:1279-1291): prepares, uploads, launches on the current stream and waits for
  it, because the executor's device buffers are released before it returns.  Registered as the
  custom op torch.ops.grouped_gemm_amd.grouped_gemm.
* GroupedGemmPlan(a, b, c, d, ...) -- prepare and upload once, then run() any number of times on
  any stream without host synchronisation, as the reference's GroupedGemmExecutor is used
  (include/grouped_gemm/grouped_gemm.cuh:94-115).  The plan holds its tensors; refill them in place
  between runs.

Around the products of a mixture-of-experts layer: moe_route (choice of experts, their weights, the counts
and the order by expert, the balance loss, with gradients), MoeGroupedGemmPlan (float16 expert
weights), moe_w4_matmul / w4_matmul (4-bit weights, for a few rows), and the 8-bit path of a feed-forward
layer: rms_norm_fp8 (norm and residual, written as 8-bit rows), moe_fp8_gated / fp8_gated (both projections and
their product, 8-bit rows again) and moe_fp8_matmul / fp8_matmul.

All work runs in the HIP library (lib/libgrouped_gemm_amd.so); there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import importlib.util
import operator
from typing import NamedTuple, Optional, Sequence, Union

import numpy as np
import torch

from . import _lib
from .api import GroupedGemmExecutor, KernelConfig, ProblemDesc, SortMode, prepare_problem_set

Scalars = Union[float, Sequence[float]]

_OP_NAME = "grouped_gemm_amd::grouped_gemm"
_placeholders: dict = {}
_gg_torch = None


def _placeholder(device: torch.device) -> int:
    """A valid device address for operands with no elements (the library rejects null a/b/d
    pointers even where nothing is read, src/grouped_gemm.cu:1304-1307)."""
    key = (device.type, device.index)
    if key not in _placeholders:
        _placeholders[key] = torch.zeros(64, dtype=torch.float32, device=device)
    return _placeholders[key].data_ptr()


def _row_stride(t: torch.Tensor) -> int:
    rows, cols = t.shape
    if rows <= 1 or t.numel() == 0:  # the stride of an empty or one-row matrix is never used
        return max(1, cols)
    return t.stride(0)


def _check_matrix(t: torch.Tensor, name: str, dtype: torch.dtype, shape, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    rows, cols = t.shape
    if t.numel() == 0:
        return
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have contiguous rows (stride(1) == 1)")
    if rows > 1 and t.stride(0) < max(1, cols):
        raise ValueError(f"{name} rows overlap (stride(0) < shape[1])")


def _per_problem(values: Scalars, count: int, name: str) -> list:
    if isinstance(values, (int, float)):
        return [float(values)] * count
    values = [float(v) for v in values]
    if len(values) != count:
        raise ValueError(f"{name} has {len(values)} entries for {count} problems")
    return values


def _problems(a, b, c, d, alpha, beta):
    count = len(a)
    if len(b) != count or len(d) != count or (c is not None and len(c) != count):
        raise ValueError("a, b, c and d must hold one tensor per problem")
    if count == 0:
        return []
    device = a[0].device
    if device.type != "cuda":
        raise ValueError(f"tensors must be on a GPU, got {device}")
    alpha = _per_problem(alpha, count, "alpha")
    beta = _per_problem(beta, count, "beta")
    dummy = _placeholder(device)
    problems = []
    for i in range(count):
        _check_matrix(a[i], f"a[{i}]", torch.float16, None, device)
        m, k = a[i].shape
        _check_matrix(b[i], f"b[{i}]", torch.float16, None, device)
        if b[i].shape[0] != k:
            raise ValueError(f"b[{i}] has {b[i].shape[0]} rows, a[{i}] has {k} columns")
        n = b[i].shape[1]
        _check_matrix(d[i], f"d[{i}]", torch.float32, (m, n), device)
        ci = None if c is None else c[i]
        if ci is not None:
            _check_matrix(ci, f"c[{i}]", torch.float32, (m, n), device)
        problems.append(ProblemDesc(
            m=m, n=n, k=k,
            a=a[i].data_ptr() or dummy, b=b[i].data_ptr() or dummy,
            c=(ci.data_ptr() or dummy) if ci is not None else None,
            d=d[i].data_ptr() or dummy,
            lda=_row_stride(a[i]), ldb=_row_stride(b[i]),
            ldc=_row_stride(ci) if ci is not None else max(1, n), ldd=_row_stride(d[i]),
            alpha=alpha[i], beta=beta[i]))
    return problems


# gg_problem_desc (include/grouped_gemm_amd.h) as a numpy record: one array of them is passed to the
# C ABI as is.
_DESC_DTYPE = np.dtype([("m", "<i4"), ("n", "<i4"), ("k", "<i4"), ("_pad", "<i4"), ("a", "<u8"), ("b", "<u8"),
                        ("c", "<u8"), ("d", "<u8"), ("lda", "<i4"), ("ldb", "<i4"), ("ldc", "<i4"),
                        ("ldd", "<i4"), ("alpha", "<f4"), ("beta", "<f4")])
assert _DESC_DTYPE.itemsize == ctypes.sizeof(_lib.GGProblemDesc)


def _ld(shape, stride) -> int:
    """_row_stride from a shape and stride already read."""
    rows, cols = shape
    if rows <= 1 or rows * cols == 0:
        return max(1, cols)
    return stride[0]


def _problem_table(a, b, c, d, alpha, beta) -> np.ndarray:
    """The problems of tensor lists as gg_problem_desc records, with the checks of _problems: each
    tensor's metadata is read once, in bulk, and any failed check is reported by _problems' own
    per-tensor messages."""
    count = len(a)
    if len(b) != count or len(d) != count or (c is not None and len(c) != count):
        raise ValueError("a, b, c and d must hold one tensor per problem")
    table = np.zeros(count, _DESC_DTYPE)
    if count == 0:
        return table
    device = a[0].device
    if device.type != "cuda":
        raise ValueError(f"tensors must be on a GPU, got {device}")
    cs = list(c) if c is not None else [None] * count
    f16, f32 = torch.float16, torch.float32
    try:
        sa = [t.shape for t in a]
        sb = [t.shape for t in b]
        sd = [t.shape for t in d]
        ok = (all(t.dtype is f16 and t.device == device for t in a) and
              all(t.dtype is f16 and t.device == device for t in b) and
              all(t.dtype is f32 and t.device == device for t in d) and
              all(t is None or (t.dtype is f32 and t.device == device) for t in cs) and
              all(len(x) == 2 and len(y) == 2 and x[1] == y[0] for x, y in zip(sa, sb)) and
              all(z == (x[0], y[1]) for x, y, z in zip(sa, sb, sd)) and
              all(t is None or t.shape == z for t, z in zip(cs, sd)))
        if ok:
            ta = [t.stride() for t in a]
            tb = [t.stride() for t in b]
            td = [t.stride() for t in d]
            tc = [t.stride() if t is not None else None for t in cs]
            # rows contiguous and not overlapping (see _check_matrix)
            for shapes, strides in ((sa, ta), (sb, tb), (sd, td)):
                ok = ok and all((x[1] <= 1 or s[1] == 1 or x[0] * x[1] == 0) and
                                (x[0] <= 1 or s[0] >= max(1, x[1]) or x[0] * x[1] == 0)
                                for x, s in zip(shapes, strides))
            ok = ok and all(t is None or ((z[1] <= 1 or s[1] == 1 or z[0] * z[1] == 0) and
                                          (z[0] <= 1 or s[0] >= max(1, z[1]) or z[0] * z[1] == 0))
                            for t, s, z in zip(cs, tc, sd))
    except (AttributeError, TypeError):
        ok = False
    if not ok:
        _problems(a, b, c, d, alpha, beta)  # raises with the failed check's message
        raise ValueError("tensor lists do not describe grouped GEMM problems")
    dummy = _placeholder(device)
    table["m"] = [x[0] for x in sa]
    table["k"] = [x[1] for x in sa]
    table["n"] = [x[1] for x in sb]
    table["a"] = [t.data_ptr() or dummy for t in a]
    table["b"] = [t.data_ptr() or dummy for t in b]
    table["d"] = [t.data_ptr() or dummy for t in d]
    table["c"] = [(t.data_ptr() or dummy) if t is not None else 0 for t in cs]
    table["lda"] = [_ld(x, s) for x, s in zip(sa, ta)]
    table["ldb"] = [_ld(x, s) for x, s in zip(sb, tb)]
    table["ldd"] = [_ld(x, s) for x, s in zip(sd, td)]
    table["ldc"] = [_ld(z, s) if t is not None else max(1, z[1]) for t, s, z in zip(cs, tc, sd)]
    table["alpha"] = _per_problem(alpha, count, "alpha")
    table["beta"] = _per_problem(beta, count, "beta")
    return table


class GroupedGemmPlan:
    """A prepared grouped GEMM over fixed tensors: prepare_problem_set + executor build once,
    run() per use.  Runs are stream-ordered and must not overlap each other (one scheduler state
    per plan, as one per executor in the reference)."""

    def __init__(self, a: Sequence[torch.Tensor], b: Sequence[torch.Tensor],
                 c: Optional[Sequence[Optional[torch.Tensor]]], d: Sequence[torch.Tensor],
                 alpha: Scalars = 1.0, beta: Scalars = 0.0, *, sort_mode: int = SortMode.kByK,
                 config: Optional[KernelConfig] = None):
        self.config = config if config is not None else KernelConfig.named("128x64x32")
        self.problems = _problems(a, b, c, d, alpha, beta)
        self._tensors = (list(a), list(b), None if c is None else list(c), list(d))
        self.prepared = prepare_problem_set(self.problems, self.config, sort_mode)
        self.executor = GroupedGemmExecutor()
        self.device = a[0].device if len(a) else None
        if self.problems:
            with torch.cuda.device(self.device):
                _lib.check(self.executor.build(self.prepared, self.config), "GroupedGemmExecutor.build")

    @property
    def outputs(self) -> list:
        return self._tensors[3]

    def run(self, stream: Optional[torch.cuda.Stream] = None) -> list:
        if not self.problems:
            return self.outputs
        with torch.cuda.device(self.device):
            stream = stream if stream is not None else torch.cuda.current_stream(self.device)
            _lib.check(self.executor.run(stream), "GroupedGemmExecutor.run")
        return self.outputs

    def close(self) -> None:
        self.executor.close()


def run_grouped_gemm(a: Sequence[torch.Tensor], b: Sequence[torch.Tensor],
                     c: Optional[Sequence[Optional[torch.Tensor]]] = None, alpha: Scalars = 1.0,
                     beta: Scalars = 0.0, *, sort_mode: int = SortMode.kByK,
                     config: Optional[KernelConfig] = None,
                     out: Optional[Sequence[torch.Tensor]] = None) -> list:
    """One grouped launch on the current stream; returns d (allocated unless given as out).
    Waits for the launch before returning (see the module docstring)."""
    if out is None:
        if len(a) and len(b) != len(a):
            raise ValueError("a and b must hold one tensor per problem")
        out = [torch.empty((ai.shape[0], bi.shape[1] if bi.dim() == 2 else 0), dtype=torch.float32,
                           device=ai.device) for ai, bi in zip(a, b)]
    # One C call (prepare, build, launch, wait, release) on a table read from the tensors in bulk.
    table = _problem_table(a, b, c, out, alpha, beta)
    if len(table) == 0:
        return list(out)
    config = config if config is not None else KernelConfig.named("128x64x32")
    device = a[0].device
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        status = _lib.lib().gg_run_grouped_gemm_once(
            table.ctypes.data_as(ctypes.POINTER(_lib.GGProblemDesc)), len(table), int(sort_mode),
            ctypes.byref(config.to_c()), stream or None)
    _lib.check(status, "run_grouped_gemm_once")
    return list(out)


# ---------------------------------------------------------------- mixture of experts

class MoeGroupedGemmPlan:
    """The grouped GEMM of a mixture-of-experts layer with device-side token counts:

        d[rows of e] = alpha * a[rows of e] @ b[e] + beta * c[rows of e]     for every expert e

    a: float16 [T, K], the tokens grouped by expert (expert e owns rows [r_e, r_e + counts[e]),
    r_e = sum of the counts before e); b: float16 [E, K, N]; d (and c): float32 [T, N].  The
    problem set is prepared on the GPU from the int32 counts tensor at every run() (see
    ggk_moe_prepare): no host synchronisation, no allocation, so runs can be captured in a CUDA/HIP
    graph and replayed with new counts.  Rows past T are never touched: counts that add up to more
    are clamped (status() reports it)."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, d: torch.Tensor, c: Optional[torch.Tensor] = None,
                 alpha: float = 1.0, beta: float = 0.0, *, sort_mode: int = SortMode.kByTiles,
                 config: Optional[KernelConfig] = None):
        from .api import MoeGroupedGemm, MoeLayout

        if a.device.type != "cuda":
            raise ValueError(f"tensors must be on a GPU, got {a.device}")
        if b.dim() != 3:
            raise ValueError(f"b must be [experts, K, N], got shape {tuple(b.shape)}")
        experts, k, n = b.shape
        _check_matrix(a, "a", torch.float16, None, a.device)
        if a.shape[1] != k:
            raise ValueError(f"a has {a.shape[1]} columns, b has K = {k}")
        rows = a.shape[0]
        _check_matrix(d, "d", torch.float32, (rows, n), a.device)
        if c is not None:
            _check_matrix(c, "c", torch.float32, (rows, n), a.device)
        if b.dtype != torch.float16 or b.device != a.device:
            raise TypeError("b must be float16 on the same device as a")
        if n > 1 and b.stride(2) != 1:
            raise ValueError("b[e] must have contiguous rows")
        if b.numel() and experts > 1 and b.stride(0) < 1:
            raise ValueError("b experts overlap")
        self.device = a.device
        self.experts = experts
        self.config = config if config is not None else KernelConfig.named("128x64x32")
        dummy = _placeholder(a.device)
        layout = MoeLayout(
            experts=experts, n=n, k=k,
            a=a.data_ptr() or dummy, lda=_row_stride(a),
            b=b.data_ptr() or dummy, ldb=b.stride(1) if k > 1 else max(1, n), stride_b=b.stride(0) if experts > 1 else 0,
            c=(c.data_ptr() or dummy) if c is not None else None, ldc=_row_stride(c) if c is not None else max(1, n),
            d=d.data_ptr() or dummy, ldd=_row_stride(d), alpha=float(alpha), beta=float(beta), max_rows=rows)
        self._tensors = (a, b, c, d)
        with torch.cuda.device(self.device):
            self.moe = MoeGroupedGemm(layout, self.config, int(sort_mode))

    @property
    def output(self) -> torch.Tensor:
        return self._tensors[3]

    def run(self, counts: torch.Tensor, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        if counts.dtype != torch.int32 or counts.device != self.device or counts.numel() != self.experts:
            raise ValueError(f"counts must be int32 [{self.experts}] on {self.device}")
        if not counts.is_contiguous():
            raise ValueError("counts must be contiguous")
        with torch.cuda.device(self.device):
            stream = stream if stream is not None else torch.cuda.current_stream(self.device)
            _lib.check(self.moe.run(counts.data_ptr(), stream), "MoeGroupedGemm.run")
        return self.output

    def status(self) -> int:
        """Status bits of the last run (GGK_MOE_NEGATIVE, GGK_MOE_CLAMPED); reads device memory,
        so it waits for the run."""
        header = self.moe.device_buffers()[3]
        out = torch.empty(_lib.GGK_MOE_HEADER_INTS, dtype=torch.int32)
        torch.cuda.synchronize(self.device)
        _lib.check(_lib.lib().ggk_copy_to_host(out.data_ptr(), header, out.numel() * 4), "copy header")
        return int(out[_lib.GGK_MOE_STATUS])

    def close(self) -> None:
        self.moe.close()


# ---------------------------------------------------------------- routing

_TYPES = {torch.float32: _lib.GGK_TYPE_F32, torch.float16: _lib.GGK_TYPE_F16, torch.bfloat16: _lib.GGK_TYPE_BF16}


class Routing(NamedTuple):
    """What moe_route returns; T tokens, k slots each, E experts, all on the logits' device."""
    weights: torch.Tensor  # float32 [T, k]
    ids: torch.Tensor  # int32 [T, k], -1 where a slot has no expert
    counts: torch.Tensor  # int32 [E], slots on each expert: what MoeGroupedGemmPlan.run takes
    order: torch.Tensor  # int32 [T * k], slot indices t * k + s grouped by expert
    balance_loss: Optional[torch.Tensor]  # float32 scalar, None unless asked for


def _binding():
    """The C++ binding of the calls below (csrc/torch_binding.cpp); raises if it has not been built, or with another torch:
    tensors and autograd nodes are C++ classes whose layout may differ from version to version."""
    global _gg_torch
    if _gg_torch is None:
        if not _lib.TORCH_PATH.exists():
            raise RuntimeError(f"{_lib.TORCH_PATH} is missing: build it with `python -m grouped_gemm_gpu_kernel_amd.build` "
                               "(or __graft_entry__.build()); there is no fallback implementation")
        _lib.lib()
        spec = importlib.util.spec_from_file_location("gg_torch", _lib.TORCH_PATH)
        again = "build it again with `python -m grouped_gemm_gpu_kernel_amd.build`"
        try:
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
        except ImportError as error:  # symbols that this torch does not have, or another Python
            raise RuntimeError(f"{_lib.TORCH_PATH} does not fit this torch ({torch.__version__}): {again}") from error
        built_for = getattr(module, "torch_version", "another version")
        if built_for != str(torch.__version__):
            raise RuntimeError(f"{_lib.TORCH_PATH} was built for torch {built_for}, this is {torch.__version__}: {again}")
        _gg_torch = module
    return _gg_torch


def _check_vector(t: torch.Tensor, name: str, dtype: torch.dtype, count: int, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.numel() != count:
        raise ValueError(f"{name} has {t.numel()} entries, expected {count}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_stored(**tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (t.is_neg() or t._is_zerotensor()):
            raise ValueError(f"{name} is a view whose memory does not hold its values: call resolve_neg() (or add 0)")


def _check_no_tangent(what: str, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} no forward-mode derivative: {name} is a dual tensor (take its primal)")


def moe_route(logits: torch.Tensor, top_k: Optional[int] = None, *, ids: Optional[torch.Tensor] = None,
              token_mask: Optional[torch.Tensor] = None, normalize: bool = True, scale: float = 1.0,
              balance: bool = False) -> Routing:
    """The routing of a mixture-of-experts layer from its router's logits [T, E] (float32, float16 or
    bfloat16; rows may be padded).

    Each token takes its top_k experts of the largest logits, in descending order, ties to the lower
    expert, NaN above everything; an expert with logit -inf is closed to the token.  Instead of
    top_k, ids (int32 [T, k]) gives the experts: they are taken as they stand, the same one twice
    included.  token_mask (bool [T]) is False for padding.  A slot with no expert -- too few open
    ones, an id outside [0, E) or of a closed expert, a padding token -- gets id -1 and weight 0 and is
    not counted.

    weights: scale * softmax over the token's chosen logits (normalize) or scale * the chosen entries
    of the softmax over all experts.  counts and order are what the experts' products take: a token's
    row for slot o is o // k, `order` lists the slots by expert (ascending within one, those without an
    expert last), so MoeGroupedGemmPlan runs on tokens[order // k] with counts, and moe_w4_matmul takes
    both as they are.  balance_loss (with balance): E * sum_e f_e P_e, f_e expert e's share of all
    counted slots and P_e the mean of softmax(logits)[:, e] over the tokens with an expert; 0 if there
    is none.

    weights and balance_loss carry gradients to logits (f_e counts as a constant; no second derivative, and no
    forward-mode one: dual tensors are refused).  Everything runs on the
    current stream of the logits' device without waiting for it, and can be captured in a graph (its
    backward pass with it, unless that leads into an eager graph made on the default stream, the logits' own or
    another of the same leaves that is alive, which is refused); the same call gives the same bits.  E at most 1024, k at most 64."""
    try:
        out = _binding().route(logits, top_k, ids, token_mask, normalize, scale, balance)
    except TypeError:  # an argument of another kind
        _check_route(logits, top_k, ids, token_mask)
        raise
    if out.__class__ is tuple:
        return Routing._make(out)
    if out is None:
        _check_route(logits, top_k, ids, token_mask)
        raise ValueError("moe_route: arguments not in order")
    raise _lib.HipError(out, "ggk_route")


def _check_route(logits, top_k, ids, token_mask) -> None:
    """Says what is wrong with moe_route's arguments (the binding has the same checks)."""
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a torch.Tensor")
    if logits.device.type != "cuda":
        raise ValueError(f"tensors must be on a GPU, got {logits.device}")
    if logits.dtype not in _TYPES:
        raise TypeError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    _check_matrix(logits, "logits", logits.dtype, None, logits.device)
    tokens, experts = logits.shape
    if not 1 <= experts <= _lib.GGK_MOE_MAX_EXPERTS:
        raise ValueError(f"logits has {experts} experts, expected 1 to {_lib.GGK_MOE_MAX_EXPERTS}")
    if (top_k is None) == (ids is None):
        raise ValueError("give one of top_k and ids")
    if ids is not None:
        if not isinstance(ids, torch.Tensor):
            raise TypeError("ids must be a torch.Tensor")
        if ids.dim() != 2 or ids.shape[0] != tokens:
            raise ValueError(f"ids must be [{tokens}, k], got shape {tuple(ids.shape)}")
        _check_vector(ids, "ids", torch.int32, ids.numel(), logits.device)
        slots = ids.shape[1]
        if not 1 <= slots <= _lib.GGK_ROUTE_MAX_SLOTS:
            raise ValueError(f"ids has {slots} slots, expected 1 to {_lib.GGK_ROUTE_MAX_SLOTS}")
    else:
        slots = operator.index(top_k)
        if not 1 <= slots <= min(experts, _lib.GGK_ROUTE_MAX_SLOTS):
            raise ValueError(f"top_k is {slots}, expected 1 to {min(experts, _lib.GGK_ROUTE_MAX_SLOTS)}")
    if tokens * slots > _lib.GGK_ROUTE_MAX_TOTAL_SLOTS:
        raise ValueError(f"{tokens} tokens with {slots} slots each: more than 2^30 slots")
    if token_mask is not None:
        _check_vector(token_mask, "token_mask", torch.bool, tokens, logits.device)
    _check_stored(logits=logits, ids=ids, token_mask=token_mask)
    _check_no_tangent("moe_route has", logits=logits)


# ---------------------------------------------------------------- 4-bit weights

def _check_w4(x, q, scales, zeros, counts, order, row_weights, out_dtype, lead=0) -> None:
    """Says what is wrong with the arguments of the products (the binding has the same checks); lead: dimensions ahead of
    a matrix's two."""
    if row_weights is not None and not isinstance(row_weights, torch.Tensor):
        raise TypeError("row_weights must be a torch.Tensor")
    if not isinstance(x, torch.Tensor) or not isinstance(q, torch.Tensor) or not isinstance(scales, torch.Tensor):
        raise TypeError("x, q and scales must be torch.Tensors")
    device = x.device
    if device.type != "cuda":
        raise ValueError(f"tensors must be on a GPU, got {device}")
    _check_matrix(x, "x", torch.float16, None, device)
    if out_dtype not in (torch.float32, torch.float16):
        raise TypeError(f"out_dtype must be float32 or float16, got {out_dtype}")
    shape = "[N, K / 2]" if lead == 0 else "[experts, N, K / 2]"
    for t, name, dtype in ((q, "q", torch.uint8), (scales, "scales", torch.float16), (zeros, "zeros", torch.uint8)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")
        if t.dim() != 2 + lead:
            raise ValueError(f"{name} must have {2 + lead} dimensions (q is {shape}), got shape {tuple(t.shape)}")
        if t.shape[:-1] != q.shape[:-1]:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, q has {tuple(q.shape)}")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} must have contiguous rows")
        if t.shape[-2] > 1 and t.stride(-2) < t.shape[-1]:
            raise ValueError(f"{name} rows overlap")
    if zeros is not None and zeros.shape != scales.shape:
        raise ValueError(f"zeros has shape {tuple(zeros.shape)}, scales has {tuple(scales.shape)}")
    k = 2 * q.shape[-1]
    if x.shape[1] != k:
        raise ValueError(f"x has {x.shape[1]} columns, q has K = {k}")
    groups = scales.shape[-1]
    if groups < 1 or k % groups != 0 or (k // groups) % 32 != 0 or k == 0:
        raise ValueError(f"scales has {groups} groups for K = {k}: a group is a multiple of 32 values that divides K")
    if max(k, q.shape[-2]) > _lib.GGK_W4_MAX_EXTENT:
        raise ValueError(f"q stands for [{q.shape[-2]}, {k}] weights: N and K are at most 2^28")
    if q.data_ptr() % 16 != 0 or any(n > 1 and s % 16 != 0 for n, s in zip(q.shape[:-1], q.stride()[:-1])):
        raise ValueError("q must start on a multiple of 16 bytes, and so must its rows and matrices")
    _check_stored(x=x, q=q, scales=scales, zeros=zeros, row_weights=row_weights)
    if torch.is_grad_enabled() and (x.requires_grad or scales.requires_grad or
                                    (row_weights is not None and row_weights.requires_grad)):
        raise RuntimeError("the products with 4-bit weights have no gradient: detach x, scales and row_weights")
    _check_no_tangent("the products with 4-bit weights have", x=x, scales=scales, row_weights=row_weights)


def w4_matmul(x: torch.Tensor, q: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *,
              out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y = x @ w.T for a few rows x (float16 [M, K]) and a matrix w [N, K] of 4-bit weights:

        w[j, k] = scales[j, k // G] * (q[j, k] - zeros[j, k // G])

    q: uint8 [N, K / 2], two values a byte along K, the low half the even k; scales: float16 [N, K / G];
    zeros: uint8 [N, K / G], 8 everywhere if not given.  The group G is a multiple of 32 that divides
    K.  Rows of x, scales and zeros may be padded, those of q by multiples of 16 bytes.  Weights are
    never rounded: products and sums are float32, y is float32 or float16, rounded once.

    Runs on the current stream of x's device, without waiting; no gradient (inputs that require one are
    refused, and dual tensors of forward mode).  Any number of rows is right; it is made for up to 64 or so."""
    return _w4(_check_w4, x, q, scales, zeros, None, None, None, out_dtype)


def moe_w4_matmul(x: torch.Tensor, q: torch.Tensor, scales: torch.Tensor, counts: torch.Tensor, order: torch.Tensor,
                  zeros: Optional[torch.Tensor] = None, *, row_weights: Optional[torch.Tensor] = None,
                  out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """w4_matmul for the expert matrices of a mixture-of-experts layer, q uint8 [E, N, K / 2], scales (and zeros)
    [E, N, K / G], each slot with its expert's:

        y[o] = row_weights[o] * x[o // fan] @ w[expert of o].T       o = 0 .. R - 1, fan = R // x.shape[0]

    counts (int32 [E]) and order (int32 [R]) as moe_route returns them: with x [T, K] the tokens, R = T * k
    and y [T * k, N] holds token t's slots at rows t * k ...; with x already one row a slot, fan is 1.
    Slots without an expert (the end of order, past the counts' sum) get zeros.  row_weights: float32, R
    entries (e.g. the routing's weights), 1 if not given.  Counts and order stay on the GPU and
    are not trusted: a negative count is taken as 0, counts past R and entries outside [0, R) are dropped;
    rows that order does not name are left unwritten, and one that it names twice gets one of its products."""
    if counts is None or order is None:
        raise TypeError("counts and order must be torch.Tensors")
    return _w4(_check_moe_w4, x, q, scales, zeros, counts, order, row_weights, out_dtype)


def _w4(check, x, q, scales, zeros, counts, order, row_weights, out_dtype):
    try:
        out = _binding().w4(x, q, scales, zeros, counts, order, row_weights, out_dtype)
    except TypeError:  # an argument of another kind
        check(x, q, scales, zeros, counts, order, row_weights, out_dtype)
        raise
    if isinstance(out, torch.Tensor):
        return out
    if out is None:
        check(x, q, scales, zeros, counts, order, row_weights, out_dtype)
        raise ValueError("products with 4-bit weights: arguments not in order")
    raise _lib.HipError(out, "ggk_w4_multiply")


def _check_moe_w4(x, q, scales, zeros, counts, order, row_weights, out_dtype) -> None:
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q must be [experts, N, K / 2]")
    _check_w4(x, q, scales, zeros, counts, order, row_weights, out_dtype, lead=1)
    experts = q.shape[0]
    if not 1 <= experts <= _lib.GGK_MOE_MAX_EXPERTS:
        raise ValueError(f"q has {experts} experts, expected 1 to {_lib.GGK_MOE_MAX_EXPERTS}")
    _check_vector(counts, "counts", torch.int32, experts, x.device)
    if not isinstance(order, torch.Tensor):
        raise TypeError("order must be a torch.Tensor")
    rows = order.numel()
    _check_vector(order, "order", torch.int32, rows, x.device)
    if rows > _lib.GGK_ROUTE_MAX_TOTAL_SLOTS:
        raise ValueError(f"order has {rows} entries: more than 2^30")
    if rows and (x.shape[0] == 0 or rows % x.shape[0] != 0):
        raise ValueError(f"order has {rows} entries, not a multiple of x's {x.shape[0]} rows")
    if row_weights is not None:
        _check_vector(row_weights, "row_weights", torch.float32, rows, x.device)
    _check_stored(counts=counts, order=order)


# ---------------------------------------------------------------- 8-bit rows

_FP8 = torch.float8_e4m3fn
_GATES = {"silu": _lib.GGK_GATE_SILU, "gelu": _lib.GGK_GATE_GELU}


class Fp8Rows(NamedTuple):
    """Rows of 8-bit numbers: a value is its number times its block's scale."""
    q: torch.Tensor  # float8_e4m3fn [T, N]
    scales: torch.Tensor  # float32 [T, ceil(N / 128)], one for each 128 columns


class Fp8Norm(NamedTuple):
    """What rms_norm_fp8 returns."""
    q: torch.Tensor  # float8_e4m3fn [T, H]
    scales: torch.Tensor  # float32 [T, ceil(H / 128)]
    y: Optional[torch.Tensor]  # [T, H] in x's type, None unless asked for
    residual: Optional[torch.Tensor]  # x + residual in x's type, None without a residual


def _blocks(n: int) -> int:
    return (n + _lib.GGK_FP8_BLOCK - 1) // _lib.GGK_FP8_BLOCK


def _check_no_gradient(what: str, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and torch.is_grad_enabled() and t.requires_grad:
            raise RuntimeError(f"{what} no gradient: detach {name}")


def rms_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-6, plain: bool = False) -> Fp8Norm:
    """The residual's addition, the root-mean-square norm and its rounding to 8 bits, in one pass over x [T, H]
    (float32, float16 or bfloat16; rows may be padded):

        h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight                   (float32)
        scale of 128 columns = max(max |y| / 448, 2^-126),  q = y / scale to the nearest float8_e4m3fn

    weight: [H] of x's type or float32, ones if not given; residual: like x.  Returns q and scales, what fp8_matmul,
    fp8_gated and their expert forms take (for H a multiple of 16); with `plain` y in x's type too (what a router
    reads), with a residual h in x's type, the next one.  y, q and scales are made from h in float32, before that
    rounding.  A block with a NaN has a NaN scale and NaN numbers, one with an infinity an infinite scale.

    Runs on the current stream of x's device, without waiting; no gradient (inputs that require one are
    refused, and dual tensors of forward mode).  H at most 32768."""
    try:
        out = _binding().norm_fp8(x, weight, residual, eps, plain)
    except TypeError:  # an argument of another kind
        _check_norm_fp8(x, weight, residual)
        raise
    if out.__class__ is tuple:
        return Fp8Norm._make(out)
    if out is None:
        _check_norm_fp8(x, weight, residual)
        raise ValueError("rms_norm_fp8: arguments not in order")
    raise _lib.HipError(out, "ggk_norm_fp8")


def _check_norm_fp8(x, weight, residual) -> None:
    """Says what is wrong with rms_norm_fp8's arguments (the binding has the same checks)."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    if x.device.type != "cuda":
        raise ValueError(f"tensors must be on a GPU, got {x.device}")
    if x.dtype not in _TYPES:
        raise TypeError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    _check_matrix(x, "x", x.dtype, None, x.device)
    rows, columns = x.shape
    if not 1 <= columns <= _lib.GGK_NORM_MAX_COLUMNS:
        raise ValueError(f"x has {columns} columns, expected 1 to {_lib.GGK_NORM_MAX_COLUMNS}")
    if rows > _lib.GGK_ROUTE_MAX_TOTAL_SLOTS:
        raise ValueError(f"x has {rows} rows: more than 2^30")
    if weight is not None:
        if not isinstance(weight, torch.Tensor):
            raise TypeError("weight must be a torch.Tensor")
        if weight.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"weight must be {x.dtype} or float32, got {weight.dtype}")
        if weight.dim() != 1:
            raise ValueError(f"weight must be 1-D, got shape {tuple(weight.shape)}")
        _check_vector(weight, "weight", weight.dtype, columns, x.device)
    if residual is not None:
        _check_matrix(residual, "residual", x.dtype, x.shape, x.device)
    _check_stored(x=x, weight=weight, residual=residual)
    _check_no_gradient("rms_norm_fp8 has", x=x, weight=weight, residual=residual)
    _check_no_tangent("rms_norm_fp8 has", x=x, weight=weight, residual=residual)


def fp8_matmul(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *,
               out_dtype: torch.dtype = torch.bfloat16, fast: bool = False) -> torch.Tensor:
    """y = x @ w.T for 8-bit rows x [M, K] and an 8-bit matrix w [N, K] (float8_e4m3fn) with float32 scales: x_scales
    [M, ceil(K / 128)], one for each 128 values of a row, w_scales [ceil(N / 128), ceil(K / 128)], one for each block of
    128 x 128 (the last ones may be cut).

    K is a multiple of 16; x and w start on multiples of 16 bytes, and so do their rows, which may be padded; rows
    of scales may be padded too.  Sums are float32, of products in binary16, which holds 8-bit numbers exactly.  y is
    float32, float16 or bfloat16, rounded once.  A product of two scales is a float32: below 2^-126 it has fewer bits,
    above 2^128 it is infinite.

    fast=True (for the 16-bit types) lets the call use the 8-bit matrix instructions where that is quicker: up to twice as
    fast for many rows.  They align 8 products at a time to the largest and drop what lies 2^-13 of its power of two and more
    below it.  Of normal terms that loses about 1.5e-5 of a sum; where single products are 2^13 times the ones beside them
    those are lost whole, also where the large ones cancel.

    Runs on the current stream of x's device, without waiting; no gradient (inputs that require one are
    refused, and dual tensors of forward mode)."""
    return _fp8(x, x_scales, w, w_scales, None, None, _lib.GGK_GATE_NONE, None, None, None, out_dtype, fast)


def fp8_gated(x: torch.Tensor, x_scales: torch.Tensor, gate: torch.Tensor, gate_scales: torch.Tensor, up: torch.Tensor,
              up_scales: torch.Tensor, *, activation: str = "silu") -> Fp8Rows:
    """act(x @ gate.T) * (x @ up.T) as 8-bit rows, both projections of a gated feed-forward block, the activation and
    their product in one kernel; operands as fp8_matmul's, gate and up [N, K] (the halves of one matrix of both can be given
    as views).  activation: "silu", or "gelu" (the form with tanh).  Rows are made of float32 as rms_norm_fp8 makes
    them, of products in binary16 as fp8_matmul's."""
    return _fp8(x, x_scales, gate, gate_scales, up, up_scales, _gate(activation), None, None, None, torch.float32)


def moe_fp8_matmul(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, counts: torch.Tensor,
                   order: torch.Tensor, *, row_weights: Optional[torch.Tensor] = None,
                   out_dtype: torch.dtype = torch.bfloat16, fast: bool = False) -> torch.Tensor:
    """fp8_matmul for the expert matrices of a mixture-of-experts layer, w [E, N, K], w_scales [E, ceil(N / 128),
    ceil(K / 128)], each slot with its expert's:

        y[o] = row_weights[o] * x[o // fan] @ w[expert of o].T       o = 0 .. R - 1, fan = R // x.shape[0]

    counts (int32 [E]) and order (int32 [R]) as moe_route returns them; row_weights (float32, R entries) as for
    moe_w4_matmul; out_dtype and fast as for fp8_matmul.  Slots without an expert get zeros.  Counts and order stay on the GPU and are not trusted: a
    negative count is taken as 0, counts past R and entries outside [0, R) are dropped; rows that order does not name are
    left unwritten, and each value of one that it names twice is one of its products'."""
    if counts is None or order is None:
        raise TypeError("counts and order must be torch.Tensors")
    return _fp8(x, x_scales, w, w_scales, None, None, _lib.GGK_GATE_NONE, counts, order, row_weights, out_dtype, fast)


def moe_fp8_gated(x: torch.Tensor, x_scales: torch.Tensor, gate: torch.Tensor, gate_scales: torch.Tensor,
                  up: torch.Tensor, up_scales: torch.Tensor, counts: torch.Tensor, order: torch.Tensor, *,
                  activation: str = "silu") -> Fp8Rows:
    """fp8_gated for expert matrices, slots as in moe_fp8_matmul, whose next call reads these rows (one a slot) with the
    same counts and order.  Slots without an expert get numbers 0 and scales 2^-126; a slot that order names twice
    may get one product's numbers with the other's scales."""
    if counts is None or order is None:
        raise TypeError("counts and order must be torch.Tensors")
    return _fp8(x, x_scales, gate, gate_scales, up, up_scales, _gate(activation), counts, order, None, torch.float32)


def _gate(activation) -> int:
    if not isinstance(activation, str) or activation not in _GATES:
        raise ValueError(f"activation must be one of {sorted(_GATES)}, got {activation!r}")
    return _GATES[activation]


def _fp8(x, x_scales, w, w_scales, up, up_scales, gate, counts, order, row_weights, out_dtype, fast=False):
    """out_dtype is not read with a gate: the rows are 8-bit ones."""
    try:
        out = _binding().fp8(x, x_scales, w, w_scales, up, up_scales, gate, counts, order, row_weights, out_dtype, fast)
    except TypeError:  # an argument of another kind
        _check_fp8(x, x_scales, w, w_scales, up, up_scales, gate, counts, order, row_weights, out_dtype, fast)
        raise
    if isinstance(out, torch.Tensor):
        return out
    if out.__class__ is tuple:
        return Fp8Rows._make(out)
    if out is None:
        _check_fp8(x, x_scales, w, w_scales, up, up_scales, gate, counts, order, row_weights, out_dtype, fast)
        raise ValueError("8-bit products: arguments not in order")
    raise _lib.HipError(out, "ggk_fp8_multiply")


def _check_fp8_matrix(w, w_scales, name, scales_name, shape, lead, device) -> None:
    for t, which, dtype in ((w, name, _FP8), (w_scales, scales_name, torch.float32)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{which} must be a torch.Tensor")
        if t.dtype != dtype:
            raise TypeError(f"{which} must be {dtype}, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{which} is on {t.device}, expected {device}")
        if t.dim() != 2 + lead:
            raise ValueError(f"{which} must have {2 + lead} dimensions, got shape {tuple(t.shape)}")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{which} must have contiguous rows")
        if t.shape[-2] > 1 and t.stride(-2) < t.shape[-1]:
            raise ValueError(f"{which} rows overlap")
    if shape is not None and w.shape != shape:
        raise ValueError(f"{name} has shape {tuple(w.shape)}, expected {tuple(shape)}")
    expected = (*w.shape[:-2], _blocks(w.shape[-2]), _blocks(w.shape[-1]))
    if tuple(w_scales.shape) != expected:
        raise ValueError(f"{scales_name} has shape {tuple(w_scales.shape)}, expected {expected} for {name} "
                         f"{tuple(w.shape)}: a scale for each block of 128 x 128")
    if w.shape[-2] > _lib.GGK_FP8_MAX_N or w.shape[-1] > _lib.GGK_FP8_MAX_K:
        raise ValueError(f"{name} has shape {tuple(w.shape)}: N is at most 2^28, K at most 2^22")
    if w.shape[-2] > 1 and w.stride(-2) > _lib.GGK_FP8_MAX_LD:
        raise ValueError(f"{name}'s rows are more than 2^22 bytes apart")
    if w.data_ptr() % 16 != 0 or any(n > 1 and s % 16 != 0 for n, s in zip(w.shape[:-1], w.stride()[:-1])):
        raise ValueError(f"{name} must start on a multiple of 16 bytes, and so must its rows and matrices")


def _check_fp8(x, x_scales, w, w_scales, up, up_scales, gate, counts, order, row_weights, out_dtype, fast) -> None:
    """Says what is wrong with the arguments of the 8-bit products (the binding has the same checks)."""
    if not isinstance(x, torch.Tensor) or not isinstance(x_scales, torch.Tensor) or not isinstance(w, torch.Tensor):
        raise TypeError("x, x_scales and the matrices must be torch.Tensors")
    device = x.device
    if device.type != "cuda":
        raise ValueError(f"tensors must be on a GPU, got {device}")
    _check_matrix(x, "x", _FP8, None, device)
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    if fast and out_dtype == torch.float32:
        raise ValueError("fast products give 16-bit results: out_dtype is torch.float32")
    lead = 0 if counts is None else 1
    name = "w" if gate == _lib.GGK_GATE_NONE else "gate"
    _check_fp8_matrix(w, w_scales, name, f"{name}_scales", None, lead, device)
    if gate != _lib.GGK_GATE_NONE:
        _check_fp8_matrix(up, up_scales, "up", "up_scales", w.shape, lead, device)
    k = w.shape[-1]
    if x.shape[1] != k:
        raise ValueError(f"x has {x.shape[1]} columns, {name} has K = {k}")
    if k < 16 or k % 16 != 0:
        raise ValueError(f"K is {k}, expected a multiple of 16")
    if x.data_ptr() % 16 != 0 or (x.shape[0] > 1 and x.stride(0) % 16 != 0):
        raise ValueError("x must start on a multiple of 16 bytes, and so must its rows")
    _check_matrix(x_scales, "x_scales", torch.float32, (x.shape[0], _blocks(k)), device)
    rows = x.shape[0]
    if counts is not None:
        experts = w.shape[0]
        if not 1 <= experts <= _lib.GGK_MOE_MAX_EXPERTS:
            raise ValueError(f"{name} has {experts} experts, expected 1 to {_lib.GGK_MOE_MAX_EXPERTS}")
        _check_vector(counts, "counts", torch.int32, experts, device)
        if not isinstance(order, torch.Tensor):
            raise TypeError("order must be a torch.Tensor")
        rows = order.numel()
        _check_vector(order, "order", torch.int32, rows, device)
        if rows and (x.shape[0] == 0 or rows % x.shape[0] != 0):
            raise ValueError(f"order has {rows} entries, not a multiple of x's {x.shape[0]} rows")
        if row_weights is not None:
            _check_vector(row_weights, "row_weights", torch.float32, rows, device)
    if rows > _lib.GGK_ROUTE_MAX_TOTAL_SLOTS:
        raise ValueError(f"{rows} rows: more than 2^30")
    floats = {"x": x, "x_scales": x_scales, name: w, f"{name}_scales": w_scales, "up": up, "up_scales": up_scales,
              "row_weights": row_weights}
    _check_stored(**floats, counts=counts, order=order)
    _check_no_gradient("the 8-bit products have", **floats)
    _check_no_tangent("the 8-bit products have", **floats)


# ---------------------------------------------------------------- custom op

@torch.library.custom_op(_OP_NAME, mutates_args=())
def _grouped_gemm_op(a: list[torch.Tensor], b: list[torch.Tensor], c: list[Optional[torch.Tensor]],
                     alpha: list[float], beta: list[float], sort_mode: int) -> list[torch.Tensor]:
    """c: one entry per problem (None where C is not read), or an empty list for no C at all."""
    return run_grouped_gemm(a, b, c if len(c) else None, alpha, beta, sort_mode=sort_mode)


@_grouped_gemm_op.register_fake
def _grouped_gemm_fake(a, b, c, alpha, beta, sort_mode):
    return [ai.new_empty((ai.shape[0], bi.shape[1]), dtype=torch.float32) for ai, bi in zip(a, b)]


grouped_gemm_op = _grouped_gemm_op
