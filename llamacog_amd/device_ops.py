"""MXFP4 products and expert routing on torch tensors of an MI355X: the operators of
include/ggml-mi355x.h that need no ggml graph, called on device memory in place.

Every function launches on torch's current stream of its tensors' device and returns without
waiting; nothing is kept between calls, and a call may be captured into a graph.  Arguments are
checked on the host (ValueError, TypeError); what depends on values on the device is defined
instead: expert ids outside 0 .. n_expert - 1 belong to no expert.  There is no CPU form, and no
gradient is recorded: an input that asks for one is refused (moe_combine_back and, for moe_gather,
moe_combine are the gradients).

    plan = moe_sort(ids, n_expert)                       # ids [T, used] from the router
    h = mx4_mul_mat_id(w_up, x, plan)                    # [T * used, F], rows sorted by expert
    y = mx4_mul_mat_id(w_down, act(h), plan, x_sorted=True)
    out = moe_combine(y, plan, weights)                  # [T, D]
"""
from __future__ import annotations

import ctypes
import os
from typing import NamedTuple

import torch

from . import PKG, BackendMissing

LIBRARY = os.path.join(PKG, "libmi355x-ops.so")
MAX_EXPERTS, MAX_USED = 1024, 16

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_MX4 = -4
_ERRORS = {-1: (TypeError, "unsupported element type"), -2: (ValueError, "unsupported shape"),
           -3: (ValueError, "misaligned tensor"), -4: (ValueError, "workspace too small"), -5: (RuntimeError, "HIP error")}
_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
_SIGNATURES = {
    "mi355x_mx4_quantize": [_I, _P, _L, _L, _L, _P, _P, _P],
    "mi355x_mx4_dequantize": [_P, _P, _L, _L, _I, _P, _P],
    "mi355x_mx4_mul_mat": [_P, _P, _L, _L, _I, _P, _P, _L, _L, _I, _P, _P, _L, _P],
    "mi355x_mx4_mul_mat_id": [_P, _P, _L, _L, _L, _I, _P, _P, _L, _L, _L, _I, _P, _P, _I, _P, _P, _L, _P],
    "mi355x_moe_sort": [_P, _I, _L, _L, _L, _P, _P, _P, _P, _L, _P],
    "mi355x_moe_gather": [_I, _P, _L, _L, _L, _L, _P, _P, _P, _P],
    "mi355x_moe_combine": [_I, _P, _L, _L, _L, _L, _P, _P, _P, _P],
    "mi355x_moe_combine_back": [_I, _P, _L, _P, _L, _L, _L, _L, _P, _P, _P, _P, _P, _P],
    "mi355x_mx4_scales_bytes": [_L, _L],
    "mi355x_mx4_mul_mat_workspace": [_L, _L],
    "mi355x_moe_sort_workspace": [_L, _L, _L],
}
_lib = None


def library() -> ctypes.CDLL:
    """libmi355x-ops.so; BackendMissing if it is not built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIBRARY):
            raise BackendMissing(f"operators not built: {LIBRARY} is missing (run __graft_entry__.build())")
        lib = ctypes.CDLL(LIBRARY)
        for name, args in _SIGNATURES.items():
            f = getattr(lib, name)
            f.argtypes = args
            f.restype = _L if name.endswith(("_bytes", "_workspace")) else _I
        _lib = lib
    return _lib


class Mx4(NamedTuple):
    """MXFP4 rows.  codes uint8 [..., rows, K / 2]: element 2 i in the low half of byte i, E2M1.
    scales uint8 [..., ceil(K / 256), rows, 8]: byte b of plane s is the exponent (2^(byte - 127),
    255 = NaN) of a row's elements 256 s + 32 b to 256 s + 32 b + 31; bytes past K have no meaning
    (mx4_quantize sets them to 0)."""

    codes: torch.Tensor
    scales: torch.Tensor


class MoePlan(NamedTuple):
    """A routing step.  order int32 [T * used]: the pairs t * used + slot by expert, -1 behind the
    last; rank int32 [T, used]: each pair's place in it, -1 for an id that is no expert's; offsets
    int32 [n_expert + 1]: the first place of each expert."""

    order: torch.Tensor
    rank: torch.Tensor
    offsets: torch.Tensor


# ---- argument checks -----------------------------------------------------------------------------
def _device(t: torch.Tensor, what: str) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: a tensor is wanted, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{what}: a tensor on an MI355X is wanted, got one on {t.device}")
    return t.device


def _matrix(t: torch.Tensor, what: str, device=None, shape=None) -> torch.device:
    """A float [rows, columns] tensor whose columns lie side by side."""
    d = _device(t, what)
    if device is not None and d != device:
        raise ValueError(f"{what}: on {d}, the others on {device}")
    if t.dtype not in _TYPE:
        raise TypeError(f"{what}: float32, float16 or bfloat16 is wanted, got {t.dtype}")
    if t.dim() != 2 or (shape is not None and tuple(t.shape) != shape):
        raise ValueError(f"{what}: shape {shape if shape is not None else '[rows, columns]'} is wanted, got {tuple(t.shape)}")
    if t.stride(1) != 1 and t.shape[1] > 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{what}: columns have to lie side by side and rows apart, got strides {t.stride()}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: no gradient is recorded here; pass a detached tensor")
    return d


def _ints(t: torch.Tensor, what: str, device, shape, dtype=torch.int32) -> None:
    if _device(t, what) != device:
        raise ValueError(f"{what}: on {t.device}, the others on {device}")
    if t.dtype != dtype:
        raise TypeError(f"{what}: {dtype} is wanted, got {t.dtype}")
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous tensor of shape {tuple(shape)} is wanted, got {tuple(t.shape)}, strides {t.stride()}")


def _mx4(m: Mx4, what: str, dims: int) -> tuple[torch.device, int, int]:
    """(device, rows, K) of checked MXFP4 rows with `dims` dimensions."""
    if not isinstance(m, Mx4):
        raise TypeError(f"{what}: Mx4 is wanted, got {type(m).__name__}")
    codes, scales = m
    d = _device(codes, what + ".codes")
    if codes.dtype != torch.uint8:
        raise TypeError(f"{what}.codes: uint8 is wanted, got {codes.dtype}")
    if codes.dim() != dims or not codes.is_contiguous():
        raise ValueError(f"{what}.codes: a contiguous tensor of {dims} dimensions is wanted, got {tuple(codes.shape)}")
    rows, k = codes.shape[-2], codes.shape[-1] * 2
    _k(k, what)
    _ints(scales, what + ".scales", d, tuple(codes.shape[:-2]) + (-(-k // 256), rows, 8), torch.uint8)
    return d, rows, k


def _k(k: int, what: str) -> None:
    if k <= 0 or k % 32:
        raise ValueError(f"{what}: rows of a multiple of 32 elements are wanted, got {k}")


def _plan(plan: MoePlan, device) -> tuple[int, int, int]:
    """(T, used, n_expert) of a checked plan."""
    if not isinstance(plan, MoePlan):
        raise TypeError(f"plan: MoePlan is wanted, got {type(plan).__name__}")
    order, rank, offsets = plan
    if not isinstance(rank, torch.Tensor) or rank.dim() != 2 or not isinstance(offsets, torch.Tensor) or offsets.dim() != 1:
        raise ValueError("plan: rank [T, used] and offsets [n_expert + 1] are wanted")
    t, used = rank.shape
    n_expert = offsets.shape[0] - 1
    _routing(used, n_expert)
    _ints(rank, "plan.rank", device, (t, used))
    _ints(order, "plan.order", device, (t * used,))
    _ints(offsets, "plan.offsets", device, (n_expert + 1,))
    return t, used, n_expert


def _routing(used: int, n_expert: int) -> None:
    if not 1 <= used <= MAX_USED:
        raise ValueError(f"1 to {MAX_USED} slots per token are supported, got {used}")
    if not 1 <= n_expert <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts are supported, got {n_expert}")


def _type(dtype, what: str) -> int:
    if dtype not in _TYPE:
        raise TypeError(f"{what}: float32, float16 or bfloat16 is wanted, got {dtype}")
    return _TYPE[dtype]


def _call(name: str, device: torch.device, *args) -> None:
    """Launches on the current stream of `device`, whatever device is current."""
    f = getattr(_lib or library(), name)
    # the default stream's handle is 0, which the flat ABI takes for a private stream: it has a value of its own there
    stream = torch.cuda.current_stream(device).cuda_stream or 1
    if device.index == torch.cuda.current_device():
        rc = f(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = f(*args, stream)
    if rc:
        kind, text = _ERRORS.get(rc, (RuntimeError, "error"))
        raise kind(f"{name}: {text} ({rc})")


# ---- MXFP4 ---------------------------------------------------------------------------------------
def mx4_quantize(x: torch.Tensor) -> Mx4:
    """x [rows, K] -> MXFP4: per 32 elements the exponent floor(log2 max|x|) - 2, elements rounded to
    nearest even, at most 6.  A block that holds an infinity or a NaN becomes NaN."""
    d = _matrix(x, "x")
    rows, k = x.shape
    _k(k, "x")
    codes = torch.empty((rows, k // 2), dtype=torch.uint8, device=d)
    scales = torch.empty((-(-k // 256), rows, 8), dtype=torch.uint8, device=d)
    _call("mi355x_mx4_quantize", d, _TYPE[x.dtype], x.data_ptr(), x.stride(0), rows, k, codes.data_ptr(), scales.data_ptr())
    return Mx4(codes, scales)


def mx4_dequantize(m: Mx4, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [rows, K] that MXFP4 rows stand for, rounded to `dtype` (exact in float32)."""
    d, rows, k = _mx4(m, "m", 2)
    y = torch.empty((rows, k), dtype=dtype, device=d)
    _call("mi355x_mx4_dequantize", d, m.codes.data_ptr(), m.scales.data_ptr(), rows, k, _type(dtype, "dtype"), y.data_ptr())
    return y


def _operand(x, what: str, device, k: int, rows: int | None):
    """(type, pointer, scales' pointer, row stride, rows, the workspace to keep) of a product's x."""
    if isinstance(x, Mx4):
        d, n, kx = _mx4(x, what, 2)
        args = (_MX4, x.codes.data_ptr(), x.scales.data_ptr(), kx)
        work = None
    else:
        d = _matrix(x, what)
        n, kx = x.shape
        args = (_TYPE[x.dtype], x.data_ptr(), None, x.stride(0))
        work = torch.empty(-(-n * k // 512) * 256 + -(-k // 256) * n * 8, dtype=torch.uint8, device=d)
    if d != device:
        raise ValueError(f"{what}: on {d}, the weights on {device}")
    if kx != k or (rows is not None and n != rows):
        raise ValueError(f"{what}: shape {[rows if rows is not None else 'rows', k]} is wanted, got {[n, kx]}")
    return args, n, work


def _out_dtype(x, dtype):
    return dtype if dtype is not None else torch.float32 if isinstance(x, Mx4) else x.dtype


def mx4_mul_mat(w: Mx4, x, dtype: torch.dtype | None = None) -> torch.Tensor:
    """y [T, M] = x [T, K] . w [M, K]^T.  x: MXFP4 rows, or float rows that are quantised to MXFP4
    within the call.  float32 sums, rounded once to `dtype` (x's own; float32 for MXFP4 rows)."""
    d, m, k = _mx4(w, "w", 2)
    args, t, work = _operand(x, "x", d, k, None)
    dtype = _out_dtype(x, dtype)
    ytype = _type(dtype, "dtype")
    y = torch.empty((t, m), dtype=dtype, device=d)
    _call("mi355x_mx4_mul_mat", d, w.codes.data_ptr(), w.scales.data_ptr(), m, k, *args, t, ytype, y.data_ptr(),
          work.data_ptr() if work is not None else None, work.numel() if work is not None else 0)
    return y


def mx4_mul_mat_id(w: Mx4, x, plan: MoePlan, x_sorted: bool = False, dtype: torch.dtype | None = None) -> torch.Tensor:
    """y [T * used, M]: row p is w[e] times x's row for the pairs p of expert e, in the plan's order,
    zero behind the last.  w holds MXFP4 [n_expert, M, K].  x, as in mx4_mul_mat: [T, K], a row per
    token, or with x_sorted [T * used, K], rows in the plan's order already."""
    d, m, k = _mx4(w, "w", 3)
    t, used, n_expert = _plan(plan, d)
    if w.codes.shape[0] != n_expert:
        raise ValueError(f"w: {w.codes.shape[0]} experts, the plan has {n_expert}")
    args, _, work = _operand(x, "x", d, k, t * used if x_sorted else t)
    dtype = _out_dtype(x, dtype)
    ytype = _type(dtype, "dtype")
    y = torch.empty((t * used, m), dtype=dtype, device=d)
    _call("mi355x_mx4_mul_mat_id", d, w.codes.data_ptr(), w.scales.data_ptr(), m, k, n_expert, *args, t, used,
          1 if x_sorted else 0, plan.order.data_ptr(), plan.offsets.data_ptr(), ytype, y.data_ptr(),
          work.data_ptr() if work is not None else None, work.numel() if work is not None else 0)
    return y


# ---- routing -------------------------------------------------------------------------------------
def moe_sort(ids: torch.Tensor, n_expert: int) -> MoePlan:
    """The pairs of ids [T, used] (int32 or int64) sorted by expert, stably.  An id outside
    0 .. n_expert - 1 (a padded token's -1) belongs to no expert."""
    d = _device(ids, "ids")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids: int32 or int64 is wanted, got {ids.dtype}")
    if ids.dim() != 2 or not ids.is_contiguous():
        raise ValueError(f"ids: a contiguous [T, used] tensor is wanted, got {tuple(ids.shape)}, strides {ids.stride()}")
    t, used = ids.shape
    _routing(used, n_expert)
    order = torch.empty(t * used, dtype=torch.int32, device=d)
    rank = torch.empty((t, used), dtype=torch.int32, device=d)
    offsets = torch.empty(n_expert + 1, dtype=torch.int32, device=d)
    size = library().mi355x_moe_sort_workspace(t, used, n_expert)
    work = torch.empty(size, dtype=torch.uint8, device=d) if size > 0 else None
    _call("mi355x_moe_sort", d, ids.data_ptr(), ids.element_size(), t, used, n_expert, order.data_ptr(), rank.data_ptr(),
          offsets.data_ptr(), work.data_ptr() if work is not None else None, size)
    return MoePlan(order, rank, offsets)


def moe_gather(x: torch.Tensor, plan: MoePlan) -> torch.Tensor:
    """xs [T * used, D]: x [T, D]'s rows in the plan's order, zero behind the last expert's."""
    d = _matrix(x, "x")
    t, used, _ = _plan(plan, d)
    if x.shape[0] != t:
        raise ValueError(f"x: {x.shape[0]} rows, the plan has {t} tokens")
    xs = torch.empty((t * used, x.shape[1]), dtype=x.dtype, device=d)
    _call("mi355x_moe_gather", d, _TYPE[x.dtype], x.data_ptr(), x.stride(0), t, x.shape[1], used, plan.order.data_ptr(),
          plan.rank.data_ptr(), xs.data_ptr())
    return xs


def _weights(w: torch.Tensor, device, shape) -> None:
    _ints(w, "weights", device, shape, torch.float32)
    if w.requires_grad and torch.is_grad_enabled():
        raise ValueError("weights: no gradient is recorded here; pass a detached tensor")


def moe_combine(ys: torch.Tensor, plan: MoePlan, weights: torch.Tensor | None = None) -> torch.Tensor:
    """y [T, D] = sum over slots of weights[t, j] * ys[rank[t, j]], float32 sums in slot order.  Slots
    without an expert add nothing, whatever their weight holds.  Without weights: the gather's gradient."""
    d = _matrix(ys, "ys")
    t, used, _ = _plan(plan, d)
    if ys.shape[0] != t * used:
        raise ValueError(f"ys: {ys.shape[0]} rows, the plan has {t * used} pairs")
    if weights is not None:
        _weights(weights, d, (t, used))
    y = torch.empty((t, ys.shape[1]), dtype=ys.dtype, device=d)
    _call("mi355x_moe_combine", d, _TYPE[ys.dtype], ys.data_ptr(), ys.stride(0), t, ys.shape[1], used, plan.rank.data_ptr(),
          weights.data_ptr() if weights is not None else None, y.data_ptr())
    return y


def moe_combine_back(dy: torch.Tensor, ys: torch.Tensor, plan: MoePlan, weights: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The combine's gradient: (dys [T * used, D] = weights[t, j] * dy[t] at rank[t, j], zero behind the
    last expert's; dweights [T, used] float32 = dy[t] . ys[rank[t, j]], zero without an expert)."""
    d = _matrix(ys, "ys")
    t, used, _ = _plan(plan, d)
    if ys.shape[0] != t * used:
        raise ValueError(f"ys: {ys.shape[0]} rows, the plan has {t * used} pairs")
    _matrix(dy, "dy", d, (t, ys.shape[1]))
    if dy.dtype != ys.dtype:
        raise TypeError(f"dy: {ys.dtype} is wanted, as ys has, got {dy.dtype}")
    _weights(weights, d, (t, used))
    dys = torch.empty((t * used, ys.shape[1]), dtype=ys.dtype, device=d)
    dw = torch.empty((t, used), dtype=torch.float32, device=d)
    _call("mi355x_moe_combine_back", d, _TYPE[ys.dtype], dy.data_ptr(), dy.stride(0), ys.data_ptr(), ys.stride(0), t, ys.shape[1],
          used, plan.order.data_ptr(), plan.rank.data_ptr(), weights.data_ptr(), dys.data_ptr(), dw.data_ptr())
    return dys, dw
