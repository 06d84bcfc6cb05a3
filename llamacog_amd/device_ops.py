"""MXFP4 products and expert routing on torch tensors of an MI355X: the operators of
include/ggml-mi355x.h that need no ggml graph, called on device memory in place.

Every function launches on torch's current stream of its tensors' device and returns without
waiting; nothing is kept between calls, and a call may be captured into a graph.  Arguments are
checked on the host (ValueError, TypeError); what depends on values on the device is defined
instead: expert ids outside 0 .. n_expert - 1 belong to no expert.  There is no CPU form, and no
gradient is recorded: an input that asks for one, or carries a tangent of forward mode, is refused
(moe_combine_back and, for moe_gather, moe_combine are the gradients).

    plan = moe_sort(ids, n_expert)                       # ids [T, used] from the router
    h = mx4_mul_mat_id(w_up, x, plan)                    # [T * used, F], rows sorted by expert
    y = mx4_mul_mat_id(w_down, act(h), plan, x_sorted=True)
    out = moe_combine(y, plan, weights)                  # [T, D]
"""
from __future__ import annotations

import ctypes
import glob
import importlib.util
import os
import sys
from typing import NamedTuple


def _hip_runtimes() -> set[str]:
    with open("/proc/self/maps") as maps:
        return {os.path.realpath(line.split()[-1]) for line in maps if "libamdhip64" in line}


def _refuse(runtimes: set[str]):
    raise ImportError("two HIP runtimes in this process: import llamacog_amd.device_ops (or torch) before the plugin is loaded: "
                      + ", ".join(sorted(runtimes)))


# torch brings a HIP runtime of its own.  The plugin, loaded later, uses that one too; loaded before, it
# has brought the system's, and two runtimes in a process do not know of each other's work (and may abort it
# at its end): torch is not imported then.
if "torch" not in sys.modules and _hip_runtimes():
    _torch = importlib.util.find_spec("torch")
    _own = {os.path.realpath(f) for d in (_torch.submodule_search_locations if _torch else ())
            for f in glob.glob(os.path.join(d, "lib", "libamdhip64.so*"))}
    if _own and not _own & _hip_runtimes():
        _refuse(_own | _hip_runtimes())

import torch  # noqa: E402

from . import PKG, BackendMissing  # noqa: E402

LIBRARY = os.path.join(PKG, "libmi355x-ops.so")   # the flat ABI
BINDING = os.path.join(PKG, "_device_ops.so")     # csrc/devops_torch.cpp


def library() -> ctypes.CDLL:
    """libmi355x-ops.so, the flat ABI that include/ggml-mi355x.h declares; BackendMissing if it is not built."""
    if not os.path.exists(LIBRARY):
        raise BackendMissing(f"operators not built: {LIBRARY} is missing (run __graft_entry__.build())")
    return ctypes.CDLL(LIBRARY)


if not os.path.exists(BINDING):
    raise BackendMissing(f"operators not built: {BINDING} is missing (run __graft_entry__.build())")
from . import _device_ops as _ops  # noqa: E402

if len(_hip_runtimes()) > 1:
    _refuse(_hip_runtimes())


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


def _is(v, kind, what: str):
    if not isinstance(v, kind):
        raise TypeError(f"{what}: {kind.__name__} is wanted, got {type(v).__name__}")
    return v


# ---- MXFP4 ---------------------------------------------------------------------------------------
def mx4_quantize(x: torch.Tensor) -> Mx4:
    """x [rows, K] -> MXFP4: per 32 elements the exponent floor(log2 max|x|) - 2, elements rounded to
    nearest even, at most 6.  A block that holds an infinity or a NaN becomes NaN.  K is a multiple of
    32; x float32, float16 or bfloat16, its rows any distance apart, as everywhere here."""
    return Mx4(*_ops.quantize(x))


def mx4_dequantize(m: Mx4, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [rows, K] that MXFP4 rows stand for, rounded to `dtype` (exact in float32, but for those past its
    largest number, which are infinite: 2 and more under the exponent byte 254, 4 and more under 253)."""
    return _ops.dequantize(*_is(m, Mx4, "m"), dtype)


def mx4_mul_mat(w: Mx4, x, dtype: torch.dtype | None = None) -> torch.Tensor:
    """y [T, M] = x [T, K] . w [M, K]^T.  x: MXFP4 rows, or float rows that are quantised to MXFP4
    within the call.  float32 sums, rounded once to `dtype` (x's own; float32 for MXFP4 rows)."""
    codes, scales = x if isinstance(x, Mx4) else (x, None)
    return _ops.mul_mat(*_is(w, Mx4, "w"), codes, scales, dtype)


def mx4_mul_mat_id(w: Mx4, x, plan: MoePlan, x_sorted: bool = False, dtype: torch.dtype | None = None) -> torch.Tensor:
    """y [T * used, M]: row p is w[e] times x's row for the pairs p of expert e, in the plan's order,
    zero behind the last.  w holds MXFP4 [n_expert, M, K].  x, as in mx4_mul_mat: [T, K], a row per
    token, or with x_sorted [T * used, K], rows in the plan's order already."""
    codes, scales = x if isinstance(x, Mx4) else (x, None)
    return _ops.mul_mat_id(*_is(w, Mx4, "w"), codes, scales, *_is(plan, MoePlan, "plan"), x_sorted, dtype)


# ---- routing -------------------------------------------------------------------------------------
def moe_sort(ids: torch.Tensor, n_expert: int) -> MoePlan:
    """The pairs of ids [T, used] (int32 or int64, used up to 16) sorted by expert (up to 1024), stably.
    An id outside 0 .. n_expert - 1 (a padded token's -1) belongs to no expert."""
    return MoePlan(*_ops.sort(ids, n_expert))


def moe_gather(x: torch.Tensor, plan: MoePlan) -> torch.Tensor:
    """xs [T * used, D]: x [T, D]'s rows in the plan's order, zero behind the last expert's."""
    return _ops.gather(x, *_is(plan, MoePlan, "plan"))


def moe_combine(ys: torch.Tensor, plan: MoePlan, weights: torch.Tensor | None = None) -> torch.Tensor:
    """y [T, D] = sum over slots of weights[t, j] * ys[rank[t, j]], float32 sums in slot order.  Slots
    without an expert add nothing, whatever their weight holds.  Without weights: the gather's gradient."""
    return _ops.combine(ys, *_is(plan, MoePlan, "plan"), weights)


def moe_combine_back(dy: torch.Tensor, ys: torch.Tensor, plan: MoePlan, weights: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The combine's gradient: (dys [T * used, D] = weights[t, j] * dy[t] at rank[t, j], zero behind the
    last expert's; dweights [T, used] float32 = dy[t] . ys[rank[t, j]], zero without an expert)."""
    return _ops.combine_back(dy, ys, *_is(plan, MoePlan, "plan"), weights)
