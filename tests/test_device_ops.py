"""The operators on device tensors (llamacog_amd.device_ops): MXFP4 quantisation and products, expert
sort, gather, combine and their gradients, against plain numpy in 64 bits.

Tolerances are bounds, not fits.  Quantisation, values, sorting and gathering are exact.  A product
adds K products of at most 4 significant bits each (exact in float32) in some order: each of fewer
than K additions rounds by at most 2^-24 of a partial sum that sum |w x| bounds, hence
K 2^-24 sum |w x|, and the result is rounded once to y's type (half a step: eps / 2).  A combine adds
`used` rounded products: (2 used) 2^-24 sum |w y|, and so on."""
import ctypes
import os
import re
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

import llamacog_amd as la
from llamacog_amd import device_ops as ops

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
U32 = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def least_step(t):
    """Half a step below the normal range, where steps stop shrinking: a rounding to t there is off by
    at most this, however small the number (float16: 2^-25)."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


# ---- plain forms ---------------------------------------------------------------------------------
def np_quantize(x):
    """float64 [rows, K] -> (codes [rows, K], exponent bytes [rows, K / 32])."""
    b = x.reshape(x.shape[0], -1, 32)
    top = np.abs(b).max(-1)
    finite = np.isfinite(b).all(-1)
    safe = np.where(finite & (top > 0), top, 1.0)
    e = np.clip(np.where(top > 0, np.frexp(safe)[1] - 3, -127), -127, 127)
    with np.errstate(invalid="ignore"):
        a = np.abs(b) * np.exp2(-e.astype(np.float64))[..., None]
        r = np.where(a < 2, np.rint(a * 2) / 2, np.where(a < 4, np.rint(a), np.rint(a / 2) * 2))
    r = np.where(finite[..., None], np.minimum(r, 6), 0)
    code = np.where(r < 2, r * 2, np.where(r < 4, r + 2, r / 2 + 4)).astype(np.uint8)
    code |= ((np.signbit(b) & finite[..., None]).astype(np.uint8) << 3)
    return code.reshape(x.shape), np.where(finite, e + 127, 255).astype(np.uint8)


def np_values(code, e):
    s = np.where(e == 255, np.nan, np.exp2(e.astype(np.float64) - 127))
    return (GRID[code].reshape(*e.shape, 32) * s[..., None]).reshape(code.shape)


def np_rounded(x):
    return np_values(*np_quantize(x))


def pack(code, e):
    """codes and exponent bytes [..., rows, *] -> Mx4 on the GPU; the bytes past K hold rubbish."""
    rows, nb = e.shape[-2:]
    planes = np.full(e.shape[:-1] + (-(-nb // 8) * 8,), 0xFF, np.uint8)
    planes[..., :nb] = e
    planes = np.moveaxis(planes.reshape(e.shape[:-1] + (-1, 8)), -2, -3)
    both = code[..., 0::2] | (code[..., 1::2] << 4)
    return ops.Mx4(torch.from_numpy(np.ascontiguousarray(both)).cuda(), torch.from_numpy(np.ascontiguousarray(planes)).cuda())


def unpack(m):
    c, s = m.codes.cpu().numpy(), m.scales.cpu().numpy()
    code = np.stack((c & 15, c >> 4), -1).reshape(*c.shape[:-1], -1)
    e = np.moveaxis(s, -3, -2).reshape(*s.shape[:-3], s.shape[-2], -1)[..., : code.shape[-1] // 32]
    return code, e


def random_mx4(rng, *shape):
    """Random codes and exponents of a few octaves: (Mx4, values in 64 bits)."""
    code = rng.integers(0, 16, shape, dtype=np.uint8)
    e = rng.integers(120, 130, shape[:-1] + (shape[-1] // 32,), dtype=np.uint8)
    return pack(code, e), np_values(code, e)


def rows_of(rng, rows, k, dtype):
    x = torch.from_numpy(rng.standard_normal((rows, k)) * (1 + 8 * (rng.random(k) < 0.02))).to(dtype).cuda()
    return x, x.double().cpu().numpy()


def check_product(y, w, x, dtype, what=""):
    """y against x w^T in 64 bits within the bound of the docstring."""
    got, want = y.double().cpu().numpy(), x @ w.T
    room = np.abs(x) @ np.abs(w).T * w.shape[1] * U32
    off = np.abs(got - want) - room - half_step(dtype) * (np.abs(want) + room) - least_step(dtype)
    assert not np.isnan(got).any() and off.max(initial=-1) <= 0, f"{what}: off by {off.max():.3g} more than the bound"


def np_sort(ids, n_expert):
    flat = ids.reshape(-1)
    held = [(e, p) for p, e in enumerate(flat) if 0 <= e < n_expert]
    order = [p for _, p in sorted(held)]
    rank = np.full(flat.shape, -1, np.int32)
    rank[order] = np.arange(len(order))
    offsets = np.searchsorted(np.sort(np.array([e for e, _ in held], int)), np.arange(n_expert + 1))
    return np.array(order + [-1] * (flat.size - len(order)), np.int32), rank.reshape(ids.shape), offsets.astype(np.int32)


def routing(rng, t, used, n_expert, kind):
    if kind == "one":        # everything to one expert
        return np.full((t, used), n_expert - 1)
    if kind == "none":       # padding only
        return np.full((t, used), -1)
    ids = rng.integers(0, n_expert, (t, used))   # the same expert twice for a token now and then
    if kind == "holes":
        ids[rng.random((t, used)) < 0.3] = -1
        ids[rng.random((t, used)) < 0.1] = n_expert
        ids[-max(1, t // 4):] = -7
    return ids


# ---- without a GPU -------------------------------------------------------------------------------
def test_library_exports_what_the_header_declares():
    text = re.sub(r"//.*", "", open(os.path.join(la.REPO, "include", "ggml-mi355x.h")).read())
    names = set(re.findall(r"\bmi355x_(?:mx4|moe)_\w+(?=\s*\()", text))
    assert names == set(SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", ops.LIBRARY], capture_output=True, text=True, check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert exported == names   # nothing else, so that the plugin's copy of the kernels stays apart
    assert b"gfx950" in open(ops.LIBRARY, "rb").read()


@pytest.mark.parametrize("compiler,language", [("gcc", "c"), ("g++", "c++")])
def test_header_stands_alone(tmp_path, compiler, language):
    src = tmp_path / "t"
    src.write_text('#include "ggml-mi355x.h"\nint main(void) { return mi355x_moe_sort_workspace(1, 1, 1) != 0; }\n')
    subprocess.run([compiler, "-x", language, "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(la.REPO, "include"), str(src)],
                   check=True)


P, I, L = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
SIGNATURES = {
    "mi355x_mx4_quantize": [I, P, L, L, L, P, P, P],
    "mi355x_mx4_dequantize": [P, P, L, L, I, P, P],
    "mi355x_mx4_mul_mat": [P, P, L, L, I, P, P, L, L, I, P, P, L, P],
    "mi355x_mx4_mul_mat_id": [P, P, L, L, L, I, P, P, L, L, L, I, P, P, I, P, P, L, P],
    "mi355x_moe_sort": [P, I, L, L, L, P, P, P, P, L, P],
    "mi355x_moe_gather": [I, P, L, L, L, L, P, P, P, P],
    "mi355x_moe_combine": [I, P, L, L, L, L, P, P, P, P],
    "mi355x_moe_combine_back": [I, P, L, P, L, L, L, L, P, P, P, P, P, P],
    "mi355x_mx4_scales_bytes": [L, L],
    "mi355x_mx4_mul_mat_workspace": [L, L, I, L],
    "mi355x_mx4_mul_mat_id_workspace": [L, L, L, I, L, L, I],
    "mi355x_moe_sort_workspace": [L, L, L],
}


def flat(name):
    f = getattr(ops.library(), name)
    f.argtypes, f.restype = SIGNATURES[name], L if name.endswith(("_bytes", "_workspace")) else I
    return f


A = 1 << 20   # an aligned address that no call below gets to read

REFUSED = [
    ("mi355x_mx4_quantize", (2, A, 64, 3, 64, A, A), -1),                # type
    ("mi355x_mx4_quantize", (0, A, 64, 3, 48, A, A), -2),                # K not of whole blocks
    ("mi355x_mx4_quantize", (0, A, 64, 3, 0, A, A), -2),
    ("mi355x_mx4_quantize", (0, A, 64, -1, 64, A, A), -2),
    ("mi355x_mx4_quantize", (0, A, 32, 3, 64, A, A), -2),                # rows that overlap
    ("mi355x_mx4_quantize", (0, A, 64, 3, 1 << 25, A, A), -2),
    ("mi355x_mx4_quantize", (0, A, 64, 1 << 31, 64, A, A), -2),
    ("mi355x_mx4_quantize", (0, A + 2, 64, 3, 64, A, A), -3),
    ("mi355x_mx4_quantize", (1, A, 64, 3, 64, A + 8, A), -3),
    ("mi355x_mx4_quantize", (1, A, 64, 3, 64, A, A + 4), -3),
    ("mi355x_mx4_dequantize", (A, A, 3, 64, 39, A), -1),
    ("mi355x_mx4_dequantize", (A, A, 3, 40, 0, A), -2),
    ("mi355x_mx4_dequantize", (A, A, 3, 64, 0, A + 2), -3),
    ("mi355x_mx4_mul_mat", (A, A, 8, 64, 12, A, None, 64, 3, 0, A, A, 1 << 20), -1),
    ("mi355x_mx4_mul_mat", (A, A, 8, 64, 0, A, None, 64, 3, 8, A, A, 1 << 20), -1),
    ("mi355x_mx4_mul_mat", (A, A, 8, 65, 0, A, None, 64, 3, 0, A, A, 1 << 20), -2),
    ("mi355x_mx4_mul_mat", (A, A, 8, 64, 0, A, None, 63, 3, 0, A, A, 1 << 20), -2),
    ("mi355x_mx4_mul_mat", (A + 1, A, 8, 64, 0, A, None, 64, 3, 0, A, A, 1 << 20), -3),
    ("mi355x_mx4_mul_mat", (A, A, 8, 64, -4, A, A + 2, 64, 3, 0, A, None, 0), -3),
    ("mi355x_mx4_mul_mat", (A, A, 8, 64, 0, A, None, 64, 3, 0, A, A, 100), -4),
    ("mi355x_mx4_mul_mat_id", (A, A, 8, 64, 0, 0, A, None, 64, 3, 2, 0, A, A, 0, A, A, 1 << 20), -2),
    ("mi355x_mx4_mul_mat_id", (A, A, 8, 64, 1025, 0, A, None, 64, 3, 2, 0, A, A, 0, A, A, 1 << 20), -2),
    ("mi355x_mx4_mul_mat_id", (A, A, 8, 64, 4, 0, A, None, 64, 3, 17, 0, A, A, 0, A, A, 1 << 20), -2),
    ("mi355x_mx4_mul_mat", (A, A, 640, 14336, -4, A, A, 0, 100, 0, A, A, 100 * 640 * 4), -4),
    ("mi355x_mx4_mul_mat_id", (A, A, 8, 64, 4, 0, A, None, 64, 30, 2, 1, A, A, 0, A, A, 2000), -4),
    ("mi355x_moe_sort", (A, 4, 3, 0, 4, A, A, A, None, 0), -2),
    ("mi355x_moe_sort", (A, 4, 1 << 30, 2, 4, A, A, A, None, 0), -2),
    ("mi355x_moe_sort", (A, 2, 3, 2, 4, A, A, A, None, 0), -1),
    ("mi355x_moe_sort", (A + 4, 8, 3, 2, 4, A, A, A, None, 0), -3),
    ("mi355x_moe_sort", (A, 4, 1 << 20, 2, 4, A, A, A, None, 0), -4),
    ("mi355x_moe_gather", (0, A, 8, 3, 9, 2, A, A, A), -2),
    ("mi355x_moe_gather", (0, A + 1, 9, 3, 9, 2, A, A, A), -3),
    ("mi355x_moe_combine", (5, A, 9, 3, 9, 2, A, A, A), -1),
    ("mi355x_moe_combine", (0, A, 9, 3, -1, 2, A, A, A), -2),
    ("mi355x_moe_combine_back", (0, A, 8, A, 9, 3, 9, 2, A, A, A, A, A), -2),
    ("mi355x_moe_combine_back", (0, A, 9, A, 9, 3, 9, 2, A, A, None, A, A), -2),
    ("mi355x_moe_combine_back", (1, A, 9, A, 9, 3, 9, 2, A, A, A, A + 1, A), -3),
]


N = None
REFUSED += [(n, a, -2) for n, a in [
    ("mi355x_mx4_quantize", (0, N, 64, 3, 64, A, A)), ("mi355x_mx4_quantize", (0, A, 64, 3, 64, N, A)),
    ("mi355x_mx4_quantize", (0, A, 64, 3, 64, A, N)), ("mi355x_mx4_dequantize", (A, N, 3, 64, 0, A)),
    ("mi355x_mx4_dequantize", (A, A, 3, 64, 0, N)), ("mi355x_mx4_mul_mat", (N, A, 8, 64, 0, A, N, 64, 3, 0, A, A, 1 << 20)),
    ("mi355x_mx4_mul_mat", (A, A, 8, 64, -4, A, N, 64, 3, 0, A, A, 1 << 20)), ("mi355x_mx4_mul_mat", (A, A, 8, 64, 0, A, N, 64, 3, 0, N, A, 1 << 20)),
    ("mi355x_mx4_mul_mat_id", (A, A, 8, 64, 4, 0, A, N, 64, 3, 2, 0, N, A, 0, A, A, 1 << 20)),
    ("mi355x_mx4_mul_mat_id", (A, A, 8, 64, 4, 0, A, N, 64, 3, 2, 0, A, N, 0, A, A, 1 << 20)),
    ("mi355x_moe_sort", (N, 4, 3, 2, 4, A, A, A, N, 0)), ("mi355x_moe_sort", (A, 4, 3, 2, 4, A, A, N, N, 0)), ("mi355x_moe_sort", (N, 4, 0, 2, 4, N, N, N, N, 0)),
    ("mi355x_moe_gather", (0, A, 9, 3, 9, 2, N, A, A)), ("mi355x_moe_combine", (0, A, 9, 3, 9, 2, N, A, A)),
    ("mi355x_moe_combine_back", (0, A, 9, A, 9, 3, 9, 2, A, A, A, A, N)),
]]
REFUSED += [("mi355x_mx4_mul_mat", (A, A, 8, 64, 0, A, N, 64, 3, 0, A, N, 1 << 20), -4), ("mi355x_moe_sort", (A, 4, 1 << 20, 2, 4, A, A, A, N, 1 << 30), -4)]

# sizes whose product passes 64 bits
REFUSED += [(n, a, -2) for n, a in [
    ("mi355x_moe_sort", (A, 4, 1 << 62, 4, 4, A, A, A, N, 0)), ("mi355x_moe_gather", (0, A, 9, 1 << 62, 9, 4, A, A, A)),
    ("mi355x_moe_combine", (0, A, 9, 1 << 60, 9, 16, A, A, A)), ("mi355x_moe_combine_back", (0, A, 9, A, 9, 1 << 61, 9, 8, A, A, A, A, A)),
    ("mi355x_mx4_mul_mat_id", (A, A, 8, 64, 4, 0, A, N, 64, 1 << 62, 4, 1, A, A, 0, A, A, 1 << 20)),
    ("mi355x_moe_gather", (0, A, 9, 3, 9, (1 << 62) + 2, A, A, A)),
]]
# integers and weights that lie between elements
REFUSED += [(n, a, -3) for n, a in [
    ("mi355x_moe_sort", (A, 4, 3, 2, 4, A + 2, A, A, N, 0)), ("mi355x_moe_sort", (A, 4, 3, 2, 4, A, A + 1, A, N, 0)),
    ("mi355x_moe_sort", (A, 4, 3, 2, 4, A, A, A + 2, N, 0)), ("mi355x_moe_gather", (0, A, 9, 3, 9, 2, A + 2, A, A)),
    ("mi355x_moe_gather", (0, A, 9, 3, 9, 2, A, A + 2, A)), ("mi355x_moe_combine", (1, A, 9, 3, 9, 2, A + 2, A, A)),
    ("mi355x_moe_combine", (1, A, 9, 3, 9, 2, A, A + 2, A)), ("mi355x_moe_combine_back", (1, A, 9, A, 9, 3, 9, 2, A + 2, A, A, A, A)),
    ("mi355x_moe_combine_back", (1, A, 9, A, 9, 3, 9, 2, A, A + 2, A, A, A)), ("mi355x_moe_combine_back", (1, A, 9, A, 9, 3, 9, 2, A, A, A + 2, A, A)),
    ("mi355x_moe_combine_back", (1, A, 9, A, 9, 3, 9, 2, A, A, A, A, A + 2)),
    ("mi355x_mx4_mul_mat_id", (A, A, 8, 64, 4, 0, A, N, 64, 3, 2, 0, A + 2, A, 0, A, A, 1 << 20)),
    ("mi355x_mx4_mul_mat_id", (A, A, 8, 64, 4, 0, A, N, 64, 3, 2, 0, A, A + 2, 0, A, A, 1 << 20)),
]]


@pytest.mark.parametrize("name,args,code", REFUSED, ids=[f"{n[7:]}-{i}" for i, (n, _, _) in enumerate(REFUSED)])
def test_flat_calls_refused_before_any_launch(name, args, code):
    assert flat(name)(*args, None) == code


EMPTY = [
    ("mi355x_mx4_quantize", (0, A, 64, 0, 64, A, A)),
    ("mi355x_mx4_dequantize", (A, A, 0, 64, 0, A)),
    ("mi355x_mx4_mul_mat", (A, A, 8, 64, 0, A, None, 64, 0, 0, A, A, 0)),
    ("mi355x_mx4_mul_mat", (A, A, 0, 64, 0, A, None, 64, 3, 0, A, A, 1 << 20)),
    ("mi355x_mx4_mul_mat_id", (A, A, 8, 64, 4, 0, A, None, 64, 0, 2, 0, A, A, 0, A, A, 0)),
    ("mi355x_moe_gather", (0, A, 9, 0, 9, 2, A, A, A)),
    ("mi355x_moe_combine", (0, A, 9, 3, 0, 2, A, A, A)),
    ("mi355x_moe_combine_back", (0, A, 9, A, 9, 0, 9, 2, A, A, A, A, A)),
]


@pytest.mark.parametrize("name,args", EMPTY, ids=[f"{n[7:]}-{i}" for i, (n, _) in enumerate(EMPTY)])
def test_flat_calls_with_nothing_to_do(name, args):
    assert flat(name)(*args, None) == 0


def test_sizes():
    scales, work, sort = flat("mi355x_mx4_scales_bytes"), flat("mi355x_mx4_mul_mat_workspace"), flat("mi355x_moe_sort_workspace")
    assert scales(3, 288) == 2 * 3 * 8 and scales(3, 289) == -1
    assert work(8, 0, 0, 3) == -1 and work(8, 288, 7, 3) == -1 and work(8, 288, 0, 0) == 0
    assert work(8, 288, 0, 1) == 0                      # quantised where it is used
    assert work(8, 288, 0, 3) == 512 + 256 and work(8, 288, -4, 3) == 0
    assert work(640, 14336, -4, 100) % (100 * 640 * 4) == 0 and work(640, 14336, -4, 100) > 0   # sums of shares of K
    shares = [work(m, k, -4, t) // (m * t * 4) for t, m, k in ((33, 48, 8192), (129, 70, 4128), (100, 17, 2592))]
    assert shares == [16, 4, 0]
    ids = flat("mi355x_mx4_mul_mat_id_workspace")
    assert ids(8, 288, 4, 0, 100, 2, 0) > 0 and ids(8, 288, 0, 0, 100, 2, 0) == -1 and ids(8, 288, 4, 0, 100, 17, 0) == -1
    assert sort(10, 2, 8) == 0 and sort(1, 17, 8) == -1 and sort(1 << 20, 2, 8) > 0


def test_tensors_of_the_host_are_refused():
    x, ids = torch.zeros(2, 64), torch.zeros(2, 2, dtype=torch.int32)
    m = ops.Mx4(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(1, 2, 8, dtype=torch.uint8))
    plan = ops.MoePlan(torch.zeros(4, dtype=torch.int32), ids, torch.zeros(5, dtype=torch.int32))
    for call in (lambda: ops.mx4_quantize(x), lambda: ops.mx4_dequantize(m), lambda: ops.mx4_mul_mat(m, x),
                 lambda: ops.mx4_mul_mat_id(m, x, plan), lambda: ops.moe_sort(ids, 4), lambda: ops.moe_gather(x, plan),
                 lambda: ops.moe_combine(x, plan), lambda: ops.moe_combine_back(x, x, plan, x)):
        with pytest.raises(ValueError, match="on an MI355X is wanted"):
            call()
    with pytest.raises(TypeError):
        ops.mx4_mul_mat(x, x)
    with pytest.raises(TypeError):
        ops.mx4_quantize(np.zeros((2, 64), np.float32))


# ---- MXFP4 ---------------------------------------------------------------------------------------
def special_blocks():
    """Blocks at the edges: zeros, ties, the largest and least numbers, infinities and NaNs."""
    rng = np.random.default_rng(5)
    b = [np.zeros(32), -np.zeros(32), np.full(32, 2.0 ** -149), np.linspace(-6, 6, 32), np.full(32, 7.99), np.full(32, 3.4e38)]
    b.append(np.concatenate(([4.0], (np.arange(31) - 15) * 0.25)))     # ties of every step, kept by the 4
    b.append(np.concatenate(([6.5], (np.arange(31) - 15) * 0.5)))
    b += [rng.standard_normal(32) * 2.0 ** e for e in (-140, -127, -126, -125, -124, -20, 100, 124)]
    for bad in (np.inf, -np.inf, np.nan):
        v = rng.standard_normal(32)
        v[rng.integers(32)] = bad
        b.append(v)
    return np.array(b, np.float32).reshape(1, -1)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_special_blocks(dtype):
    x = torch.from_numpy(special_blocks()).to(dtype)
    code, e = unpack(ops.mx4_quantize(x.cuda()))
    want_code, want_e = np_quantize(x.double().numpy())
    assert (e == want_e).all() and (code == want_code).all()
    for out in TYPES:
        y = ops.mx4_dequantize(ops.mx4_quantize(x.cuda()), out).cpu()
        assert torch.equal(y.nan_to_num(99.0), torch.from_numpy(np_values(code, e)).to(out).nan_to_num(99.0))
        assert torch.equal(y.isnan(), torch.from_numpy(np_values(code, e)).isnan())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 64), (17, 96), (5, 288), (1, 4096), (33, 1056), (257, 2048), (2, 14336)])
def test_quantize(rows, k, dtype):
    rng = np.random.default_rng(rows * k)
    x, x64 = rows_of(rng, rows, k, dtype)
    m = ops.mx4_quantize(x)
    code, e = unpack(m)
    want_code, want_e = np_quantize(x64)
    assert (e == want_e).all() and (code == want_code).all()
    if k % 256:
        assert int(m.scales[-1, :, k // 32 % 8:].sum()) == 0
    assert torch.equal(ops.mx4_dequantize(m).double().cpu(), torch.from_numpy(np_values(code, e)))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("first", [0, 1, 4, 8])
def test_quantize_strided_rows(dtype, first):
    rng = np.random.default_rng(7)
    big, _ = rows_of(rng, 9, 333, dtype)
    x = big[1::2, first:first + 288]
    assert not x.is_contiguous()
    a, b = ops.mx4_quantize(x), ops.mx4_quantize(x.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


PRODUCTS = [(1, 16, 32), (1, 17, 4096), (1, 4096, 544), (2, 5, 64), (3, 33, 288), (15, 64, 256), (16, 16, 512), (17, 100, 2080),
            (31, 257, 1024), (33, 48, 96), (64, 130, 768), (65, 1, 320), (129, 300, 1280), (300, 129, 224), (512, 1000, 576)]


@gpu
@pytest.mark.parametrize("t,m,k", PRODUCTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_product(t, m, k, dtype):
    rng = np.random.default_rng(t * m + k)
    w, w64 = random_mx4(rng, m, k)
    x, x64 = rows_of(rng, t, k, dtype)
    y = ops.mx4_mul_mat(w, x)
    assert y.dtype == dtype and y.shape == (t, m)
    check_product(y, w64, np_rounded(x64), dtype)
    # quantised by the caller, and to another type
    assert torch.equal(ops.mx4_mul_mat(w, ops.mx4_quantize(x), dtype), y)
    check_product(ops.mx4_mul_mat(w, x, torch.float32), w64, np_rounded(x64), torch.float32)


@gpu
@pytest.mark.parametrize("t,m,k", [(33, 48, 8192), (40, 70, 8224), (129, 70, 4128), (64, 300, 14336), (100, 17, 2592), (257, 64, 5120)])
def test_product_in_shares_of_k(t, m, k):
    """Few tiles and a long K: sums of shares joined by a second kernel, a last share that is shorter, and
    a K that is just not cut (test_sizes says which are)."""
    rng = np.random.default_rng(t)
    w, w64 = random_mx4(rng, m, k)
    x, x64 = rows_of(rng, t, k, torch.bfloat16)
    for dtype in TYPES:
        check_product(ops.mx4_mul_mat(w, x, dtype), w64, np_rounded(x64), dtype)


@gpu
@pytest.mark.parametrize("kind", ["even", "holes", "one", "none"])
def test_experts_product_in_shares_of_k(kind):
    assert flat("mi355x_mx4_mul_mat_id_workspace")(33, 8224, 2, -4, 90, 2, 0) > 0
    rng = np.random.default_rng(9)
    ids, order, rank, plan = plan_of(rng, 90, 2, 2, kind)
    held = int((order >= 0).sum())
    w, w64 = random_mx4(rng, 2, 33, 8224)
    x, x64 = rows_of(rng, 90, 8224, torch.float16)
    y = ops.mx4_mul_mat_id(w, x, plan)
    assert (y[held:] == 0).all()
    for e in range(2):
        at = np.flatnonzero(ids.reshape(-1)[order[:held]] == e)
        check_product(y[torch.from_numpy(at).cuda()], w64[e], np_rounded(x64)[order[at] // 2], torch.float16)


@gpu
@pytest.mark.parametrize("t", [1, 5, 100, 400])
def test_product_strided_rows(t):
    rng = np.random.default_rng(t)
    w, _ = random_mx4(rng, 70, 288)
    big, _ = rows_of(rng, 2 * t, 300, torch.float16)
    x = big[::2, 3:291]
    assert torch.equal(ops.mx4_mul_mat(w, x), ops.mx4_mul_mat(w, x.contiguous()))


@gpu
@pytest.mark.parametrize("t,m,k", [(1, 40, 512), (20, 40, 544), (300, 300, 544)])
def test_product_nan_blocks_stay_in_their_row(t, m, k):
    rng = np.random.default_rng(3)
    code, e = rng.integers(0, 16, (m, k), dtype=np.uint8), rng.integers(120, 130, (m, k // 32), dtype=np.uint8)
    e[m // 2, -1] = 255
    x, x64 = rows_of(rng, t, k, torch.float32)
    x[t // 2, 5] = float("inf")
    y = ops.mx4_mul_mat(pack(code, e), x).cpu().numpy()
    nan = np.zeros((t, m), bool)
    nan[t // 2] = nan[:, m // 2] = True
    assert (np.isnan(y) == nan).all()
    x64[t // 2] = 0
    e[m // 2, -1] = 0
    want = np_rounded(x64) @ np_values(code, e).T
    assert np.abs(np.where(nan, 0, y - want)).max() <= 1e-4 * np.abs(want).max()


@gpu
def test_product_extreme_exponents():
    """Exponents that cancel: 2^120 times 2^-120; both so small that the result is zero."""
    code = np.full((4, 64), 2, np.uint8)   # ones
    one = lambda b: (code, np.full((4, 2), b, np.uint8))  # noqa: E731
    big, small = one(247), one(7)
    y = ops.mx4_mul_mat(pack(*big), pack(*small), torch.float32)
    assert (y == 64).all()
    assert (ops.mx4_mul_mat(pack(*small), pack(*small), torch.float32) == 0).all()
    assert (ops.mx4_mul_mat(pack(*big), pack(*big), torch.float32) == float("inf")).all()


# ---- routing -------------------------------------------------------------------------------------
SORTS = [(1, 1, 1), (1, 2, 8), (3, 2, 8), (7, 16, 5), (64, 1, 64), (65, 3, 33), (1000, 4, 256), (511, 8, 1024), (2048, 2, 7),
         (5000, 2, 100), (40000, 4, 1000), (140000, 4, 9)]


@gpu
@pytest.mark.parametrize("t,used,n_expert", SORTS)
@pytest.mark.parametrize("kind", ["even", "holes", "one", "none"])
def test_sort(t, used, n_expert, kind):
    rng = np.random.default_rng(t)
    ids = routing(rng, t, used, n_expert, kind)
    want = np_sort(ids, n_expert)
    for dtype in (torch.int32, torch.int64):
        plan = ops.moe_sort(torch.from_numpy(ids).to(dtype).cuda(), n_expert)
        for got, w in zip(plan, want):
            assert got.dtype == torch.int32 and (got.cpu().numpy() == w).all()


@gpu
def test_sort_of_wide_ids_and_no_tokens():
    ids = torch.tensor([[1 << 32, 1], [-(1 << 32), (1 << 32) + 1]]).cuda()
    plan = ops.moe_sort(ids, 2)
    assert plan.rank.tolist() == [[-1, 0], [-1, -1]] and plan.offsets.tolist() == [0, 0, 1] and plan.order.tolist() == [1, -1, -1, -1]
    plan = ops.moe_sort(ids[:0], 3)
    assert plan.offsets.tolist() == [0, 0, 0, 0] and plan.order.numel() == 0
    assert ops.moe_gather(torch.zeros(0, 8, device="cuda"), plan).shape == (0, 8)
    assert ops.moe_combine(torch.zeros(0, 8, device="cuda"), plan).shape == (0, 8)


ROWS = [(1, 1, 3, 1), (1, 2, 8, 4096), (5, 3, 4, 33), (9, 2, 6, 34), (17, 16, 9, 36), (40, 8, 128, 2048), (130, 1, 3, 257), (300, 4, 8, 1000)]


def plan_of(rng, t, used, n_expert, kind):
    ids = routing(rng, t, used, n_expert, kind)
    order, rank, offsets = np_sort(ids, n_expert)
    return ids, order, rank, ops.MoePlan(*(torch.from_numpy(v).cuda() for v in (order, rank, offsets)))


@gpu
@pytest.mark.parametrize("t,used,n_expert,d", ROWS)
@pytest.mark.parametrize("kind", ["even", "holes", "none"])
@pytest.mark.parametrize("dtype", TYPES)
def test_gather_combine_and_gradients(t, used, n_expert, d, kind, dtype):
    rng = np.random.default_rng(t * d)
    ids, order, rank, plan = plan_of(rng, t, used, n_expert, kind)
    held = int((order >= 0).sum())
    x, x64 = rows_of(rng, t, d, dtype)
    xs = ops.moe_gather(x, plan).double().cpu().numpy()
    assert (xs[:held] == x64[order[:held] // used]).all() and (xs[held:] == 0).all()

    ys, ys64 = rows_of(rng, t * used, d, dtype)
    ys[held:] = float("nan")        # rows and weights of slots without an expert are not looked at
    w = torch.from_numpy(rng.random((t, used), dtype=np.float32)).cuda()
    w[torch.from_numpy(rank < 0).cuda()] = float("inf")
    w64 = np.where(rank < 0, 0, w.double().cpu().numpy())
    rows = np.where((rank >= 0)[..., None], ys64[np.maximum(rank, 0)], 0)
    for weights, f in ((w, w64), (None, np.ones((t, used)))):
        got = ops.moe_combine(ys, plan, weights).double().cpu().numpy()
        want, room = (rows * f[..., None]).sum(1), np.abs(rows * f[..., None]).sum(1) * 2 * used * U32
        assert (np.abs(got - want) <= room + half_step(dtype) * (np.abs(want) + room) + least_step(dtype)).all()

    dy, dy64 = rows_of(rng, t, d, dtype)
    dys, dw = ops.moe_combine_back(dy, ys, plan, w)
    want = np.zeros((t * used, d))
    want[:held] = w64.reshape(-1)[order[:held], None] * dy64[order[:held] // used]
    got = dys.double().cpu().numpy()
    assert (np.abs(got - want) <= (U32 + half_step(dtype) * (1 + U32)) * np.abs(want) + least_step(dtype)).all() and (got[held:] == 0).all()
    want, room = (rows * dy64[:, None]).sum(-1), np.abs(rows * dy64[:, None]).sum(-1) * (d + 1) * U32
    assert (np.abs(dw.double().cpu().numpy() - want) <= room).all()


@gpu
def test_gradients_against_differences():
    """y is linear in the rows and in the weights: differences of the combine itself, taken in steps of
    powers of two on small whole numbers, are exact."""
    rng = np.random.default_rng(11)
    _, _, rank, plan = plan_of(rng, 6, 3, 4, "holes")
    ys = torch.from_numpy(rng.integers(-8, 9, (18, 5)).astype(np.float32)).cuda()
    w = torch.from_numpy(rng.integers(-8, 9, (6, 3)).astype(np.float32)).cuda()
    dy = torch.from_numpy(rng.integers(-8, 9, (6, 5)).astype(np.float32)).cuda()
    dys, dw = ops.moe_combine_back(dy, ys, plan, w)
    loss = lambda a, b: float((ops.moe_combine(a, plan, b) * dy).sum())  # noqa: E731
    base = loss(ys, w)
    for i in range(18):
        for j in range(5):
            a = ys.clone()
            a[i, j] += 2
            assert loss(a, w) - base == 2 * float(dys[i, j])
    for i in range(6):
        for j in range(3):
            b = w.clone()
            b[i, j] += 2
            assert loss(ys, b) - base == 2 * float(dw[i, j])
    x = torch.from_numpy(rng.integers(-8, 9, (6, 5)).astype(np.float32)).cuda()
    dx = ops.moe_combine(dys, plan)     # the gather's gradient for a loss of xs . dys
    for i in range(6):
        for j in range(5):
            a = x.clone()
            a[i, j] += 1
            assert float(((ops.moe_gather(a, plan) - ops.moe_gather(x, plan)) * dys).sum()) == float(dx[i, j])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_of_the_routing(dtype):
    rng = np.random.default_rng(2)
    _, _, _, plan = plan_of(rng, 10, 2, 4, "holes")
    big, _ = rows_of(rng, 40, 90, dtype)
    w = torch.rand(10, 2, device="cuda")
    for first, d in ((0, 64), (1, 64), (2, 33), (8, 72)):
        x, ys = big[:20:2, first:first + d], big[::2, first:first + d]
        assert torch.equal(ops.moe_gather(x, plan), ops.moe_gather(x.contiguous(), plan))
        assert torch.equal(ops.moe_combine(ys, plan, w), ops.moe_combine(ys.contiguous(), plan, w))
        for a, b in zip(ops.moe_combine_back(x, ys, plan, w), ops.moe_combine_back(x.contiguous(), ys.contiguous(), plan, w)):
            assert torch.equal(a, b)


# ---- the experts' product ------------------------------------------------------------------------
EXPERTS = [(1, 2, 8, 48, 64), (1, 1, 1, 16, 32), (3, 2, 8, 33, 288), (20, 6, 64, 40, 160), (37, 2, 3, 130, 512), (100, 4, 100, 17, 96),
           (200, 2, 4, 300, 320), (700, 1, 2, 257, 288), (90, 8, 300, 64, 256)]


@gpu
@pytest.mark.parametrize("t,used,n_expert,m,k", EXPERTS)
@pytest.mark.parametrize("kind", ["even", "holes", "one", "none"])
@pytest.mark.parametrize("sorted_rows", [False, True])
def test_experts_product(t, used, n_expert, m, k, kind, sorted_rows):
    rng = np.random.default_rng(t + m)
    dtype = TYPES[(t + m + sorted_rows) % 3]
    ids, order, rank, plan = plan_of(rng, t, used, n_expert, kind)
    held = int((order >= 0).sum())
    w, w64 = random_mx4(rng, n_expert, m, k)
    x, x64 = rows_of(rng, t * used if sorted_rows else t, k, dtype)
    if sorted_rows:
        x[held:] = float("nan")     # rows that no expert takes are not looked at
    y = ops.mx4_mul_mat_id(w, x, plan, x_sorted=sorted_rows)
    assert y.dtype == dtype and y.shape == (t * used, m) and (y[held:] == 0).all()
    xr = np_rounded(x64)
    flat = ids.reshape(-1)
    for e in range(n_expert):
        at = np.flatnonzero(flat[order[:held]] == e)
        rows = at if sorted_rows else order[at] // used
        check_product(y[torch.from_numpy(at).cuda()], w64[e], xr[rows], dtype, f"expert {e}")
    assert torch.equal(ops.mx4_mul_mat_id(w, ops.mx4_quantize(x), plan, sorted_rows, dtype), y)


# ---- together ------------------------------------------------------------------------------------
def expert_layer(x, ids, weights, up, down, n_expert):
    plan = ops.moe_sort(ids, n_expert)
    h = ops.mx4_mul_mat_id(up, x, plan)
    f = h.shape[1] // 2
    h = torch.nn.functional.silu(h[:, :f]) * h[:, f:]
    return ops.moe_combine(ops.mx4_mul_mat_id(down, h, plan, x_sorted=True), plan, weights)


def layer_case(t, seed=1, n_expert=8, used=2, d=512, f=288):
    rng = np.random.default_rng(seed)
    up, up64 = random_mx4(rng, n_expert, 2 * f, d)
    down, down64 = random_mx4(rng, n_expert, d, f)
    x, x64 = rows_of(rng, t, d, torch.float32)
    logits = torch.from_numpy(rng.standard_normal((t, n_expert))).float().cuda()
    weights, ids = torch.topk(torch.softmax(logits, 1), used)
    return (x, ids, weights, up, down, n_expert), (x64, up64, down64)


@gpu
@pytest.mark.parametrize("t", [1, 4, 50, 300])
def test_expert_layer(t):
    """A layer of experts as a model runs it.  The second quantisation rounds what the first product
    left off by float32 sums, so an activation next to a border may fall to either side: the second
    product is checked from the activations that the framework computed."""
    args, (x64, up64, down64) = layer_case(t)
    x, ids, weights, up, down, n_expert = args
    y = expert_layer(*args)
    plan = ops.moe_sort(ids, n_expert)
    h = ops.mx4_mul_mat_id(up, x, plan)
    f = h.shape[1] // 2
    a = torch.nn.functional.silu(h[:, :f]) * h[:, f:]
    ids, rank, w64 = ids.cpu().numpy(), plan.rank.cpu().numpy(), weights.double().cpu().numpy()
    xr, ar = np_rounded(x64), np_rounded(a.double().cpu().numpy())
    want, room = np.zeros_like(x64), np.zeros_like(x64)
    for i in range(t):
        for j in range(2):
            e, p = ids[i, j], rank[i, j]
            check_product(h[p][None], up64[e], xr[i][None], torch.float32)
            one, size = down64[e] @ ar[p], np.abs(down64[e]) @ np.abs(ar[p])
            want[i] += w64[i, j] * one
            room[i] += w64[i, j] * size * (ar.shape[1] + 5) * U32
    assert (np.abs(y.double().cpu().numpy() - want) <= room).all()


@gpu
@pytest.mark.parametrize("t", [1, 40])
def test_expert_layer_in_a_graph(t):
    """Captured once, replayed on new inputs with eager work between; the eager calls agree bit for bit."""
    args, _ = layer_case(t)
    x, ids, weights = (v.clone() for v in args[:3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        expert_layer(x, ids, weights, *args[3:])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = expert_layer(x, ids, weights, *args[3:])
    for seed in range(4):
        fresh, _ = layer_case(t, seed)
        for to, src in zip((x, ids, weights), fresh[:3]):
            to.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, expert_layer(x, ids, weights, *args[3:]))


@gpu
def test_streams_and_repeatability():
    args, _ = layer_case(64)
    want = expert_layer(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([expert_layer(*args) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(want, y) for ys in got for y in ys)


@gpu
def test_two_threads_at_once():
    """Calls from two threads, each on its own stream, give what one call gives."""
    args, _ = layer_case(33)
    want = expert_layer(*args)
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            ys = [expert_layer(*args) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
            got[i] = all(torch.equal(want, y) for y in ys)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got == [True, True]


@gpu
def test_offsets_past_32_bits_in_weights():
    """Codes of 4.6 GB: the last rows of a long matrix and of the last of many experts."""
    m, k = 1_100_000, 8384
    codes = torch.randint(0, 256, (m, k // 2), dtype=torch.uint8, device="cuda")
    scales = torch.randint(120, 130, (-(-k // 256), m, 8), dtype=torch.uint8, device="cuda")
    assert codes.numel() > 1 << 32
    w, end = ops.Mx4(codes, scales), ops.Mx4(codes[-100:].clone(), scales[:, -100:].contiguous())
    for t in (1, 20, 40):
        x = torch.randn(t, k, device="cuda")
        y, want = ops.mx4_mul_mat(w, x), ops.mx4_mul_mat(end, x)
        assert torch.allclose(y[:, -100:], want, rtol=1e-5, atol=float(want.abs().max()) * 1e-5)   # other kernels, other sums
    del w
    n_expert, rows = 1000, 1100
    stack = ops.Mx4(codes.view(n_expert, rows, k // 2), scales.view(n_expert, -(-k // 256), rows, 8))
    ids = torch.tensor([[999, 0], [5, 999], [999, 998]], device="cuda")
    x = torch.randn(3, k, device="cuda")
    plan = ops.moe_sort(ids, n_expert)
    y = ops.mx4_mul_mat_id(stack, x, plan)
    for t, j in ((0, 0), (1, 1), (2, 0), (2, 1)):
        e = int(ids[t, j])
        want = ops.mx4_mul_mat(ops.Mx4(stack.codes[e], stack.scales[e]), x[t:t + 1])
        assert torch.allclose(y[int(plan.rank[t, j])], want[0], rtol=1e-5, atol=float(want.abs().max()) * 1e-5)


@gpu
def test_offsets_past_32_bits_in_rows():
    """2.3 G elements of sorted rows: gathered, combined and back, looked at from the far end."""
    t, used, d = 70_000, 8, 4096
    ids = torch.randint(0, 16, (t, used), dtype=torch.int32, device="cuda")
    plan = ops.moe_sort(ids, 16)
    x = torch.randint(-8, 9, (t, d), device="cuda").to(torch.bfloat16)
    xs = ops.moe_gather(x, plan)
    assert xs.numel() > 1 << 31
    order = plan.order.long()
    for at in (0, t * used - 1000):
        assert torch.equal(xs[at:at + 1000], x[order[at:at + 1000] // used])
    w = torch.randint(-2, 3, (t, used), device="cuda").float()     # small whole numbers: every sum is exact
    y = ops.moe_combine(xs, plan, w)
    assert torch.equal(y[-500:].float(), (x[-500:].float() * w[-500:].sum(1, keepdim=True)).to(torch.bfloat16).float())
    dys, dw = ops.moe_combine_back(x, xs, plan, w)
    assert torch.equal(dw[-500:], (x[-500:].float() ** 2).sum(1, keepdim=True).expand(-1, used))
    at = t * used - 1000
    assert torch.equal(dys[at:], x[order[at:] // used] * w.flatten()[order[at:], None].to(torch.bfloat16))
    q = ops.mx4_quantize(xs)
    end = ops.mx4_quantize(xs[-100:])
    assert torch.equal(q.codes[-100:], end.codes) and torch.equal(q.scales[:, -100:], end.scales)
    assert torch.equal(ops.mx4_dequantize(q, torch.bfloat16)[-100:], ops.mx4_dequantize(end, torch.bfloat16))


def far_rows(t, d, dtype):
    """[t, d] whose rows differ: 1024 random ones over and over, the row's number in the first three columns."""
    torch.cuda.empty_cache()
    x = torch.empty(t, d, dtype=dtype, device="cuda")
    some = torch.randn(1024, d, device="cuda").to(dtype)
    whole = t // 1024 * 1024
    x[:whole].view(-1, 1024, d)[:] = some
    x[whole:] = some[:t - whole]
    n = torch.arange(t, device="cuda")
    for c in range(3):
        x[:, c] = (n >> 8 * c & 255).to(dtype)
    return x


def enough_memory(bytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < bytes:
        pytest.skip(f"{bytes >> 30} GiB of the card's memory are wanted")


@gpu
def test_rows_past_32_bits_of_threads():
    """More tokens than one axis of a launch has workgroups of 256, each with one token's row."""
    t, d = (1 << 24) + 77, 2048
    enough_memory(215 << 30)
    x = far_rows(t, d, torch.bfloat16)
    plan = ops.moe_sort(torch.randint(-1, 3, (t, 1), dtype=torch.int32, device="cuda"), 3)
    rank = plan.rank.view(-1).long()
    xs = ops.moe_gather(x, plan)
    parts = [slice(i, i + (1 << 18)) for i in range(0, t, 1 << 18)]
    for s in parts:
        held = rank[s] >= 0
        assert torch.equal(xs[rank[s][held]], x[s][held])
    assert not xs[int(plan.offsets[-1]):].any()
    weights = torch.full((t, 1), 0.5, device="cuda")
    y = ops.moe_combine(xs, plan, weights)
    for s in parts:
        assert torch.equal(y[s], torch.where(rank[s][:, None] >= 0, x[s] * 0.5, 0.0))
    del y
    dys, dw = ops.moe_combine_back(x, xs, plan, weights)
    for s in parts:
        assert torch.equal(dys[s], xs[s] * 0.5)
        want = torch.where(rank[s] >= 0, (x[s].float() ** 2).sum(1), 0.0)
        # two float32 sums of 2048 squares
        assert torch.allclose(dw[s, 0], want, rtol=2 * 2048 * half_step(torch.float32), atol=0)


@gpu
def test_quantize_past_32_bits_of_threads():
    """As many workgroups, four rows in each."""
    t, d = (1 << 26) + 77, 1056
    enough_memory(215 << 30)
    x = far_rows(t, d, torch.bfloat16)
    m = ops.mx4_quantize(x)
    parts = [slice(i, i + (1 << 20)) for i in range(0, t, 1 << 20)]
    for s in parts:
        want = ops.mx4_quantize(x[s])
        assert torch.equal(m.codes[s], want.codes) and torch.equal(m.scales[:, s], want.scales)
    del x
    torch.cuda.empty_cache()
    y = ops.mx4_dequantize(m, torch.bfloat16)
    for s in parts:
        assert torch.equal(y[s], ops.mx4_dequantize(ops.Mx4(m.codes[s], m.scales[:, s].contiguous()), torch.bfloat16))


@gpu
def test_flat_abi_on_a_private_stream():
    """stream NULL: done when the call returns."""
    rng = np.random.default_rng(0)
    x, x64 = rows_of(rng, 4, 64, torch.float32)
    codes, scales = torch.empty(4, 32, dtype=torch.uint8, device="cuda"), torch.empty(1, 4, 8, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert flat("mi355x_mx4_quantize")(0, x.data_ptr(), 64, 4, 64, codes.data_ptr(), scales.data_ptr(), None) == 0
    code, e = unpack(ops.Mx4(codes, scales))
    assert (code == np_quantize(x64)[0]).all() and (e == np_quantize(x64)[1]).all()


@gpu
def test_tensors_refused_on_the_host():
    rng = np.random.default_rng(0)
    x = torch.zeros(4, 64, device="cuda")
    w, _ = random_mx4(rng, 8, 64)
    we, _ = random_mx4(rng, 3, 8, 64)
    _, _, _, plan = plan_of(rng, 4, 2, 3, "even")
    rows, weights = torch.zeros(8, 64, device="cuda"), torch.zeros(4, 2, device="cuda")
    bad = [
        (ValueError, lambda: ops.mx4_quantize(x[:, :40])), (ValueError, lambda: ops.mx4_quantize(x[0])),
        (TypeError, lambda: ops.mx4_quantize(x.double())), (ValueError, lambda: ops.mx4_quantize(torch.zeros(64, 4, device="cuda").t())),
        (ValueError, lambda: ops.mx4_quantize(x.expand(4, 64)[:1].expand(4, 64))), (ValueError, lambda: ops.mx4_quantize(x.clone().requires_grad_())),
        (TypeError, lambda: ops.mx4_dequantize(w, torch.int32)), (ValueError, lambda: ops.mx4_dequantize(we)),
        (ValueError, lambda: ops.mx4_dequantize(ops.Mx4(w.codes[:, :24], w.scales))),
        (ValueError, lambda: ops.mx4_dequantize(ops.Mx4(w.codes, w.scales[:, :7]))),
        (TypeError, lambda: ops.mx4_dequantize(ops.Mx4(w.codes.to(torch.int8), w.scales))),
        (ValueError, lambda: ops.mx4_mul_mat(w, x[:, :32])), (TypeError, lambda: ops.mx4_mul_mat(w, x.long())),
        (TypeError, lambda: ops.mx4_mul_mat(w, x, torch.float64)), (ValueError, lambda: ops.mx4_mul_mat(we, x)),
        (ValueError, lambda: ops.mx4_mul_mat_id(we, x[:3], plan)), (ValueError, lambda: ops.mx4_mul_mat_id(we, x, plan, x_sorted=True)),
        (ValueError, lambda: ops.mx4_mul_mat_id(ops.Mx4(we.codes[:2], we.scales[:2]), x, plan)),
        (TypeError, lambda: ops.mx4_mul_mat_id(we, x, tuple(plan))),
        (TypeError, lambda: ops.moe_sort(weights, 3)), (ValueError, lambda: ops.moe_sort(plan.rank, 0)),
        (ValueError, lambda: ops.moe_sort(plan.rank, 1025)), (ValueError, lambda: ops.moe_sort(plan.rank.t(), 3)),
        (ValueError, lambda: ops.moe_sort(torch.zeros(2, 17, dtype=torch.int32, device="cuda"), 3)),
        (ValueError, lambda: ops.moe_gather(rows, plan)), (ValueError, lambda: ops.moe_combine(x, plan, weights)),
        (ValueError, lambda: ops.moe_combine(rows, plan, weights[:3])), (TypeError, lambda: ops.moe_combine(rows, plan, weights.half())),
        (TypeError, lambda: ops.moe_combine(rows, plan._replace(order=plan.order.long()), weights)),
        (ValueError, lambda: ops.moe_combine(rows, plan._replace(order=plan.order[:4]), weights)),
        (TypeError, lambda: ops.moe_combine_back(x.half(), rows, plan, weights)), (ValueError, lambda: ops.moe_combine_back(x[:3], rows, plan, weights)),
        (ValueError, lambda: ops.moe_combine_back(x, rows, plan, weights.clone().requires_grad_())),
    ]
    bad += [(ValueError, call) for call in [
        lambda: ops.mx4_quantize(torch._neg_view(x)), lambda: ops.mx4_quantize(x.to_sparse()), lambda: ops.mx4_mul_mat(w, torch._neg_view(x)),
        lambda: ops.moe_combine(rows, plan, torch._neg_view(weights)), lambda: ops.moe_sort(torch._neg_view(plan.rank), 3),
        lambda: ops.moe_combine_back(torch._neg_view(x), rows, plan, weights),
    ]]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {i} was not refused")
    with torch.no_grad():
        ops.mx4_quantize(x.clone().requires_grad_())


def hip_runtime():
    """The HIP runtime of this process."""
    with open("/proc/self/maps") as maps:
        return ctypes.CDLL(next(line.split()[-1] for line in maps if "libamdhip64" in line))


@gpu
def test_calls_after_an_earlier_failure_of_the_thread():
    """A HIP call that failed before, elsewhere in the program, neither fails a valid call nor is taken from
    the one who has yet to ask for it."""
    args, _ = layer_case(4)
    x, ids, weights, up, _, n_expert = args
    rng = np.random.default_rng(0)
    w, _ = random_mx4(rng, 70, 4128)
    many = torch.randn(129, 4128, device="cuda")          # tiles, K in shares
    plan = ops.moe_sort(ids, n_expert)
    wide = torch.randint(0, n_expert, (5000, 2), device="cuda")   # two launches
    ys = torch.randn(8, 512, device="cuda")
    calls = [lambda: ops.mx4_quantize(x), lambda: (ops.mx4_dequantize(up._replace(codes=up.codes[0], scales=up.scales[0])),),
             lambda: (ops.mx4_mul_mat(w, many[:1]),), lambda: (ops.mx4_mul_mat(w, many),), lambda: (ops.mx4_mul_mat_id(up, x, plan),),
             lambda: plan, lambda: ops.moe_sort(ids, n_expert), lambda: ops.moe_sort(wide, n_expert), lambda: (ops.moe_gather(x, plan),),
             lambda: (ops.moe_combine(ys, plan, weights),), lambda: ops.moe_combine_back(x, ys, plan, weights)]
    hip = hip_runtime()
    for i, call in enumerate(calls):
        want = call()
        torch.cuda.synchronize()
        failed = hip.hipSetDevice(-1)
        assert failed != 0
        try:
            got = call()
        finally:
            left = hip.hipGetLastError()
        assert left == failed, f"call {i}"
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"call {i}"


def tangent_calls(x, device):
    """Calls with a tensor that carries a tangent: (call, does it get as far without a GPU)."""
    dual = lambda *shape: torch.autograd.forward_ad.make_dual(torch.zeros(shape, device=device), torch.ones(shape, device=device))  # noqa: E731
    tokens, rows, weights = (2, 64), (4, 64), (2, 2)
    dual_x, dual_ys, dual_w = dual(*tokens), dual(*rows), dual(*weights)
    ys, w = torch.zeros(rows, device=device), torch.zeros(weights, device=device)
    plan = ops.MoePlan(torch.arange(4, dtype=torch.int32, device=device), torch.arange(4, dtype=torch.int32, device=device).view(2, 2),
                       torch.tensor([0, 4], dtype=torch.int32, device=device))
    m = ops.Mx4(torch.zeros(1, 3, 32, dtype=torch.uint8, device=device), torch.zeros(1, 1, 3, 8, dtype=torch.uint8, device=device))
    return [
        (lambda: ops.mx4_quantize(dual_x), True), (lambda: ops.moe_gather(dual_x, plan), True),
        (lambda: ops.moe_combine(dual_ys, plan), True), (lambda: ops.moe_combine_back(x, dual_ys, plan, w), True),
        (lambda: ops.mx4_mul_mat(ops.Mx4(m.codes[0], m.scales[0]), dual_x), False), (lambda: ops.mx4_mul_mat_id(m, dual_x, plan), False),
        (lambda: ops.moe_combine(ys, plan, dual_w), False), (lambda: ops.moe_combine_back(dual_x, ys, plan, w), False),
        (lambda: ops.moe_combine_back(x, ys, plan, dual_w), False),
    ]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_tangents_are_refused(device):
    """Forward mode: a tangent would be dropped without a word.  no_grad() does not turn it off."""
    with torch.autograd.forward_ad.dual_level():
        for i, (call, anywhere) in enumerate(tangent_calls(torch.zeros(2, 64, device=device), device)):
            if device == "cpu" and not anywhere:
                continue
            for mode in (torch.enable_grad(), torch.no_grad()):
                with mode, pytest.raises(ValueError, match="tangent"):
                    call()
                    pytest.fail(f"call {i} was not refused")
            if device == "cuda":
                with torch.autograd.forward_ad._set_fwd_grad_enabled(False):
                    call()


@pytest.mark.parametrize("target,binding", [("all", False), ("ops", False), ("torch", True)])
def test_only_the_binding_is_built_against_torch(target, binding):
    """What make would run for a target from nothing: the plugin and the flat library on a host without torch."""
    csrc = os.path.join(la.PKG, "csrc")
    out = subprocess.run(["make", "-n", "-B", "-C", csrc, target], capture_output=True, text=True, check=True).stdout
    assert ("torch" in re.sub(r"make.*directory.*", "", out)) == binding
    assert "libmi355x-ops.so" in out


@gpu
def test_every_exponent():
    """All codes with all exponents as values, and as products of one block: zeros under float32's least number,
    infinities past its largest, NaN for 255; tiles and few rows."""
    rng = np.random.default_rng(4)
    byte = np.arange(256, dtype=np.uint8)[:, None]
    code = np.tile(np.arange(16, dtype=np.uint8), 2)[None].repeat(256, 0)
    with np.errstate(over="ignore"):
        want = torch.from_numpy(np_values(code, byte))
    for dtype in TYPES:
        y = ops.mx4_dequantize(pack(code, byte), dtype).cpu()
        assert torch.equal(y.nan_to_num(99.0), want.to(dtype).nan_to_num(99.0)) and torch.equal(y.isnan(), want.isnan())
    cw, cx = rng.integers(0, 16, (2, 256, 32), dtype=np.uint8)
    s = GRID[cx] @ GRID[cw].T                 # exact, and so is its product with a power of two in 64 bits
    with np.errstate(over="ignore"):
        want = np.ldexp(s, byte.astype(int) + byte.T.astype(int) - 254).astype(np.float32)
    want[255] = want[:, 255] = np.nan
    for t in (1, 16, 32, 256):
        for at in range(0, 256, max(t, 32)):
            rows = slice(at, at + t)
            y = ops.mx4_mul_mat(pack(cw, byte), pack(cx[rows], byte[rows]), torch.float32).cpu().numpy()
            assert np.array_equal(y, want[rows], equal_nan=True)


@gpu
def test_tensors_without_rows_or_columns():
    rng = np.random.default_rng(0)
    w, _ = random_mx4(rng, 8, 64)
    we, _ = random_mx4(rng, 3, 8, 64)
    none_w = ops.Mx4(w.codes[:0], w.scales[:, :0].contiguous())
    none_e = ops.Mx4(we.codes[:, :0].contiguous(), we.scales[:, :, :0].contiguous())
    x, weights = torch.ones(4, 64, device="cuda"), torch.ones(4, 2, device="cuda")
    _, _, _, plan = plan_of(rng, 4, 2, 3, "even")
    no_plan = ops.moe_sort(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 3)
    q = ops.mx4_quantize(x[:0])
    assert q.codes.shape == (0, 32) and q.scales.shape == (1, 0, 8) and ops.mx4_dequantize(q).shape == (0, 64)
    assert ops.mx4_mul_mat(w, x[:0]).shape == ops.mx4_mul_mat(w, q).shape == (0, 8) and ops.mx4_mul_mat(none_w, x).shape == (4, 0)
    assert ops.mx4_mul_mat_id(we, x[:0], no_plan).shape == (0, 8) and ops.mx4_mul_mat_id(none_e, x, plan).shape == (8, 0)
    assert ops.moe_gather(x[:, :0], plan).shape == (8, 0) and ops.moe_combine(x.repeat(2, 1)[:, :0], plan, weights).shape == (4, 0)
    dys, dw = ops.moe_combine_back(x[:0], x[:0], no_plan, weights[:0])
    assert dys.shape == (0, 64) and dw.shape == (0, 2)
    dys, dw = ops.moe_combine_back(x[:, :0], x.repeat(2, 1)[:, :0], plan, weights)
    assert dys.shape == (8, 0) and not dw.any()          # a sum of nothing


@gpu
def test_large_expert_layer_in_a_graph():
    """Two launches of the sort, products in tiles; replayed on new routings with eager work between."""
    args, _ = layer_case(3000)
    x, ids, weights = (v.clone() for v in args[:3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        expert_layer(x, ids, weights, *args[3:])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = expert_layer(x, ids, weights, *args[3:])
    for seed in range(3):
        fresh, _ = layer_case(3000, seed)
        for to, src in zip((x, ids, weights), fresh[:3]):
            to.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, expert_layer(x, ids, weights, *args[3:]))


@gpu
def test_weights_of_experts_stacked():
    """The experts' weights out of one quantisation each, as the documentation stacks them."""
    rng = np.random.default_rng(6)
    matrices = [rows_of(rng, 40, 288, torch.bfloat16)[0] for _ in range(3)]
    w = ops.Mx4(*map(torch.stack, zip(*map(ops.mx4_quantize, matrices))))
    ids, order, _, plan = plan_of(rng, 20, 2, 3, "even")
    x, x64 = rows_of(rng, 20, 288, torch.float32)
    y = ops.mx4_mul_mat_id(w, x, plan)
    for e in range(3):
        at = np.flatnonzero(ids.reshape(-1)[order] == e)
        check_product(y[torch.from_numpy(at).cuda()], np_rounded(matrices[e].double().cpu().numpy()), np_rounded(x64)[order[at] // 2], torch.float32)


def test_a_second_hip_runtime_is_refused_before_it_is_loaded():
    """The flat library (as the plugin would) has brought the system's runtime: torch's is not loaded beside it."""
    code = f"""
import ctypes, sys
ctypes.CDLL({ops.LIBRARY!r}, mode=ctypes.RTLD_GLOBAL)
sys.path.insert(0, {la.REPO!r})
try:
    import llamacog_amd.device_ops
    print("imported")
except ImportError as e:
    print("refused" if "two HIP runtimes" in str(e) else e, "torch" in sys.modules)
"""
    if not os.path.exists(os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so")):
        pytest.skip("this torch brings no HIP runtime of its own")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.split() == ["refused", "False"], (out.returncode, out.stdout, out.stderr)


# the flat ABI on launchers that do nothing: the quantisation in front of a product succeeds, the product fails
LAUNCHERS = r"""
#include "devops.h"
#include "ggml-mi355x.h"
#include <cstdio>
static int launched, waited_for, destroyed;
extern "C" hipError_t hipStreamCreateWithFlags(hipStream_t * s, unsigned) { *s = (hipStream_t) 16; return hipSuccess; }
extern "C" hipError_t hipStreamSynchronize(hipStream_t) { waited_for = launched; return hipSuccess; }
extern "C" hipError_t hipStreamDestroy(hipStream_t) { ++destroyed; return hipSuccess; }
namespace mi355x_ops {
hipError_t mx4_quantize(int, const void *, int64_t, int64_t, int64_t, uint8_t *, uint8_t *, hipStream_t) { ++launched; return hipSuccess; }
mx4_needs mx4_product_needs(const mx4_mat &, int64_t, const moe_view *) { return {true, 0}; }
hipError_t mx4_product(const mx4_mat &, const mx4_mat &, const moe_view *, int, void *, void *, hipStream_t) { return hipErrorLaunchFailure; }
hipError_t mx4_product_float(const mx4_mat &, int, const void *, int64_t, int64_t, const moe_view *, int, void *, hipStream_t) { return hipSuccess; }
hipError_t mx4_dequantize(const mx4_mat &, int, void *, hipStream_t) { return hipSuccess; }
size_t moe_sort_workspace(int64_t, int) { return 0; }
hipError_t moe_sort(const void *, int, int64_t, int, int32_t *, int32_t *, int32_t *, void *, hipStream_t) { return hipSuccess; }
hipError_t moe_gather(int, const void *, int64_t, int64_t, int64_t, int, const int32_t *, const int32_t *, void *, hipStream_t) { return hipSuccess; }
hipError_t moe_combine(int, const void *, int64_t, int64_t, int64_t, int, const int32_t *, const float *, void *, hipStream_t) { return hipSuccess; }
hipError_t moe_combine_back(int, const void *, int64_t, const void *, int64_t, int64_t, int64_t, int, const int32_t *, const int32_t *, const float *,
                            void *, float *, hipStream_t) { return hipSuccess; }
}
int main() {
    uint8_t * a = (uint8_t *) (1 << 20);
    const int rc = mi355x_mx4_mul_mat(a, a, 8, 64, 0, a, nullptr, 64, 3, 0, a, a, 1 << 20, nullptr);
    std::printf("%d %d %d %d", rc, launched, waited_for, destroyed);
}
"""


def test_private_stream_is_waited_for_after_a_failed_launch(tmp_path):
    """What a call had launched before it failed is done when it returns: the caller may free its memory."""
    (tmp_path / "t.cpp").write_text(LAUNCHERS)
    csrc, objects = os.path.join(la.PKG, "csrc"), []
    for src in (os.path.join(csrc, "devops_capi.cpp"), str(tmp_path / "t.cpp")):
        objects.append(str(tmp_path / f"{len(objects)}.o"))
        subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "-std=c++20", "-fPIC", "-I", csrc, "-I", os.path.join(la.REPO, "include"),
                        "-c", src, "-o", objects[-1]], check=True)
    subprocess.run(["g++", *objects, "-o", str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout
    assert out.split() == ["-5", "1", "1", "1"]   # MI355X_ERR_HIP; one launch, waited for; the stream is gone
