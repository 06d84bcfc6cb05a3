"""The MXFP4 product's kernels one by one (llamacog_amd.device_ops): sizes that take each tile, ring and
number of shares of K, dense and by experts, and the few-row kernel's splits.  Which kernel a size takes is
asked of the rules themselves, compiled for the host: a change of the rules that leaves a kernel without a
test fails here.

Codes are multiples of 1/2 and exponents lie within a few octaves, so that every partial sum is a whole
number of units that float32 holds (sum |w x| below 2^24 units, asserted): results have to be equal to those in 64 bits,
rounded once."""
import os
import subprocess
import threading

import pytest
import torch

import llamacog_amd as la
from llamacog_amd import device_ops as ops

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]

# rows of y, rows of the weights, K, experts (0: dense) -> side, planes in the ring, shares of K
TILES = {
    (33, 70, 96, 0): (64, 4, 1),
    (129, 70, 4128, 0): (64, 4, 4),
    (257, 257, 65568, 0): (64, 4, 16),
    (1000, 2050, 1056, 0): (128, 4, 1),
    (257, 8200, 2080, 0): (128, 4, 1),
    (257, 500, 32800, 0): (128, 4, 8),
    (1000, 4100, 64, 0): (128, 2, 1),
    (2100, 8200, 1056, 0): (128, 2, 1),
    (1023, 8200, 288, 0): (256, 2, 1),
    (400, 20000, 64, 0): (256, 2, 1),
    (3000, 8200, 800, 0): (256, 2, 1),     # more tiles than CUs
    (1000, 2050, 65568, 0): (256, 2, 4),
    (132, 130, 64, 3): (64, 2, 1),
    (130, 257, 4128, 2): (64, 2, 4),
    (2100, 1000, 8224, 3): (128, 4, 1),
    (700, 1000, 32800, 2): (128, 4, 4),
    (2100, 8200, 1056, 5): (128, 2, 1),
    (1000, 500, 131104, 1): (128, 2, 16),
    (3000, 8200, 800, 5): (256, 2, 1),
    (2100, 1000, 65568, 2): (256, 2, 8),
}
# the same -> tiles of 16 rows in a workgroup, waves that share a group of weight rows
FEW = {
    (1, 40000, 544, 0): (1, 1),
    (3, 17000, 1056, 0): (1, 2),
    (16, 9000, 2080, 0): (1, 4),
    (9, 70, 4128, 0): (1, 8),
    (17, 40000, 288, 0): (2, 1),
    (32, 70, 288, 0): (2, 2),
    (31, 257, 1024, 0): (2, 4),
    (29, 4100, 4128, 0): (2, 8),
    (30, 100, 14336, 0): (1, 8),           # two tiles of x do not fit
    (2000, 1000, 288, 256): (1, 1),        # more groups than workgroups take at a time
    (12, 9000, 800, 3): (1, 2),
    (100, 70, 1056, 40): (1, 8),
    (4, 4100, 2080, 8): (1, 2),
    (6, 1000, 2080, 6): (1, 8),
    (16, 1400, 2080, 8): (1, 4),
}
HARNESS = """#include "mx4_rules.h"
#include <cstdio>
using namespace mi355x_ops;
int main() {
    long long t, m, k, e;
    while (std::scanf("%lld %lld %lld %lld", &t, &m, &k, &e) == 4) {
        const product_size a{m, (int) (k / 32), t, (int) e};
        const tile_choice c = pick_tile(a);
        if (few_rows(a)) std::printf("%d %d\\n", mv_tiles(a), mv_split(a, mv_tiles(a)));
        else std::printf("%d %d %d\\n", c.side, c.stages, c.shares);
    }
}
"""


def compiled(tmp_path, text):
    src, out = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(text)
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Werror", "-I", os.path.join(la.PKG, "csrc"), str(src), "-o", str(out)], check=True)
    return out


def test_each_kernel_has_its_sizes(tmp_path):
    sizes = {**TILES, **FEW}
    text = "\n".join("%d %d %d %d" % s for s in sizes)
    out = subprocess.run([str(compiled(tmp_path, HARNESS))], input=text, capture_output=True, text=True, check=True).stdout
    got = {s: tuple(int(v) for v in line.split()) for s, line in zip(sizes, out.splitlines())}
    assert got == sizes
    # every instantiation, with K whole and in shares
    for ids, rings in ((False, {(256, 2), (128, 4), (128, 2), (64, 4)}), (True, {(256, 2), (128, 4), (128, 2), (64, 2)})):
        of = [v for s, v in TILES.items() if (s[3] > 0) == ids]
        assert {v[:2] for v in of if v[2] == 1} == rings
        assert {v[0] for v in of if v[2] > 1} == {256, 128, 64}
    assert {v for s, v in FEW.items() if not s[3]} == {(n, k) for n in (1, 2) for k in (1, 2, 4, 8)}
    assert {v for s, v in FEW.items() if s[3]} == {(1, k) for k in (1, 2, 4, 8)}


def test_tiles_of_nearly_all_32_bits(tmp_path):
    """One expert's pairs may be as many as 2^31 - 1: their tiles are counted without passing 32 bits."""
    cases = [(0, 64), (1, 64), (64, 64), (65, 64), (2 ** 31 - 1, 256), (2 ** 31 - 16, 64), (2 ** 31 - 64, 64), (2 ** 31 - 1, 16)]
    checks = "".join(f"static_assert(mi355x_ops::tiles_of({n}, {rows}) == {-(-n // rows)});" for n, rows in cases)
    compiled(tmp_path, f'#include "mx4_rules.h"\n{checks} int main() {{}}')


# ---- on the GPU ----------------------------------------------------------------------------------
def octaves(k):
    """How far exponents may lie from 1 with whole sums of K products: on average a product is 5.06 times
    1, 1.36 or 2.4 (exponents the same, one or two octaves around), in units of 1/4, 1/16 or 1/64."""
    return 2 if k < 10000 else 1 if k < 70000 else 0


def operand(g, shape):
    """(Mx4 of this shape, its values in 64 bits); bytes past K hold rubbish."""
    k, o = shape[-1], octaves(shape[-1])
    code = torch.randint(0, 16, shape, dtype=torch.uint8, device="cuda", generator=g)
    e = torch.randint(127 - o, 128 + o, shape[:-1] + (k // 32,), dtype=torch.uint8, device="cuda", generator=g)
    size = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    grid = torch.cat((size, -size))
    values = (grid[code.int()].unflatten(-1, (-1, 32)) * torch.exp2(e.double() - 127)[..., None]).flatten(-2)
    planes = torch.nn.functional.pad(e, (0, -(k // 32) % 8), value=255).unflatten(-1, (-1, 8)).transpose(-3, -2).contiguous()
    return ops.Mx4(code[..., 0::2] | (code[..., 1::2] << 4), planes), values


def check(y, w, x, what=""):
    unit = 4.0 ** -(1 + octaves(w.shape[1]))
    assert float((x.abs() @ w.abs().t()).max()) < unit * 2 ** 24, "these sums are not exact"
    want = x @ w.t()
    assert torch.equal(y, want.to(y.dtype)), f"{what}: {int((y != want.to(y.dtype)).sum())} of {y.numel()} differ"


@gpu
@pytest.mark.parametrize("t,m,k", [s[:3] for s in (*TILES, *FEW) if not s[3]])
def test_dense(t, m, k):
    g = torch.Generator(device="cuda").manual_seed(t + m + k)
    (w, w64), (x, x64) = operand(g, (m, k)), operand(g, (t, k))
    for dtype in TYPES:
        check(ops.mx4_mul_mat(w, x, dtype), w64, x64, str(dtype))


def ids_of(g, t, used, n_expert, kind):
    if kind == "one":
        return torch.full((t, used), n_expert - 1, device="cuda")
    if kind == "none":
        return torch.full((t, used), -1, device="cuda")
    ids = torch.randint(0, n_expert, (t, used), device="cuda", generator=g)
    if kind == "skewed":      # nearly all to the first expert, single rows to others
        ids[torch.rand(t, used, device="cuda", generator=g) < 0.95] = 0
    if kind == "holes":
        ids[torch.rand(t, used, device="cuda", generator=g) < 0.2] = -1
        ids[-(t // 4 or 1):] = n_expert
    return ids


@gpu
@pytest.mark.parametrize("pairs,m,k,n_expert", [s for s in (*TILES, *FEW) if s[3]])
@pytest.mark.parametrize("kind", ["even", "skewed", "holes", "one", "none"])
def test_by_experts(pairs, m, k, n_expert, kind):
    g = torch.Generator(device="cuda").manual_seed(pairs + m + k)
    used = 2
    ids = ids_of(g, pairs // used, used, n_expert, kind)
    plan = ops.moe_sort(ids, n_expert)
    (w, w64), (x, x64) = operand(g, (n_expert, m, k)), operand(g, (pairs // used, k))
    offsets, order = plan.offsets.tolist(), plan.order.long()
    for dtype in TYPES:
        y = ops.mx4_mul_mat_id(w, x, plan, dtype=dtype)
        for e in range(n_expert):
            rows = slice(offsets[e], offsets[e + 1])
            check(y[rows], w64[e], x64[order[rows] // used], f"{dtype}, expert {e}") if offsets[e] < offsets[e + 1] else None
        assert not y[offsets[-1]:].any()
    # rows in the plan's order already
    held = offsets[-1]
    codes, scales = torch.zeros(pairs, k // 2, dtype=torch.uint8, device="cuda"), torch.zeros(-(-k // 256), pairs, 8, dtype=torch.uint8, device="cuda")
    codes[:held], scales[:, :held] = x.codes[order[:held] // used], x.scales[:, order[:held] // used]
    assert torch.equal(ops.mx4_mul_mat_id(w, ops.Mx4(codes, scales), plan, True, torch.bfloat16), y)


def several():
    """Calls through the tiles: joined shares of K, a 256 tile, experts in tiles."""
    g = torch.Generator(device="cuda").manual_seed(1)
    float_x = torch.randn(1023, 288, device="cuda", generator=g)
    (w, _), (x, _), (big, _), (experts, _) = operand(g, (70, 4128)), operand(g, (129, 4128)), operand(g, (8200, 288)), operand(g, (3, 1000, 8224))
    xe, _ = operand(g, (1050, 8224))
    plan = ops.moe_sort(ids_of(g, 1050, 2, 3, "holes"), 3)
    return [lambda: ops.mx4_mul_mat(w, x), lambda: ops.mx4_mul_mat(big, float_x), lambda: ops.mx4_mul_mat_id(experts, xe, plan)]


@gpu
def test_tiles_on_several_streams():
    calls = several()
    want = [call() for call in calls]
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(4)]:
        with torch.cuda.stream(s):
            got += [[call() for call in calls] for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for ys in got for a, b in zip(ys, want))


@gpu
def test_tiles_from_two_threads():
    calls = several()
    want = [call() for call in calls]
    torch.cuda.synchronize()
    same = [False, False]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            ys = [[call() for call in calls] for _ in range(5)]
            torch.cuda.current_stream().synchronize()
            same[i] = all(torch.equal(a, b) for y in ys for a, b in zip(y, want))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert same == [True, True]


@gpu
def test_tiles_in_a_graph():
    """Captured once, replayed with eager calls between."""
    calls = several()
    want = [call() for call in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for call in calls:
            call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = [call() for call in calls]
    for _ in range(4):
        for y in ys:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ys, want))
        assert all(torch.equal(call(), b) for call, b in zip(calls, want))


def numbered_rows(g, rows):
    """MXFP4 rows of 32 elements that all differ: the row's number, then a million random rows over and over."""
    codes = torch.empty(rows, 16, dtype=torch.uint8, device="cuda")
    some = torch.randint(0, 256, (1 << 20, 16), dtype=torch.uint8, device="cuda", generator=g)
    for at in range(0, rows, 1 << 20):
        codes[at:at + (1 << 20)] = some[:rows - at]
    codes.view(torch.int32)[:, 0] = torch.arange(rows, dtype=torch.int32, device="cuda")
    return ops.Mx4(codes, torch.full((1, rows, 8), 127, dtype=torch.uint8, device="cuda"))


@gpu
def test_tiles_past_32_bits_of_threads():
    """As many rows as a call may have: more tiles than one axis of a launch has room for."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 110 << 30:
        pytest.skip("110 GiB of the card's memory are wanted")
    g = torch.Generator(device="cuda").manual_seed(1)
    w, _ = operand(g, (1, 32))
    rows = 2 ** 31 - 1
    x = numbered_rows(g, rows)
    y = ops.mx4_mul_mat(w, x, torch.float16)
    step = 1 << 24
    for at in range(0, rows, step):
        part = ops.Mx4(x.codes[at:at + step], x.scales[:, at:at + step])
        assert torch.equal(y[at:at + step], ops.mx4_mul_mat(w, part, torch.float16)), at
    assert y[:1 << 20].unique().numel() > 100
    # by experts: all of 2^31 - 16 pairs but the last token's belong to one
    tokens = rows // 16
    y = y[:tokens].clone()
    x = ops.Mx4(x.codes[:tokens].clone(), x.scales[:, :tokens].clone())
    ids = torch.zeros(tokens, 16, dtype=torch.int32, device="cuda")
    ids[-1] = -1
    plan = ops.moe_sort(ids, 1)
    del ids
    ye = ops.mx4_mul_mat_id(ops.Mx4(w.codes[None], w.scales[None]), x, plan, dtype=torch.float16).view(tokens, 16)
    assert plan.offsets.tolist() == [0, 16 * (tokens - 1)] and not ye[-1].any()
    assert torch.equal(ye[:-1], y[:-1].expand(-1, 16))
