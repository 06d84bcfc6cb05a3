"""What is measured of the MXFP4 products and the expert routing (llamacog_amd.device_ops): the cases, their inputs,
and each operator in plain torch operations.

MXFP4 storage, as the framework keeps it: `codes` uint8 [..., rows, K / 2], element 2 i in the low half of byte i, each
an E2M1 number (sign, 0 0.5 1 1.5 2 3 4 6); `scales` uint8 [..., ceil(K / 256), rows, 8], byte b of plane s of row r
the exponent (2^(byte - 127), 255 = NaN) of that row's elements 256 s + 32 b to 256 s + 32 b + 31.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- the cases -------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token's activations on their way into a 4-bit product, and back as values
        {"name": "quantize-token", "op": "quantize", "rows": 1, "k": 4096, "type": "float32"},
        # a weight matrix of the 70B shape (gate or up) converted once, with the values it then stands for
        {"name": "quantize-weight", "op": "quantize", "rows": 28672, "k": 8192, "type": "bfloat16"},
        # decoding one token: the 8B shape's down projection
        {"name": "product-token", "op": "product", "t": 1, "m": 4096, "k": 14336, "type": "float32"},
        # a ragged decode batch into a vocabulary of 32000 and one added token
        {"name": "product-ragged", "op": "product", "t": 29, "m": 32001, "k": 4096, "type": "float16"},
        # a prompt batch through the 70B shape's gate projection
        {"name": "product-prompt", "op": "product", "t": 2048, "m": 28672, "k": 8192, "type": "bfloat16"},
        # decoding one token: gate and up of its two experts of eight
        {"name": "experts-token", "op": "experts", "t": 1, "m": 28672, "k": 4096, "e": 8, "used": 2, "type": "float32",
         "sorted": False, "skew": 0.0, "pad": 0},
        # a small batch over many small experts, most of them with a few tokens or none, with padded rows
        {"name": "experts-ragged", "op": "experts", "t": 37, "m": 1408, "k": 2048, "e": 64, "used": 6, "type": "bfloat16",
         "sorted": False, "skew": 1.0, "pad": 3},
        # a prompt batch through the experts' down projection, rows already sorted
        {"name": "experts-prompt", "op": "experts", "t": 4096, "m": 4096, "k": 14336, "e": 8, "used": 2, "type": "bfloat16",
         "sorted": True, "skew": 0.5, "pad": 0},
        # one token's slots sorted and its row copied to them
        {"name": "dispatch-token", "op": "dispatch", "t": 1, "d": 4096, "e": 8, "used": 2, "type": "float32", "skew": 0.0,
         "pad": 0},
        # a large batch over many experts
        {"name": "dispatch-batch", "op": "dispatch", "t": 16384, "d": 2048, "e": 128, "used": 8, "type": "bfloat16",
         "skew": 1.0, "pad": 100},
        # the weighted rows of a prompt's tokens back in token order
        {"name": "combine-prompt", "op": "combine", "back": False, "weighted": True, "t": 512, "d": 4096, "e": 8, "used": 2,
         "type": "float32", "skew": 0.5, "pad": 0},
        # the gradient of that for a large batch
        {"name": "combine-back", "op": "combine", "back": True, "weighted": True, "t": 16384, "d": 2048, "e": 128, "used": 8,
         "type": "bfloat16", "skew": 1.0, "pad": 100},
    ]


def spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("quantize", "product", "experts", "dispatch", "combine"))
    kind = rng.choice(("float32", "float16", "bfloat16"))
    if op == "quantize":
        k = 32 * spread(rng, 1, 896)
        return {"op": op, "rows": spread(rng, 1, min(65536, 28672 * 8192 // k)), "k": k, "type": kind}
    if op == "product":
        k, m = 32 * spread(rng, 4, 448), spread(rng, 64, 32768)
        return {"op": op, "t": spread(rng, 1, max(1, min(8192, 2048 * 28672 * 8192 // (m * k)))), "m": m, "k": k, "type": kind}
    e = spread(rng, 2, 256)
    used = min(e, rng.randint(1, 8))
    skew = rng.choice((0.0, 0.5, 1.0, 2.0))
    if op == "experts":
        k, m = 32 * spread(rng, 4, 448), spread(rng, 64, 28672)
        m = max(64, min(m, 28672 * 4096 * 8 // (e * k)))
        t = spread(rng, 1, max(1, min(8192, 8192 * 4096 * 14336 // (m * k * used), 3 * 10**9 // (e * max(m, k)))))
        return {"op": op, "t": t, "m": m, "k": k, "e": e, "used": used, "type": kind, "sorted": rng.random() < 0.5, "skew": skew,
                "pad": rng.choice((0, 0, t // 8))}
    d = spread(rng, 16, 8192)
    t = spread(rng, 1, max(1, min(32768, 16384 * 2048 * 8 // (d * used))))
    case = {"op": op, "t": t, "d": d, "e": e, "used": used, "type": kind, "skew": skew, "pad": rng.choice((0, 0, t // 8))}
    if op == "combine":
        case["back"] = rng.random() < 0.5
        case["weighted"] = case["back"] or rng.random() < 0.7
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------
def exponent_planes(exponents):
    """[..., rows, K / 32] exponent bytes -> the planes [..., ceil(K / 256), rows, 8]."""
    n = exponents.shape[-1]
    whole = torch.nn.functional.pad(exponents, (0, -n % 8))
    return whole.unflatten(-1, (-1, 8)).transpose(-3, -2).contiguous()


def exponent_rows(scales, k):
    """The planes back as [..., rows, K / 32]."""
    return scales.transpose(-3, -2).flatten(-2)[..., : k // 32]


def plain_codes(x):
    """Blocks x [..., 32] in float32 -> (codes [..., 32], exponent bytes [...]); every step is exact but the one rounding."""
    top = x.abs().amax(-1)
    # floor(log2(top)) from the number's own bits, those under 2^-126 after a shift by 2^64
    small = top < 2.0 ** -126
    bits = torch.where(small, top * 2.0 ** 64, top).view(torch.int32)
    exponent = (bits >> 23) - 127 - torch.where(small, 64, 0) - 2
    exponent = torch.where(top > 0, exponent, -127).clamp(-127, 127)
    inverse = ((127 - exponent).to(torch.int32) << 23).view(torch.float32)  # 2^-exponent
    a = (x.abs() * inverse[..., None]).clamp(max=8.0)
    a = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp(max=6.0)
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4))
    finite = torch.isfinite(top)
    code = torch.where(finite[..., None], code, 0.0).to(torch.uint8) | (torch.signbit(x).to(torch.uint8) << 3)
    return code, torch.where(finite, exponent + 127, 255).to(torch.uint8)


def plain_values(codes, exponents):
    """codes [..., 32] and exponent bytes [...] -> float32 values."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    byte = exponents.to(torch.int32)
    scale = torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)  # 2^(byte - 127)
    scale = torch.where(byte == 255, float("nan"), scale)
    return grid[codes.long()] * scale[..., None]


def packed(x):
    """Rows [rows, K] -> MXFP4 storage."""
    code, exponents = plain_codes(x.float().unflatten(-1, (-1, 32)))
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), exponent_planes(exponents)


def unpacked(codes, scales):
    """MXFP4 storage [..., rows, K / 2] -> float32 [..., rows, K]."""
    k = codes.shape[-1] * 2
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, 32))
    return plain_values(both, exponent_rows(scales, k)).flatten(-2)


def rounded(x):
    """x as it is after a way through MXFP4, in float32."""
    return plain_values(*plain_codes(x.float().unflatten(-1, (-1, 32)))).flatten(-2)


def weights(shape, g):
    """Random weight matrices in MXFP4, made matrix by matrix."""
    matrices, m, k = shape
    codes = torch.empty(matrices, m, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(matrices, -(-k // 256), m, 8, dtype=torch.uint8, device="cuda")
    for i in range(matrices):
        codes[i], scales[i] = packed(torch.randn(m, k, device="cuda", generator=g) * (0.5 / math.sqrt(k)))
    return codes, scales


def activations(rows, d, kind, g):
    """Rows as they leave a norm: of unit size, a few channels much larger."""
    x = torch.randn(rows, d, device="cuda", generator=g)
    x *= 1.0 + 8.0 * (torch.rand(d, device="cuda", generator=g) < 0.01)
    return x.to(TYPES[kind])


def routing(case, g):
    """ids [T, used] int32 of distinct experts, some more asked for than others; -1 in the padded last rows."""
    liked = torch.randn(case["e"], device="cuda", generator=g) * case["skew"]
    noise = -torch.log(-torch.log(torch.rand(case["t"], case["e"], device="cuda", generator=g).clamp(1e-6, 1 - 1e-6)))
    ids = torch.topk(noise + liked, case["used"], dim=1).indices.to(torch.int32)
    ids[case["t"] - case["pad"]:] = -1
    return ids


def plain_sort(ids, e):
    """order [P], rank [T, used], offsets [e + 1]: the pairs by expert, in their own order within one."""
    flat = ids.flatten().long()
    kept = (flat >= 0) & (flat < e)
    key = torch.where(kept, flat, e)
    order = torch.argsort(key, stable=True)
    counts = (key[:, None] == torch.arange(e, device=key.device)).sum(0) if key.numel() * e < 1 << 24 else torch.bincount(key, minlength=e + 1)[:e]
    offsets = torch.nn.functional.pad(torch.cumsum(counts, 0), (1, 0)).to(torch.int32)
    rank = torch.empty_like(order)
    rank[order] = torch.arange(order.numel(), device=order.device)
    rank = torch.where(kept, rank, -1).to(torch.int32).view(ids.shape)
    order = torch.where(kept[order], order, -1).to(torch.int32)
    return order, rank, offsets


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "quantize":
        s["x"] = activations(case["rows"], case["k"], case["type"], g)
        return s
    if case["op"] == "product":
        s["codes"], s["scales"] = (v[0] for v in weights((1, case["m"], case["k"]), g))
        s["x"] = activations(case["t"], case["k"], case["type"], g)
        return s
    s["ids"] = routing(case, g)
    if case["op"] == "dispatch":
        s["x"] = activations(case["t"], case["d"], case["type"], g)
        return s
    s["order"], s["rank"], s["offsets"] = plain_sort(s["ids"], case["e"])
    pairs = case["t"] * case["used"]
    if case["op"] == "experts":
        s["codes"], s["scales"] = weights((case["e"], case["m"], case["k"]), g)
        s["x"] = activations(pairs if case["sorted"] else case["t"], case["k"], case["type"], g)
        return s
    s["ys"] = activations(pairs, case["d"], case["type"], g)
    s["weights"] = torch.softmax(torch.randn(case["t"], case["used"], device="cuda", generator=g), 1)
    if case["back"]:
        s["dy"] = activations(case["t"], case["d"], case["type"], g) * 0.01
    return s


# ---- the operators ---------------------------------------------------------------------------------------------------
def framework(s, case):
    from llamacog_amd import device_ops as ops

    if case["op"] == "quantize":
        return ops.mx4_dequantize(ops.mx4_quantize(s["x"]), s["x"].dtype)
    if case["op"] == "product":
        return ops.mx4_mul_mat(ops.Mx4(s["codes"], s["scales"]), s["x"])
    if case["op"] == "dispatch":
        plan = ops.moe_sort(s["ids"], case["e"])
        return plan.order, plan.rank, plan.offsets, ops.moe_gather(s["x"], plan)
    plan = ops.MoePlan(s["order"], s["rank"], s["offsets"])
    if case["op"] == "experts":
        return ops.mx4_mul_mat_id(ops.Mx4(s["codes"], s["scales"]), s["x"], plan, x_sorted=case["sorted"])
    if case["back"]:
        return ops.moe_combine_back(s["dy"], s["ys"], plan, s["weights"])
    return ops.moe_combine(s["ys"], plan, s["weights"] if case["weighted"] else None)


def run(s):
    case = s["case"]
    if own:
        return framework(s, case)
    if case["op"] == "quantize":
        return rounded(s["x"]).to(s["x"].dtype)
    if case["op"] == "product":
        return (rounded(s["x"]) @ unpacked(s["codes"], s["scales"]).t()).to(s["x"].dtype)
    if case["op"] == "dispatch":
        order, rank, offsets = plain_sort(s["ids"], case["e"])
        xs = s["x"][order.clamp(min=0) // case["used"]]
        return order, rank, offsets, torch.where(order[:, None] < 0, 0, xs)
    if case["op"] == "experts":
        # each expert's rows side by side, as many as the fullest has, multiplied as a batch
        order, offsets = s["order"], s["offsets"].long()
        x = rounded(s["x"])
        at = torch.arange(order.numel(), device=order.device)
        expert = torch.searchsorted(offsets[1:], at, right=True)
        kept = order >= 0
        expert = torch.where(kept, expert, 0)
        place = torch.where(kept, at - offsets[expert], 0)
        most = max(1, int((offsets[1:] - offsets[:-1]).max()))
        row = at if case["sorted"] else order.clamp(min=0) // case["used"]
        side = torch.zeros(case["e"], case["k"], most, device=x.device)
        side[expert[kept], :, place[kept]] = x[row[kept]]
        y = torch.bmm(unpacked(s["codes"], s["scales"]), side)
        return torch.where(kept[:, None], y[expert, :, place], 0.0).to(s["x"].dtype)
    rank, ys = s["rank"].long(), s["ys"]
    kept = (rank >= 0)[..., None]
    rows = torch.where(kept, ys[rank.clamp(min=0)].float(), 0.0)  # [T, used, d]
    if case["back"]:
        dy = s["dy"].float()
        into = torch.where(kept, s["weights"][..., None] * dy[:, None], 0.0)
        dys = torch.zeros_like(ys)
        # a dropped pair writes to a row of its own behind the others, which is cut off
        dys = torch.cat((dys, dys[:1]))
        dys[torch.where(kept[..., 0], rank, ys.shape[0]).flatten()] = into.flatten(0, 1).to(ys.dtype)
        return dys[:-1], (rows * dy[:, None]).sum(-1)
    if case["weighted"]:
        rows = rows * s["weights"][..., None]
    return rows.sum(1).to(ys.dtype)


def work(case):
    size = BYTES[case["type"]]
    if case["op"] == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 * size + 2 * 17 / 32), "flops": 4 * n}
    if case["op"] == "product":
        t, m, k = case["t"], case["m"], case["k"]
        return {"bytes": m * k * 17 / 32 + size * t * (k + m), "flops": 2 * t * m * k}
    pairs, kept = case["t"] * case["used"], (case["t"] - case["pad"]) * case["used"]
    if case["op"] == "experts":
        m, k = case["m"], case["k"]
        asked = case["e"] * (1 - (1 - 1 / case["e"]) ** kept)  # the experts that an even routing asks for
        return {"bytes": asked * m * k * 17 / 32 + size * ((pairs if case["sorted"] else case["t"]) * k + pairs * m) + 4 * pairs,
                "flops": 2 * kept * m * k}
    if case["op"] == "dispatch":
        return {"bytes": 12 * pairs + size * case["d"] * (case["t"] + pairs), "flops": 4 * pairs}
    table = 4 * pairs * (2 if case["weighted"] else 1)
    if case["back"]:
        return {"bytes": table + 4 * pairs + size * case["d"] * (case["t"] + kept + pairs), "flops": 3 * kept * case["d"]}
    return {"bytes": table + size * case["d"] * (case["t"] + kept), "flops": 2 * kept * case["d"]}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact_mx4(x):
    """x [..., K] -> its MXFP4 values in 64 bits: the nearest of the sixteen multiples, ties to the even code."""
    blocks = x.double().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    step = torch.exp2(torch.where(top > 0, torch.floor(torch.log2(top)) - 2, torch.full_like(top, -127.0)).clamp(-127, 127))
    a = blocks.abs() / step
    out = torch.zeros_like(a)
    for low, high, even_high in ((0.0, 0.5, False), (0.5, 1.0, True), (1.0, 1.5, False), (1.5, 2.0, True), (2.0, 3.0, False),
                                 (3.0, 4.0, True), (4.0, 6.0, False)):
        middle = (low + high) / 2
        out = torch.where((a >= middle) if even_high else (a > middle), high, out)
    return (out * torch.sign(blocks) * step).flatten(-2)


def exact_weights(codes, scales):
    """Stored MXFP4 weights [m, K / 2] in 64 bits."""
    k = codes.shape[-1] * 2
    nibbles = torch.empty(codes.shape[0], k, dtype=torch.long, device=codes.device)
    nibbles[:, 0::2], nibbles[:, 1::2] = codes.long() % 16, codes.long() // 16
    size, sign = nibbles % 8, 1.0 - 2.0 * (nibbles // 8)
    value = torch.where(size < 2, size * 0.5, (1 + (size % 2) * 0.5) * torch.exp2((size // 2 - 1).double()))
    block = torch.arange(k, device=codes.device) // 32
    exponent = scales[block // 8, :, block % 8].t()
    return sign * value * torch.exp2(exponent.double() - 127)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return exact_mx4(s["x"])
    if case["op"] == "product":
        x = exact_mx4(s["x"])
        y = torch.empty(case["t"], case["m"], dtype=torch.float64, device="cuda")
        for at in range(0, case["m"], 4096):
            y[:, at:at + 4096] = x @ exact_weights(s["codes"][at:at + 4096], s["scales"][:, at:at + 4096]).t()
        return y
    ids = s["ids"].flatten().tolist()
    pairs = [[p for p, v in enumerate(ids) if v == e] for e in range(case["e"])] if case["e"] * len(ids) < 1 << 24 else None
    if pairs is None:
        pairs = [[] for _ in range(case["e"])]
        for p, v in enumerate(ids):
            if 0 <= v < case["e"]:
                pairs[v].append(p)
    order = [p for those in pairs for p in those]
    held, used = len(order), case["used"]
    at = torch.tensor(order, dtype=torch.long, device="cuda")
    if case["op"] == "dispatch":
        xs = torch.zeros(len(ids), case["d"], dtype=torch.float64, device="cuda")
        xs[:held] = s["x"].double()[at // used]
        return None, None, None, xs
    if case["op"] == "experts":
        x = exact_mx4(s["x"])
        x = x[:held] if case["sorted"] else x[at // used]
        y = torch.zeros(len(ids), case["m"], dtype=torch.float64, device="cuda")
        first = 0
        for e, those in enumerate(pairs):
            if those:
                y[first:first + len(those)] = x[first:first + len(those)] @ exact_weights(s["codes"][e], s["scales"][e]).t()
            first += len(those)
        return y
    # row p of ys belongs to pair order[p]
    ys, w = s["ys"][:held].double(), s["weights"].double().flatten()[at][:, None]
    if case["back"]:
        dy = s["dy"].double()[at // used]
        dys = torch.zeros(len(ids), case["d"], dtype=torch.float64, device="cuda")
        dys[:held] = w * dy
        dw = torch.zeros(len(ids), dtype=torch.float64, device="cuda")
        dw[at] = (dy * ys).sum(1)
        return dys, dw.view(case["t"], used)
    y = torch.zeros(case["t"], case["d"], dtype=torch.float64, device="cuda")
    return y.index_add_(0, at // used, ys * w if case["weighted"] else ys)
