"""Matrices in microscaled 4-bit floating point (MXFP4) and their products: what is measured.

A matrix [rows, width] in MXFP4 holds, for every run of 32 neighbouring elements of a row (the last
one may be shorter), a scale 2^s with s in -127 .. 127 (a byte s + 127; 255 says that the run held
an infinity or a NaN and reads as NaN) and for every element four bits, a sign and one of the
magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Quantising takes s = floor(log2(max |x|)) - 2, at least
-127, divides by 2^s and rounds to the nearest magnitude, ties to the one whose code is even, 6
beyond 6.  All of that is exact but for the one rounding.

Operators, by the "kind" of a case:

* ``round``: rows into MXFP4 and back into their own type;
* ``linear``: rows in bfloat16 times a weight in MXFP4, C = X W^T;
* ``gated``: silu(X Wg^T) * (X Wu^T) for the stacked weight [Wg; Wu] in MXFP4;
* ``linear4``: rows in bfloat16, quantised to MXFP4 within the pass, times a weight in MXFP4.
"""
import math

import torch

own = False

BLOCK = 32
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(kind, rows, width, outputs=0, dtype="bf16", name=None):
    """``dtype``: of the rows of a ``round``, of the result of a ``linear`` (its rows are
    bfloat16).  ``outputs``: rows of the weight (of each of its two halves, for ``gated``)."""
    case = {"kind": kind, "rows": rows, "width": width, "outputs": outputs, "dtype": dtype}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the rows of a decode step of eight sequences before a product of both operands in four bits
        _case("round", 8, 2048, name="round_8x2048"),
        # a tensor of odd sizes that a file stores in 32 bits
        _case("round", 1001, 2739, dtype="f32", name="round_1001x2739_f32"),
        # a whole weight, when a model is loaded (gate and up of a feed-forward of 14,336 on width 4,096)
        _case("round", 28672, 4096, name="round_28672x4096"),
        # one token through the output product of an attention layer of width 2,048
        _case("linear", 1, 2048, 2048, name="linear_1x2048x2048"),
        # a decode step of eight sequences through the down product of that feed-forward
        _case("linear", 8, 14336, 4096, name="linear_8x14336x4096"),
        # logits in 32 bits over a small vocabulary, a ragged batch, sizes that fill no tile
        _case("linear", 37, 2904, 1537, dtype="f32", name="linear_37x2904x1537_f32"),
        # a prompt of 2,048 tokens through the down product
        _case("linear", 2048, 14336, 4096, name="linear_2048x14336x4096"),
        # a decode step of sixteen sequences through gate and up
        _case("gated", 16, 4096, 14336, name="gated_16x4096x14336"),
        # a prompt of 1,000 tokens through gate and up of a feed-forward of 8,192 on width 2,048
        _case("gated", 1000, 2048, 8192, name="gated_1000x2048x8192"),
        # a large decode batch through a stacked query, key and value product, both operands in four bits
        _case("linear4", 128, 4096, 6144, name="linear4_128x4096x6144"),
        # a ragged prompt, odd sizes throughout
        _case("linear4", 333, 1999, 2051, name="linear4_333x1999x2051"),
        # prompts of 4,096 tokens through a stacked gate and up product
        _case("linear4", 4096, 4096, 28672, name="linear4_4096x4096x28672"),
    ]


def _spread(rng, low, high):
    """A whole number between ``low`` and ``high``, even over its logarithm; three in four are
    multiples of 32 where they are large enough, as a model's sizes are."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if n >= 64 and rng.random() < 0.75:
        n = n // 32 * 32
    return max(low, min(high, n))


def draw(rng):
    kind = rng.choice(("round", "linear", "linear", "gated", "linear4"))
    if kind == "round":
        rows, width = _spread(rng, 1, 28672), _spread(rng, 1, 8192)
        while rows * width > 28672 * 4096:
            rows = _spread(rng, 1, 28672)
        return _case(kind, rows, width, dtype=rng.choice(("bf16", "f32")))
    most = 28672 if kind != "gated" else 14336
    rows, width, outputs = _spread(rng, 1, 4096), _spread(rng, 32, 14336), _spread(rng, 16, most)
    while outputs * width > 14336 * 4096:
        width, outputs = _spread(rng, 32, 14336), _spread(rng, 16, most)
    if rng.random() < 0.4:
        rows = _spread(rng, 1, 64)              # decode steps: as often as all the others
    return _case(kind, rows, width, outputs, rng.choice(("bf16", "bf16", "f32")) if kind == "linear" else "bf16")


# ---- inputs
def _normal(shape, seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 16 + salt)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(case, seed):
    """Activations: normal, every row of a size of its own, and one channel in 64 eight times as
    large, as the stream of a decoder has them."""
    m, k = case["rows"], case["width"]
    x = _normal((m, k), seed, 1)
    x *= torch.exp(0.5 * _normal((m, 1), seed, 2))
    loud = (_normal((1, k), seed, 3) > 2.15).float()
    x *= 1.0 + 7.0 * loud
    return x.to(_TYPES[case["dtype"]] if case["kind"] == "round" else torch.bfloat16)


def _weight_codes(case, seed):
    """A weight as a file in MXFP4 holds it: codes [n, ceil(k / 2)] (the even element of a pair in
    the low half of the byte) and scales [n, ceil(k / 32)]."""
    n = case["outputs"] * (2 if case["kind"] == "gated" else 1)
    w = _normal((n, case["width"]), seed, 4) * case["width"] ** -0.5
    codes, scales = _quantise(w)
    if codes.shape[1] % 2:
        codes = torch.nn.functional.pad(codes, (0, 1))
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), scales


def prepare(case, seed):
    state = {"kind": case["kind"], "x": _rows(case, seed), "dtype": _TYPES[case["dtype"]]}
    if case["kind"] != "round":
        state["codes"], state["scales"] = _weight_codes(case, seed)
    if own:
        from libllm_amd.hip import HipOps
        state["ops"] = HipOps()
        if case["kind"] != "round":
            # the weight laid out for the matrix cores, once, as a model keeps it
            state["weight"] = state["ops"].mx4_from_codes(state["codes"], state["scales"], case["width"])
    return state


# ---- the operators in plain form
def _power(s):
    """2^s in 64 bits for whole s, from its bits."""
    return ((s.to(torch.int64) + 1023) << 52).view(torch.float64)


def _quantise(x):
    """(codes [m, k], scales [m, ceil(k / 32)]), bytes; the borders are compared in 64 bits."""
    m, k = x.shape
    blocks = -(-k // BLOCK)
    xf = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - k)).view(m, blocks, BLOCK)
    largest = xf.abs().amax(dim=-1)
    finite = torch.isfinite(xf).all(dim=-1)
    s = torch.frexp(torch.where(finite, largest, torch.ones_like(largest)).double())[1].to(torch.int32) - 3
    s = torch.where(largest == 0, torch.full_like(s, -127), s).clamp(min=-127)
    a = xf.abs().double() * _power(-s)[..., None]
    code = (a > 0.25).to(torch.uint8)
    for border, inclusive in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= border) if inclusive else (a > border)
    code |= torch.signbit(xf).to(torch.uint8) << 3
    scales = torch.where(finite, s + 127, torch.full_like(s, 255)).to(torch.uint8)
    return code.view(m, blocks * BLOCK)[:, :k].contiguous(), scales


def _values(codes, scales):
    """The numbers that codes [m, k] and scales stand for, in 32 bits."""
    m, k = codes.shape
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat([table, -table])
    scale = _power(scales.to(torch.int32) - 127).float()
    scale = torch.where(scales == 255, torch.full_like(scale, float("nan")), scale)
    return table[codes.int()] * scale.repeat_interleave(BLOCK, dim=1)[:, :k]


def _weight_values(state, width):
    packed = state["codes"]
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).view(packed.shape[0], -1)[:, :width]
    return _values(codes, state["scales"])


def run(state):
    kind, x = state["kind"], state["x"]
    if own:
        ops = state["ops"]
        if kind == "round":
            return ops.dequantize_mx4(ops.quantize_mx4(x), x.dtype)
        if kind == "gated":
            return ops.linear_swiglu(x, state["weight"])
        if kind == "linear4":
            return ops.linear(ops.quantize_mx4(x), state["weight"], None, state["dtype"])
        return ops.linear(x, state["weight"], None, state["dtype"])
    if kind == "round":
        return _values(*_quantise(x)).to(x.dtype)
    rows = _values(*_quantise(x)) if kind == "linear4" else x.float()
    y = torch.matmul(rows, _weight_values(state, x.shape[1]).t())
    if kind == "gated":
        gate, up = y.chunk(2, dim=1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(state["dtype"])


def work(case):
    kind, m, k, n = case["kind"], case["rows"], case["width"], case["outputs"]
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "round":
        return {"bytes": 2 * m * k * size, "flops": 4 * m * k}
    stacked = 2 * n if kind == "gated" else n
    weight = stacked * (-(-k // 2) + -(-k // BLOCK))
    return {"bytes": 2 * m * k + weight + m * n * size, "flops": 2 * m * k * stacked}


# ---- the same from the definition, in 64 bits
def _round_to_grid(x):
    """Rows rounded to MXFP4 by the spacing of its numbers: below 2 they lie half a unit apart,
    from 2 on one unit, from 4 on two, and none lies beyond 6."""
    m, k = x.shape
    out = torch.empty((m, k), dtype=torch.float64, device=x.device)
    for first in range(0, k, BLOCK):
        part = x[:, first:first + BLOCK].double()
        top = part.abs().max(dim=1, keepdim=True).values
        unit = torch.ones_like(top)
        ok = torch.isfinite(top) & (top > 0)
        exponent = torch.floor(torch.log2(torch.where(ok, top, unit)))
        # (the logarithm may round up to a whole number just below a power of two)
        exponent = torch.where(torch.where(ok, top, unit) < torch.exp2(exponent), exponent - 1, exponent)
        scale = torch.exp2(torch.clamp(exponent - 2, min=-127.0))
        y = part / scale
        size = y.abs()
        step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0)).to(torch.float64)
        y = torch.clamp(torch.round(y / step) * step, -6.0, 6.0) * scale
        out[:, first:first + BLOCK] = torch.where(torch.isfinite(top), y, torch.full_like(y, float("nan")))
    return out


def _weight_exact(packed, scales, k):
    n = packed.shape[0]
    out = torch.empty((n, packed.shape[1], 2), dtype=torch.float64, device=packed.device)
    for half in (0, 1):
        code = (packed >> (4 * half)) & 15
        e, mantissa = ((code >> 1) & 3).double(), (code & 1).double()
        size = torch.where(e > 0, torch.exp2(e - 1) * (1 + 0.5 * mantissa), 0.5 * mantissa)
        out[:, :, half] = torch.where(code > 7, -size, size)
    w = out.view(n, -1)[:, :k].contiguous()
    for block in range(scales.shape[1]):
        w[:, block * BLOCK:(block + 1) * BLOCK] *= torch.exp2(scales[:, block:block + 1].double() - 127.0)
    return w


def exact(case, seed):
    x = _rows(case, seed)
    if case["kind"] == "round":
        return _round_to_grid(x)
    w = _weight_exact(*_weight_codes(case, seed), case["width"])
    rows = _round_to_grid(x) if case["kind"] == "linear4" else x.double()
    if case["kind"] == "gated":
        n = case["outputs"]
        gate = rows @ w[:n].t()
        return gate * torch.sigmoid(gate) * (rows @ w[n:].t())
    return rows @ w.t()
