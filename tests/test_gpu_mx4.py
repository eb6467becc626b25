"""Matrices in MXFP4 and their products against plain implementations in float64: a quantiser, a
reader of the tiles and a product written here with numpy, from the format's definition."""
import numpy as np
import pytest
import torch

from libllm_amd.errors import KernelError

pytestmark = pytest.mark.gpu

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
HALF_BF16, HALF_F32 = 2.0 ** -8, 2.0 ** -24        # the most a rounding is off, relative to the value


@pytest.fixture(scope="module")
def ops():
    from libllm_amd.hip import HipOps
    return HipOps()


# ------------------------------------------------------------------------------- plain forms
def quantise(x):
    """Codes [m, k] and scales [m, ceil(k / 32)] of a float64 matrix, block by block."""
    x = np.asarray(x, dtype=np.float64)
    m, k = x.shape
    blocks = -(-k // 32)
    codes = np.zeros((m, k), dtype=np.uint8)
    scales = np.zeros((m, blocks), dtype=np.uint8)
    for b in range(blocks):
        part = x[:, 32 * b:32 * b + 32]
        top = np.abs(part).max(axis=1)
        bad = ~np.isfinite(part).all(axis=1)
        _, e = np.frexp(np.where(bad | (top == 0), 1.0, top))       # top = f 2^e with f in [0.5, 1)
        s = np.maximum(np.where(top == 0, -127, e - 1 - 2), -127)
        a = np.ldexp(np.abs(np.where(np.isfinite(part), part, 0.0)), -s[:, None])
        # the nearest of the grid; at equal distance the one whose code is even
        d = np.abs(a[:, :, None] - GRID)
        near = d == d.min(axis=2, keepdims=True)
        pick = np.where(near, np.arange(8) % 2 * 8 + np.arange(8), 99).argmin(axis=2)
        codes[:, 32 * b:32 * b + 32] = pick + 8 * np.signbit(part)
        scales[:, b] = np.where(bad, 255, s + 127)
    return codes, scales


def values(codes, scales):
    k = codes.shape[1]
    v = np.where(codes > 7, -1.0, 1.0) * GRID[codes & 7]
    s = np.ldexp(1.0, scales.astype(np.int64) - 127)
    s = np.where(scales == 255, np.nan, s)
    return v * np.repeat(s, 32, axis=1)[:, :k]


def file_form(codes, scales):
    """Two codes a byte, the even element in the low half."""
    if codes.shape[1] % 2:
        codes = np.pad(codes, ((0, 0), (0, 1)))
    return torch.from_numpy(codes[:, 0::2] | (codes[:, 1::2] << 4)), torch.from_numpy(scales)


def rows_of(q):
    """(codes, scales) by rows, read out of the tiles by the layout's definition (csrc/mx4.h)."""
    m, k = q.shape
    tiles, quads = -(-m // 16), -(-k // 512)
    units = 4 * quads
    c = q.codes.cpu().numpy().reshape(tiles, units, 4, 16, 16)            # tile, unit, block, row, byte
    c = np.stack([c & 15, c >> 4], axis=-1).reshape(tiles, units, 4, 16, 32)
    c = c.transpose(0, 3, 1, 2, 4).reshape(tiles * 16, units * 128)
    s = q.scales.cpu().numpy().reshape(tiles, quads, 4, 16, 4)            # tile, quad, block, row, unit of the quad
    s = s.transpose(0, 3, 1, 4, 2).reshape(tiles * 16, quads * 16)[:, :units * 4]
    return c, s


def normal(shape, seed, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def weight(n, k, seed):
    codes, scales = quantise(normal((n, k), seed, k ** -0.5).double().numpy())
    return codes, scales, values(codes, scales)


def held(n, k, seed):
    codes, scales, w = weight(n, k, seed)
    packed, s = file_form(codes, scales)
    return packed, s, w


def bound(x, w, k, dtype):
    """What a product summed in 32 bits may be off by, per element.  Products of bfloat16 and MXFP4
    numbers (8 and 2 bits) are exact in 32 bits; k of them are added, in whatever order, by at most
    k additions, each off by at most 2^-24 of a partial sum, which is at most sum |x| |w|.  The
    matrix cores may cut off instead of rounding: twice that.  Then one rounding of the result."""
    magnitude = np.abs(x) @ np.abs(w).T
    exact = np.abs(x @ w.T)
    err = 2 * k * HALF_F32 * magnitude
    half = HALF_BF16 if dtype == torch.bfloat16 else HALF_F32
    return err + half * (exact + err) + 1e-38


def gate(act, g, u):
    if act == "relu":
        return np.maximum(g, 0) * u
    if act == "gelu_tanh":
        return 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3))) * u
    return g / (1 + np.exp(-g)) * u


# ------------------------------------------------------------------------------- conversions
SIZES = [(1, 1), (1, 32), (2, 31), (3, 33), (16, 128), (17, 129), (5, 500), (40, 512), (33, 1030), (130, 96)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k", SIZES)
def test_quantize(ops, m, k, dtype):
    x = normal((m, k), 100 * m + k, 3.0, dtype)
    x[0, 0] = 0.0
    if m > 2:
        x[1] = 0.0
        x[2] *= 2.0 ** -100
    codes, scales = quantise(x.double().numpy())
    q = ops.quantize_mx4(x.cuda())
    assert q.shape == (m, k)
    got_codes, got_scales = rows_of(q)
    blocks = scales.shape[1]
    assert np.array_equal(got_scales[:m, :blocks], scales)
    assert np.array_equal(got_codes[:m, :k], codes)
    # what pads the tiles is zero
    assert not got_codes[m:].any() and not got_codes[:, k:].any()
    assert not got_scales[m:].any() and not got_scales[:, blocks:].any()
    for out in (torch.float32, torch.bfloat16):
        back = ops.dequantize_mx4(q, out)
        assert back.dtype == out and back.shape == (m, k)
        assert np.array_equal(back.double().cpu().numpy(), values(codes, scales))


def test_quantize_ties_limits_and_signs(ops):
    # one block per row, its largest magnitude 4 .. 8 in units of the scale
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.99, 4.0]
    row = np.zeros(32)
    row[:10], row[10:20] = ties, [-t for t in ties]
    row[20] = -0.0
    above = np.nextafter(row.astype(np.float32), np.float32(np.inf)).astype(np.float64)
    below = np.nextafter(row.astype(np.float32), np.float32(-np.inf)).astype(np.float64)
    tiny = np.ldexp(row, -130)                                    # scale at its least, subnormal elements
    huge = np.ldexp(row, 125)
    x = np.stack([row, above, below, tiny, huge, np.zeros(32), np.full(32, 2.0 ** -149), np.full(32, -3.4028234e38)])
    codes, scales = quantise(x.astype(np.float32).astype(np.float64))
    q = ops.quantize_mx4(torch.from_numpy(x.astype(np.float32)).cuda())
    got_codes, got_scales = rows_of(q)
    assert np.array_equal(got_scales[:8, :1], scales)
    assert np.array_equal(got_codes[:8, :32], codes)
    assert np.array_equal(ops.dequantize_mx4(q, torch.float32).double().cpu().numpy(), values(codes, scales))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_quantize_not_finite(ops, bad, dtype):
    """A block with an infinity or a NaN reads as NaN; its neighbours are untouched."""
    x = normal((20, 200), 4, dtype=dtype)
    x[3, 40] = x[19, 199] = bad
    back = ops.dequantize_mx4(ops.quantize_mx4(x.cuda()), torch.float32).cpu()
    want = values(*quantise(x.double().numpy()))
    assert torch.isnan(back[3, 32:64]).all() and torch.isnan(back[19, 192:]).all()
    assert int(torch.isnan(back).sum()) == 32 + 8
    assert np.array_equal(back.double().numpy(), want, equal_nan=True)


def test_quantising_again_changes_nothing(ops):
    q = ops.quantize_mx4(normal((50, 700), 9, dtype=torch.bfloat16).cuda())
    again = ops.quantize_mx4(ops.dequantize_mx4(q, torch.bfloat16))
    assert torch.equal(q.codes, again.codes) and torch.equal(q.scales, again.scales)


def test_quantize_rows_that_lie_apart(ops):
    big = normal((37, 300), 5, dtype=torch.bfloat16).cuda()
    for view in (big[:, :200], big[:, 3:190], big[::2, 64:128], big[5:6, 1:2]):
        q, c = ops.quantize_mx4(view), ops.quantize_mx4(view.contiguous())
        assert torch.equal(q.codes, c.codes) and torch.equal(q.scales, c.scales)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ld", [304, 300, 302, 301])
def test_quantize_ends_of_rows(ops, ld, dtype):
    """Rows that begin at every alignment and end anywhere in a piece of 8, numbers behind them: as if alone."""
    big = normal((19, ld), ld, dtype=dtype).cuda()
    for k in (1, 7, 8, 9, 127, 132, 187, 260):
        codes, scales = quantise(big[:, :k].double().cpu().numpy())
        got = rows_of(ops.quantize_mx4(big[:, :k]))
        assert np.array_equal(got[0][:19, :k], codes) and not got[0][:, k:].any()
        assert np.array_equal(got[1][:19, :scales.shape[1]], scales) and not got[1][:, scales.shape[1]:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_reading_back_more_than_the_caches_hold(ops, dtype):
    rows, width = (12304, 4112) if dtype == torch.float32 else (24600, 4104)
    q = ops.quantize_mx4(torch.randn((rows, width), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda"))
    got = ops.dequantize_mx4(q, dtype)
    assert got.numel() * got.element_size() >= 192 << 20
    part = ops.dequantize_mx4(q.leading_rows(12288), dtype)
    assert torch.equal(got[:12288], part)
    again = ops.quantize_mx4(got)
    assert torch.equal(q.codes, again.codes) and torch.equal(q.scales, again.scales)


@pytest.mark.parametrize("n,k", [(1, 1), (16, 32), (33, 63), (18, 160), (50, 1001)])
def test_from_codes(ops, n, k):
    rng = np.random.default_rng(n + k)
    codes = rng.integers(0, 16, (n, k), dtype=np.uint8)
    scales = rng.integers(100, 150, (n, -(-k // 32)), dtype=np.uint8)
    scales[0, 0] = 255
    packed, s = file_form(codes, scales)
    padded = torch.full((n, packed.shape[1] + 5), 0xAB, dtype=torch.uint8)       # more columns than the rows need
    padded[:, :packed.shape[1]] = packed
    for held in (packed.cuda(), padded.cuda(), padded.cuda()[:, :packed.shape[1]]):
        q = ops.mx4_from_codes(held, s.cuda(), k)
        got_codes, got_scales = rows_of(q)
        assert np.array_equal(got_codes[:n, :k], codes) and not got_codes[:, k:].any() and not got_codes[n:].any()
        assert np.array_equal(got_scales[:n, :s.shape[1]], scales)
        assert np.array_equal(ops.dequantize_mx4(q, torch.float32).double().cpu().numpy(), values(codes, scales),
                              equal_nan=True)
    if k % 2 == 0:
        assert ops.mx4_from_codes(packed.cuda(), s.cuda()).shape == (n, k)


# ------------------------------------------------------------------------------- products
PRODUCTS = [(1, 16, 32), (1, 64, 2048), (2, 17, 40), (5, 100, 129), (16, 48, 1000), (17, 33, 256), (31, 80, 1023),
            (33, 130, 512), (64, 96, 640), (65, 40, 1152), (100, 257, 384), (129, 64, 2000), (200, 300, 136),
            (257, 520, 1024), (520, 272, 264)]


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear(ops, m, n, k, out):
    x = normal((m, k), 7 * m + k, dtype=torch.bfloat16)
    codes, scales, w = weight(n, k, n + k)
    packed, s = file_form(codes, scales)
    q = ops.mx4_from_codes(packed.cuda(), s.cuda(), k)
    got = ops.linear(x.cuda(), q, None, out)
    assert got.dtype == out and got.shape == (m, n)
    xd = x.double().numpy()
    diff = np.abs(got.double().cpu().numpy() - xd @ w.T)
    assert (diff <= bound(xd, w, k, out)).all(), (diff - bound(xd, w, k, out)).max()


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear_both_in_mxfp4(ops, m, n, k, out):
    x = normal((m, k), 7 * m + k, dtype=torch.bfloat16)
    codes, scales, w = weight(n, k, n + k)
    packed, s = file_form(codes, scales)
    q = ops.mx4_from_codes(packed.cuda(), s.cuda(), k)
    got = ops.linear(ops.quantize_mx4(x.cuda()), q, None, out)
    assert got.dtype == out and got.shape == (m, n)
    xd = values(*quantise(x.double().numpy()))
    diff = np.abs(got.double().cpu().numpy() - xd @ w.T)
    assert (diff <= bound(xd, w, k, out)).all(), (diff - bound(xd, w, k, out)).max()


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_bias(ops, m, four):
    n, k = 77, 224
    x = normal((m, k), m, dtype=torch.bfloat16)
    b = normal((n,), 3)
    codes, scales, w = weight(n, k, 6)
    packed, s = file_form(codes, scales)
    q = ops.mx4_from_codes(packed.cuda(), s.cuda(), k)
    rows = ops.quantize_mx4(x.cuda()) if four else x.cuda()
    xd = values(*quantise(x.double().numpy())) if four else x.double().numpy()
    got = ops.linear(rows, q, b.cuda(), torch.float32).double().cpu().numpy()
    # one more addition
    lim = bound(xd, w, k, torch.float32) + 2 * HALF_F32 * (np.abs(xd @ w.T) + np.abs(b.double().numpy()))
    assert (np.abs(got - (xd @ w.T + b.double().numpy())) <= lim).all()


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("m,inter,k", [(1, 16, 64), (3, 48, 200), (16, 33, 128), (20, 112, 600), (64, 80, 333),
                                       (90, 17, 64), (150, 256, 512), (300, 144, 1024)])
def test_gated(ops, m, inter, k, four, act):
    x = normal((m, k), m + inter, dtype=torch.bfloat16)
    codes, scales, w = weight(2 * inter, k, k + inter)
    packed, s = file_form(codes, scales)
    q = ops.mx4_from_codes(packed.cuda(), s.cuda(), k)
    rows = ops.quantize_mx4(x.cuda()) if four else x.cuda()
    xd = values(*quantise(x.double().numpy())) if four else x.double().numpy()
    got = ops.linear_swiglu(rows, q, torch.bfloat16, act)
    assert got.dtype == torch.bfloat16 and got.shape == (m, inter)
    y = xd @ w.T
    g, u = y[:, :inter], y[:, inter:]
    want = gate(act, g, u)
    # gate and up are off by what a float32 sum may be (dg, du); |act'| <= 1.2 and |act(g)| <= |g|, the
    # activation itself within 2^-16 of |g| (exp and tanh of the device, the cancellation in 1 + tanh
    # near -1), then one rounding of the result
    d = bound(xd, w, k, torch.float32)
    dg, du = d[:, :inter], d[:, inter:]
    lim = 1.2 * dg * (np.abs(u) + du) + (np.abs(g) + dg) * du + 2.0 ** -16 * np.abs(g) * np.abs(u)
    lim = lim + HALF_BF16 * (np.abs(want) + lim) + 1e-38
    assert (np.abs(got.double().cpu().numpy() - want) <= lim).all()


FORMS = {False: (0, 1, 2, 3, 4), True: (0, 1, 2, 3, 4)}


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,inter,k", [(1, 16, 32), (3, 33, 32), (24, 80, 64), (40, 112, 64), (70, 33, 1100), (300, 272, 64)])
def test_gated_with_numbers_whose_product_overflows(ops, m, inter, k, out):
    """Gates of -2^70 k and ups of 2^70 k, whose product 32 bits do not hold: SiLU of such a gate is zero,
    and with it the result.  With up zero as well, and with small gates in every third column, ordinary ones."""
    g, u = np.full(inter, -1.0), np.ones(inter)
    u[1::5] = 0.0
    g[::3] = 2.0 ** -72 / k
    u[::3] = 2.0 ** -70 / k
    # one number a row, at the exponent that its block's scale gives it: 4 2^(e - 2)
    rows = torch.tensor(np.repeat(np.concatenate([g, u])[:, None], k, 1), dtype=torch.float32).cuda()
    x = torch.full((m, k), 2.0 ** 70, dtype=torch.bfloat16).cuda()
    w = ops.quantize_mx4(rows)
    held = ops.dequantize_mx4(w, torch.float32).double().cpu().numpy().sum(1) * 2.0 ** 70
    gs, us = held[:inter], held[inter:]
    want = np.where(gs < -700, 0.0, gs / (1 + np.exp(-np.maximum(gs, -700)))) * us
    got = ops.linear_swiglu(x, w, out).double().cpu().numpy()
    assert got.shape == (m, inter)
    half = HALF_BF16 if out == torch.bfloat16 else HALF_F32
    # equal terms: at most k additions a sum; the exponential, the division and two products are a few
    # units of 2^-24 each, taken for 16
    assert (np.abs(got - want) <= (half + (2 * k * 2 + 16) * HALF_F32) * np.abs(want)).all()


@pytest.mark.parametrize("four,form", [(f, i) for f in (False, True) for i in FORMS[f]])
@pytest.mark.parametrize("m,n,k,ks", [(1, 16, 100, 1), (70, 130, 128, 1), (260, 300, 700, 1), (300, 520, 1500, 2),
                                      (257, 272, 2600, 3), (40, 2064, 4200, 9), (530, 80, 3000, 1)])
def test_every_form_of_the_product_for_many_rows(ops, monkeypatch, m, n, k, ks, four, form):
    """At sizes that fill no block, with K of less than a tile, of odd numbers of tiles, and in slices of
    which the last is short; plain, with a bias, and gated."""
    monkeypatch.setattr(ops, "_mx4_plan", lambda *sizes: (form, ks))
    x, b = normal((m, k), m + k, dtype=torch.bfloat16), normal((n,), 3)
    packed, s, w = held(n, k, n + k)
    q = ops.mx4_from_codes(packed.cuda(), s.cuda(), k)
    rows = ops.quantize_mx4(x.cuda()) if four else x.cuda()
    xd = values(*quantise(x.double().numpy())) if four else x.double().numpy()
    y, lim = xd @ w.T, bound(xd, w, k, torch.float32)
    got = ops.linear(rows, q, b.cuda(), torch.float32).double().cpu().numpy()
    more = 2 * HALF_F32 * (np.abs(y) + np.abs(b.double().numpy()))
    assert (np.abs(got - (y + b.double().numpy())) <= lim + more).all()
    out = ops.linear(rows, q, None, torch.bfloat16).double().cpu().numpy()
    assert (np.abs(out - y) <= bound(xd, w, k, torch.bfloat16)).all()
    if n % 32 == 0:
        sw = ops.linear_swiglu(rows, q).double().cpu().numpy()
        g, u, dg, du = y[:, :n // 2], y[:, n // 2:], lim[:, :n // 2], lim[:, n // 2:]
        ls = 1.2 * dg * (np.abs(u) + du) + (np.abs(g) + dg) * du + 2.0 ** -16 * np.abs(g) * np.abs(u)
        assert (np.abs(sw - gate("silu", g, u)) <= ls + HALF_BF16 * (np.abs(gate("silu", g, u)) + ls) + 1e-38).all()


def test_a_row_is_the_same_whatever_the_batch(ops):
    """Up to 32 rows, which one kernel takes."""
    x = normal((32, 1056), 8, dtype=torch.bfloat16).cuda()
    q = ops.quantize_mx4(normal((208, 1056), 9, dtype=torch.bfloat16).cuda())
    whole = ops.linear(x, q, None, torch.float32)
    for m0, m in ((0, 1), (3, 4), (5, 7), (16, 16), (10, 22), (1, 31)):
        assert torch.equal(ops.linear(x[m0:m0 + m], q, None, torch.float32), whole[m0:m0 + m])


def test_rows_that_are_not_finite_stay_in_their_rows(ops):
    k, n = 200, 48
    x = normal((20, k), 8, dtype=torch.bfloat16)
    x[4, 0], x[9, 199] = float("inf"), float("nan")
    codes, scales, w = weight(n, k, 2)
    packed, s = file_form(codes, scales)
    q = ops.mx4_from_codes(packed.cuda(), s.cuda(), k)
    for rows in (x.cuda(), ops.quantize_mx4(x.cuda())):
        got = ops.linear(rows, q, None, torch.float32).cpu()
        assert torch.isfinite(got[[i for i in range(20) if i not in (4, 9)]]).all()
        assert not torch.isfinite(got[4]).any() and torch.isnan(got[9]).all()


def test_a_block_of_the_weight_that_is_nan(ops):
    k, n = 160, 40
    codes, scales, _ = weight(n, k, 2)
    scales[7, 2] = 255
    packed, s = file_form(codes, scales)
    q = ops.mx4_from_codes(packed.cuda(), s.cuda(), k)
    x = normal((5, k), 8, dtype=torch.bfloat16).cuda()
    for rows in (x, ops.quantize_mx4(x)):
        got = ops.linear(rows, q, None, torch.float32).cpu()
        assert torch.isnan(got[:, 7]).all() and int(torch.isnan(got).sum()) == 5


def test_rows_that_lie_apart_or_askew(ops):
    big = normal((40, 300), 5, dtype=torch.bfloat16).cuda()
    q = ops.quantize_mx4(normal((70, 130), 6).cuda())
    for view in (big[:, :130], big[:, 1:131], big[::3, 8:138], big[:1, 5:135]):
        assert torch.equal(ops.linear(view, q, None, torch.float32), ops.linear(view.contiguous(), q, None, torch.float32))


@pytest.mark.parametrize("far,k", [((1 << 22) + 512, 256), ((1 << 22) + 128, (1 << 22) + 128), ((1 << 22) + 8, 200)])
def test_rows_that_lie_far_apart(ops, far, k):
    """A block's rows, and a width, that the product for many rows cannot reach with 32-bit offsets: numbers
    of -1, 0 and 1, whose sums 32 bits hold."""
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randint(-1, 2, (70, far), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)[:, :k]
    w = torch.randint(-1, 2, (32, k), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    got = ops.linear(x, ops.quantize_mx4(w), None, torch.float32)
    want = torch.zeros((70, 32), dtype=torch.float64, device="cuda")
    for at in range(0, k, 1 << 18):
        want += x[:, at:at + (1 << 18)].double() @ w[:, at:at + (1 << 18)].double().t()
    assert torch.equal(got.double(), want)


def test_many_rows_that_are_padded(ops):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-4, 5, (70001, 3), generator=g, device="cuda").to(torch.bfloat16)
    w = torch.tensor([[1.0, -2.0, 3.0], [0.5, 6.0, -4.0]], device="cuda")
    got = ops.linear(x, ops.quantize_mx4(w), None, torch.float32)
    assert torch.equal(got.double(), x.double() @ w.double().t())


def test_no_rows(ops):
    q = ops.quantize_mx4(normal((32, 64), 1).cuda())
    none = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    assert ops.linear(none, q, None, torch.bfloat16).shape == (0, 32)
    assert ops.linear_swiglu(none, q).shape == (0, 16)


def test_leading_rows(ops):
    w = normal((64, 200), 1).cuda()
    q = ops.quantize_mx4(w)
    x = normal((5, 200), 2, dtype=torch.bfloat16).cuda()
    assert torch.equal(ops.linear(x, q.leading_rows(32), None, torch.float32), ops.linear(x, q, None, torch.float32)[:, :32])
    with pytest.raises(KernelError):
        q.leading_rows(20)
    with pytest.raises(KernelError):
        q.leading_rows(80)


def test_refusals(ops):
    w = normal((32, 64), 1).cuda()
    q = ops.quantize_mx4(w)
    x = normal((4, 64), 2, dtype=torch.bfloat16).cuda()
    codes = torch.zeros((4, 16), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((4, 1), dtype=torch.uint8, device="cuda")
    bad = [
        lambda: ops.quantize_mx4(w.half()),
        lambda: ops.quantize_mx4(w.t()),
        lambda: ops.quantize_mx4(w[0]),
        lambda: ops.quantize_mx4(w.cpu()),
        lambda: ops.quantize_mx4(w[:0]),
        lambda: ops.quantize_mx4(w[:, :0]),
        lambda: ops.dequantize_mx4(q, torch.float16),
        lambda: ops.dequantize_mx4(w, torch.float32),
        lambda: ops.mx4_from_codes(codes.int(), scales),
        lambda: ops.mx4_from_codes(codes, scales.float()),
        lambda: ops.mx4_from_codes(codes, scales, 33),
        lambda: ops.mx4_from_codes(codes, scales, 0),
        lambda: ops.mx4_from_codes(codes, scales[:3]),
        lambda: ops.mx4_from_codes(codes.cpu(), scales),
        lambda: ops.linear(x.float(), q, None, torch.float32),
        lambda: ops.linear(x[:, :32], q, None, torch.float32),
        lambda: ops.linear(x.t().contiguous().t(), q, None, torch.float32),
        lambda: ops.linear(x.cpu(), q, None, torch.float32),
        lambda: ops.linear(x, q, None, torch.float16),
        lambda: ops.linear(x, q, torch.zeros(31, device="cuda"), torch.float32),
        lambda: ops.linear(ops.quantize_mx4(x), w.bfloat16(), None, torch.float32),
        lambda: ops.linear_swiglu(ops.quantize_mx4(x), w.bfloat16()),
        lambda: ops.linear_swiglu(x, ops.quantize_mx4(w[:31])),
        lambda: ops.linear_swiglu(x, q, torch.bfloat16, "tanh"),
        lambda: ops.linear_swiglu(x[:, :32], q),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(KernelError):
            call()
            pytest.fail("call %d was not refused" % i)


def test_quantise_and_multiply_replayed_from_a_graph(ops):
    """A run as a step makes it (rows rounded, gated product, product) captured once and replayed
    over new rows, with eager work between the replays."""
    gate_up = ops.quantize_mx4(normal((2 * 96, 128), 1, 0.1).cuda())
    down = ops.quantize_mx4(normal((128, 96), 2, 0.1).cuda())
    x = torch.empty((24, 128), dtype=torch.bfloat16, device="cuda")
    held = {}

    def step():
        h = ops.linear_swiglu(x, gate_up)
        held["out"] = ops.linear(ops.quantize_mx4(h), down, None, torch.bfloat16)
    x.normal_()
    graph = ops.capture(step)
    replayed = held["out"]
    for i in range(4):
        x.copy_(normal((24, 128), 50 + i))
        graph.replay()
        got = replayed.clone()
        step()
        assert torch.equal(got, held["out"])
        torch.cuda.synchronize()


def test_on_another_stream(ops):
    w, x = normal((64, 256), 1).cuda(), normal((3, 256), 2, dtype=torch.bfloat16).cuda()
    want = ops.linear(x, ops.quantize_mx4(w), None, torch.float32)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.linear(x, ops.quantize_mx4(w), None, torch.float32)
    side.synchronize()
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------- as a layer uses them
@pytest.mark.parametrize("m,n,k", [(1, 64, 96), (3, 77, 200), (16, 2048, 520), (20, 48, 1000), (32, 100, 64),
                                   (50, 4112, 136), (70, 64, 2100), (140, 96, 5000)])
def test_added_into_the_stream(ops, m, n, k):
    """With ``residual`` the product for few rows adds into it; otherwise what comes back is the
    product, or its slices of K, and the norm kernel adds them."""
    packed, s, w = held(n, k, n + m)
    q = ops.mx4_from_codes(packed.cuda(), s.cuda(), k)
    x, res = normal((m, k), m, dtype=torch.bfloat16), normal((m, n), n, 3.0)
    stream = res.cuda()
    got = ops.linear(x.cuda(), q, None, torch.bfloat16, residual=stream)
    xd, rd = x.double().numpy(), res.double().numpy()
    lim = bound(xd, w, k, torch.float32)
    if got is None:
        assert ops._mx4_plan(m, n, n, k, False)[0] < 0
        total = stream.double().cpu().numpy()
    else:
        assert torch.equal(stream.cpu(), res)
        if got.dim() == 2:
            lim = bound(xd, w, k, torch.bfloat16)
        total = rd + got.double().cpu().numpy().reshape(-1, m, n).sum(0)
    # one more addition in 32 bits, and one for every slice beside the first (less than ten)
    lim = lim + 10 * HALF_F32 * (np.abs(rd) + np.abs(xd) @ np.abs(w).T)
    assert (np.abs(total - (rd + xd @ w.T)) <= lim).all()


@pytest.mark.parametrize("m", [1, 2, 7, 8, 16])
@pytest.mark.parametrize("n,k,inter", [(64, 96, 32), (512, 200, 80), (2064, 520, 48), (4096, 64, 1040)])
def test_norm_between_two_products(ops, m, n, k, inter):
    """The product that adds into the stream prepares the norm that reads it; the products behind it
    (plain, gated, with the rotation) take its rows and scale their sums."""
    pd, sd, wd = held(n, k, 1)
    pu, su, wu = held(2 * inter, n, 2)
    down, up = ops.mx4_from_codes(pd.cuda(), sd.cuda(), k), ops.mx4_from_codes(pu.cuda(), su.cuda(), n)
    x, res = normal((m, k), m, dtype=torch.bfloat16), normal((m, n), 5, 2.0)
    nw = (1 + 0.2 * normal((n,), 6)).cuda()
    stream = res.cuda()
    record = ops.linear(x.cuda(), down, None, torch.bfloat16, residual=stream, then_norm=(nw, 1e-5))
    plain_stream = res.cuda()
    assert ops.linear(x.cuda(), down, None, torch.bfloat16, residual=plain_stream) is None
    assert torch.equal(stream, plain_stream)
    # the rows: the stream times the weight, rounded once; the sums of squares of 16 columns
    assert torch.equal(record.raw, (stream * nw).to(torch.bfloat16))
    sq = (stream.double() ** 2).view(m, n // 16, 16).sum(-1)
    assert torch.allclose(record.ssq.double(), sq, rtol=2.0 ** -19, atol=0)          # 16 squares and their sum: 2^-24 each
    lazy = ops.normed(stream, nw, 1e-5, pre=record)
    s64 = stream.double().cpu().numpy()
    scale = 1 / np.sqrt((s64 ** 2).mean(1, keepdims=True) + 1e-5)
    raw = record.raw.double().cpu().numpy()
    y = ops.linear(lazy, up, None, torch.float32).double().cpu().numpy()
    # the sums' error, scaled; the scale itself: n / 16 + 4 additions of positive numbers and rsqrt (1 ulp)
    rel = (n / 16 + 12) * HALF_F32
    lim = (bound(raw, wu, n, torch.float32) + rel * (np.abs(raw) @ np.abs(wu).T)) * scale * (1 + rel) * 2
    assert (np.abs(y - (raw @ wu.T) * scale) <= lim).all()
    sw = ops.linear_swiglu(lazy, up, torch.bfloat16).double().cpu().numpy()
    g, u = ((raw @ wu.T) * scale)[:, :inter], ((raw @ wu.T) * scale)[:, inter:]
    dg, du = lim[:, :inter], lim[:, inter:]
    want = gate("silu", g, u)
    ls = 1.2 * dg * (np.abs(u) + du) + (np.abs(g) + dg) * du + 2.0 ** -16 * np.abs(g) * np.abs(u)
    assert (np.abs(sw - want) <= ls + HALF_BF16 * (np.abs(want) + ls) + 1e-38).all()
    # more rows than the norm is folded for, or another norm, go through the norm kernel
    other = ops.linear(ops.normed(stream, nw, 1e-6, pre=record), up, None, torch.float32)
    ref = ops.add_rmsnorm(stream.clone(), None, nw, 1e-6, torch.bfloat16)
    assert torch.equal(other, ops.linear(ref, up, None, torch.float32))


@pytest.mark.parametrize("rot_half", [True, False])
@pytest.mark.parametrize("write", [True, False])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("n_heads,n_kv,hd,k,seqs", [
    (4, 2, 16, 96, [(0, 0, 1)]),
    (6, 3, 48, 200, [(2, 5, 1), (0, 63, 1), (1, 64, 1)]),
    (8, 2, 64, 512, [(0, 60, 9), (3, 0, 1), (1, 100, 5)]),
    (32, 8, 64, 136, [(i, 7 * i, 1) for i in range(17)]),
    (4, 4, 128, 96, [(0, 3, 30)]),
    (6, 2, 32, 64, [(0, 0, 90)]),
])
def test_stacked_projection(ops, n_heads, n_kv, hd, k, seqs, bias, write, rot_half):
    """q rotated, k and v in the cache, against float64; from few rows in one kernel, from many by the
    product and the rotation kernel."""
    from helpers import make_ctx, make_kv, read_kv
    n = (n_heads + (2 * n_kv if write else 0)) * hd
    rot = hd if rot_half else hd // 2
    m = sum(c for _, _, c in seqs)
    packed, s, w = held(n, k, 3)
    q = ops.mx4_from_codes(packed.cuda(), s.cuda(), k)
    x = normal((m, k), 4, dtype=torch.bfloat16)
    b = normal((n,), 5) if bias else None
    ctx = make_ctx(ops, torch.bfloat16, seqs)
    slots = 1 + max(c for c, _, _ in seqs)
    kv = make_kv("cuda", torch.bfloat16, slots, 3, n_kv, hd, seed=2)
    cos, sin = torch.cos(normal((192, rot // 2), 8)), torch.sin(normal((192, rot // 2), 8))
    out = ops.qkv_rope(x.cuda(), q, None if b is None else b.cuda(), n_heads, n_kv, hd, cos.cuda(), sin.cuda(), rot, ctx,
                       kv, write, True, torch.bfloat16)
    xd = x.double().numpy()
    y = xd @ w.T + (0 if b is None else b.double().numpy())
    pos = ctx.tok_pos.cpu().numpy()
    heads = y.reshape(m, -1, hd).copy()
    c, sn = cos.double().numpy()[pos][:, None, :], sin.double().numpy()[pos][:, None, :]
    turned = heads[:, :n_heads + (n_kv if write else 0)]
    a0, a1 = turned[:, :, 0:rot:2].copy(), turned[:, :, 1:rot:2].copy()
    turned[:, :, 0:rot:2], turned[:, :, 1:rot:2] = a0 * c - a1 * sn, a1 * c + a0 * sn
    # a sum in 32 bits, a bias, two products and a sum more, each within 2^-24 of values up to |a0| + |a1|;
    # rounded to bfloat16 after the rotation, and from many rows also before it and before the bias,
    # where the value is the product p = y - b and not y
    base = (bound(xd, w, k, torch.float32) + HALF_F32 * np.abs(y)).reshape(m, -1, hd)
    pair = lambda t: np.repeat(t.reshape(m, -1, hd // 2, 2).sum(-1), 2, axis=-1)
    fused = ops._mx4_plan(m, n, n, k, False)[0] < 0
    if not fused:
        base = base + HALF_BF16 * (np.abs(xd @ w.T).reshape(m, -1, hd) + base)
    size = pair(np.abs(y).reshape(m, -1, hd))
    lim = pair(base) + 4 * HALF_F32 * size + HALF_BF16 * (size + pair(base)) + 1e-38
    got = out[:, :n_heads * hd].double().cpu().numpy().reshape(m, n_heads, hd)
    assert (np.abs(got - heads[:, :n_heads]) <= lim[:, :n_heads]).all()
    if write:
        row = 0
        for slot, pos0, count in seqs:
            keys, values = read_kv(kv, slot, pos0 + count)
            kd, vd = keys[pos0:].double().numpy(), values[pos0:].double().numpy()
            rows = slice(row, row + count)
            assert (np.abs(kd - heads[rows, n_heads:n_heads + n_kv]) <= lim[rows, n_heads:n_heads + n_kv]).all()
            assert (np.abs(vd - heads[rows, n_heads + n_kv:]) <= lim[rows, n_heads + n_kv:]).all()
            assert not keys[:pos0].any() and not values[:pos0].any()
            row += count
    else:
        assert not kv.plane("k").any() and not kv.plane("v").any()


# ------------------------------------------------------------------------------- whole models
LAYER_MATRICES = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    """Tiny models and, for the plain implementation, their weights with the layers' matrices rounded to
    MXFP4 by the quantiser above."""
    from plain import files, llama
    from tiny import TINY_A, TINY_B, TINY_C, make_model
    base, out = tmp_path_factory.mktemp("mx4"), {}
    for name, cfg in (("A", TINY_A), ("B", TINY_B), ("C", TINY_C)):
        path = make_model(base, cfg, seed=23 + len(name), name=name)
        cfg_json, weights = files.read_model_dir(path)
        rounded = {key: values(*quantise(t)) if key.split(".")[-2] in LAYER_MATRICES and t.ndim == 2 else t
                   for key, t in weights.items()}
        out[name] = (path, llama.PlainConfig(cfg_json), rounded)
    return out


@pytest.mark.parametrize("use_graphs", [True, False])
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_model_agrees_with_plain(models, tmp_path, name, use_graphs):
    """Whole prompts, tokens one by one, and batches of unequal requests, with the layers' matrices in
    MXFP4, against the plain implementation with the same numbers as weights."""
    import io

    import traces
    from helpers import assert_logits_close
    from libllm_amd.engine.trace import replay
    from libllm_amd.runtime import load_engine
    from plain import llama
    path, cfg, weights = models[name]
    rng = np.random.default_rng(4)
    lengths = [70, 33, 100, 5, 64, 1]
    requests = {"r%d" % i: rng.integers(0, cfg.vocab, size=min(n, cfg.max_pos)).tolist() for i, n in enumerate(lengths)}
    ids = list(requests)
    groups = [{r: requests[r] for r in ids[0:3]}, {r: requests[r] for r in ids[3:6]}]
    decode = {"r0": 20, "r1": 32, "r2": 3, "r3": 4, "r4": 1, "r5": 0}
    exact = {r: llama.logits_all(cfg, weights, t, store=llama.exact) for r, t in requests.items()}
    stored = {r: llama.logits_all(cfg, weights, t, store=llama.to_bfloat16) for r, t in requests.items()}
    for mode, steps in (("whole", traces.whole(requests)), ("tail", traces.tail_one_by_one(requests)),
                        ("batches", traces.batches(groups, decode))):
        engine = load_engine(path, dtype="bfloat16", max_tokens=traces.max_tokens_needed(steps), use_graphs=use_graphs,
                             weights="mxfp4")
        assert engine.model.blocks[0].feed_forward.down.weight is None
        replay(engine, traces.lines(steps), str(tmp_path / mode), log=io.StringIO())
        got = traces.collect(steps, str(tmp_path / mode), cfg.vocab)
        for r, toks in requests.items():
            out = np.stack([got[r][p] for p in range(len(toks))])
            assert_logits_close(out, exact[r], "bfloat16", "%s %s %s" % (name, mode, r), stored[r])


def test_generation_and_the_other_entry_points(models, tmp_path):
    """The same greedy tokens from the Python entry point, the C API's loader and random weights bound
    as MXFP4; refusals."""
    import json

    from libllm_amd import Model, capi
    from libllm_amd.errors import ConfigError
    path = models["B"][0]
    prompts = [[5, 8, 13, 21], [1, 2, 3, 4, 5, 6, 7, 8, 9], [42]]
    model = Model(path, max_tokens=1024, weights="mxfp4")
    want = model.generate(prompts, max_new_tokens=12, temperature=0.0, stop_tokens=())
    assert all(len(t) == 12 for t in want)
    other = capi.load(json.dumps({"filename": path, "max_tokens": 1024, "weights": "mxfp4"}))
    assert other.generate(prompts, max_new_tokens=12, temperature=0.0, stop_tokens=()) == want
    stored = Model(path, max_tokens=1024)
    assert stored.engine.model.blocks[0].feed_forward.down.weight is not None       # the format is not kept
    rnd = Model(path, max_tokens=256, random_weights=True, seed=3, weights="mxfp4")
    assert len(rnd.generate([[7, 9]], max_new_tokens=4, temperature=0.0, stop_tokens=())[0]) == 4
    with pytest.raises(ConfigError):
        Model(path, dtype="float32", weights="mxfp4")
    with pytest.raises(ConfigError):
        Model(path, weights="int4")


@pytest.mark.parametrize("program", ["python", "native"])
def test_command_lines(models, program):
    import os
    import subprocess
    import sys

    from libllm_amd import Model
    from libllm_amd.hip import build
    path = models["B"][0]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    command = {"python": [sys.executable, os.path.join(root, "bin", "llm")],
               "native": [os.path.join(os.path.dirname(build.build_capi(force=False, verbose=False)), build.CLI_NAME)]}[program]
    command += ["chat", "-m", path, "-ids", "-temperature", "0", "-max_new_tokens", "6"]
    run = lambda *flags: subprocess.run(command + list(flags), input="11 12 13 14\n", capture_output=True, text=True, timeout=120)
    got = run("-weights", "mxfp4")
    assert got.returncode == 0, got.stderr
    reply = [l for l in got.stdout.splitlines() if l.startswith("> ") and len(l) > 2][0][2:].split()
    model = Model(path, max_tokens=1024, weights="mxfp4")
    want = model.generate([[11, 12, 13, 14]], max_new_tokens=6, temperature=0.0)[0]
    assert [int(t) for t in reply] == [t for t in want if not model.is_stop(t)]
    assert run("-weights", "int4").returncode == 2
    got = run("-weights", "mxfp4", "-dtype", "float32")
    assert got.returncode != 0 and "bfloat16" in got.stderr


def test_time_per_operation(models):
    """Timed, the operations give what they give otherwise, the quantiser among them."""
    from libllm_amd import Model
    from libllm_amd.hip import HipOps
    path, prompts = models["B"][0], [[5, 6, 7, 8, 9], [11, 12]]
    plain = Model(path, max_tokens=512, weights="mxfp4").generate(prompts, max_new_tokens=6, temperature=0.0, stop_tokens=())
    ops = HipOps()
    ops.start_timing()
    timed = Model(path, max_tokens=512, weights="mxfp4", ops=ops)
    assert timed.generate(prompts, max_new_tokens=6, temperature=0.0, stop_tokens=()) == plain
    report = dict((name, (calls, ms)) for name, calls, ms in ops.timing_report())
    assert report["quantize_mx4"][0] >= 4 and all(ms > 0 for _, ms in report.values())


def test_from_two_threads(ops):
    """Two host threads with a stream each, products of many sizes at once: each as it is alone."""
    import threading
    w = ops.quantize_mx4(normal((96, 640), 1, 0.1).cuda())
    rows = [normal((m, 640), m, dtype=torch.bfloat16).cuda() for m in (1, 5, 16, 20, 40, 70, 130, 300)]
    work = lambda x: [ops.linear(x, w, None, torch.float32), ops.linear(ops.quantize_mx4(x), w, None, torch.bfloat16),
                      ops.linear_swiglu(x, w)]
    want = [work(x) for x in rows]
    torch.cuda.synchronize()
    got, failed = {}, []

    def run(name):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[name] = [work(x) for x in rows]
            stream.synchronize()
        except Exception as e:                              # (a thread's exception would be lost)
            failed.append(e)
    threads = [threading.Thread(target=run, args=(name,)) for name in "ab"]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for name in "ab":
        for a, b in zip(want, got[name]):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
