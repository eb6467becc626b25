"""Products with an MXFP4 weight at the ends of what its scales and the rows can hold."""
import numpy as np
import pytest
import torch

from test_gpu_mx4 import bound, file_form, normal, ops, quantise, values  # noqa: F401

pytestmark = pytest.mark.gpu

N, K = 64, 256


def by_plan(ops, monkeypatch, form):
    monkeypatch.setattr(ops, "_mx4_plan", lambda *sizes: (form, 1))
    monkeypatch.setattr(ops, "_mx4_plans", {})


def drawn(scales, seed):
    """A weight with codes drawn evenly and the scale bytes given, one for each block of a row."""
    codes = np.random.default_rng(seed).integers(0, 16, (N, K), dtype=np.uint8)
    return codes, np.broadcast_to(np.asarray(scales, dtype=np.uint8), (N, K // 32)).copy()


def product(ops, codes, scales, x, four):
    packed, s = file_form(codes, scales)
    w = ops.mx4_from_codes(packed.cuda(), s.cuda(), K)
    rows = ops.quantize_mx4(x.cuda()) if four else x.cuda()
    xd = x.double().numpy()
    return ops.linear(rows, w, None, torch.float32).double().cpu().numpy(), values(*quantise(xd)) if four else xd


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("form", [-1, 0, 1, 2, 3, 4])
@pytest.mark.parametrize("e", [0, 1, 2, 126, 251, 252])
@pytest.mark.parametrize("m", [1, 40])
def test_scales_at_both_ends(ops, monkeypatch, m, e, form, four):
    """Weights down to 2^-128 (no normal numbers in bfloat16) and up to 6 2^125, with rows that bring the
    sums near 1: nothing is flushed."""
    by_plan(ops, monkeypatch, form)
    codes, scales = drawn(e, e)
    x = (normal((m, K), 3).double() * 2.0 ** float(np.clip(127 - e, -120, 120))).to(torch.bfloat16)
    got, xd = product(ops, codes, scales, x, four)
    w = values(codes, scales)
    want = xd @ w.T
    assert np.abs(want).max() > 2.0 ** -10
    assert (np.abs(got - want) <= bound(xd, w, K, torch.float32)).all()


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("form", [-1, 0, 1, 2, 3, 4])
def test_rows_of_subnormal_numbers(ops, monkeypatch, form, four):
    by_plan(ops, monkeypatch, form)
    codes, scales = drawn(240, 5)
    x = (normal((40, K), 9).double() * 2.0 ** -129).to(torch.bfloat16)
    assert float(x.double().abs().max()) < 2.0 ** -126
    got, xd = product(ops, codes, scales, x, four)
    w = values(codes, scales)
    assert (np.abs(got - xd @ w.T) <= bound(xd, w, K, torch.float32)).all()


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("form", [-1, 0, 1, 2, 3, 4])
@pytest.mark.parametrize("e", [253, 254])
def test_numbers_that_32_bits_do_not_hold(ops, monkeypatch, e, form, four):
    """From 2^128 on, which scales of 2^126 and 2^127 reach: infinities to rows in bfloat16, as they are read
    back; what they are to rows in MXFP4.  Beside them, and with the codes of such blocks that stay below,
    ordinary sums."""
    by_plan(ops, monkeypatch, form)
    codes, scales = drawn(100, e)
    small = 5 if e == 253 else 3                        # the greatest magnitude below 2^128: 3 2^126, 1.5 2^127
    scales[:, 3] = e
    codes[:, 96:128] = np.where(codes[:, 96:128] & 7 > small, codes[:, 96:128] & 8 | small, codes[:, 96:128])
    codes[:5, 100] = 7                                  # +infinity: 6 2^126
    codes[3:8, 101] = 15                                # -infinity; rows 3 and 4 have both
    x = (normal((40, K), 4).double() * 2.0 ** -30).to(torch.bfloat16)
    x[7, 96:128] = 0.0
    got, xd = product(ops, codes, scales, x, four)
    w = values(codes, scales)
    if four:
        assert (np.abs(got - xd @ w.T) <= bound(xd, w, K, torch.float32)).all()
        return
    with np.errstate(invalid="ignore"):
        read = np.where(np.abs(w) >= 2.0 ** 128, np.sign(w) * np.inf, w)
        want = (xd[:, None, :] * read[None]).sum(-1)
        back = ops.dequantize_mx4(ops.mx4_from_codes(*(t.cuda() for t in file_form(codes, scales)), K), torch.float32)
        assert np.array_equal(back.double().cpu().numpy(), read)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want[7, :8]).all() and np.isnan(want[:, 3:5]).any()
        endless = np.isinf(want)
        assert endless.any() and np.array_equal(got[endless], want[endless])
        fine = np.isfinite(want)
        assert fine[:, 8:].all()
        assert (np.abs(got - want)[fine] <= bound(xd, np.where(np.isfinite(read), read, 0.0), K, torch.float32)[fine]).all()
