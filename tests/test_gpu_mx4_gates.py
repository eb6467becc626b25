"""The gate of the gated products with MXFP4 weights: what it makes of numbers that are none, and of gates far
below zero, alike in every kernel that applies it."""
import numpy as np
import pytest
import torch

from test_gpu_mx4 import gate, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def by_one_kernel(ops, monkeypatch, kernel):
    """The product for few rows, the one for many in two forms, or slices of K and the kernel that adds them."""
    plan = {"few": (-1, 1), "many": (0, 1), "many, small": (4, 1), "joined": (3, 2)}[kernel]
    monkeypatch.setattr(ops, "_mx4_plan", lambda *sizes: plan)
    monkeypatch.setattr(ops, "_mx4_plans", {})


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("kernel", ["few", "many", "many, small", "joined"])
def test_a_gate_or_an_up_that_is_no_number(ops, monkeypatch, kernel, act, out):
    """Whichever of the two is NaN, the result is, below zero too, where ReLU makes nothing of a number."""
    by_one_kernel(ops, monkeypatch, kernel)
    inter, k = 32, 1024
    w = torch.zeros((2 * inter, k))
    w[:inter, 0], w[inter:, 1] = -1.0, 2.0
    w[5, 600], w[inter + 7, 40] = float("nan"), float("nan")
    x = torch.zeros((3, k), dtype=torch.bfloat16)
    x[:, 0], x[:, 1] = torch.tensor([0.5, 1.0, 3.0]), 1.5
    got = ops.linear_swiglu(x.cuda(), ops.quantize_mx4(w.cuda()), out, act).double().cpu().numpy()
    want = np.repeat(gate(act, -x[:, :1].double().numpy(), 3.0), inter, axis=1)
    none = np.zeros(inter, dtype=bool)
    none[[5, 7]] = True
    assert np.isnan(got[:, none]).all()
    # the result's rounding, and 2^-16 of |g| |u| for the device's exp and tanh and the cancellation in 1 + tanh
    assert (np.abs(got[:, ~none] - want[:, ~none]) <= 2.0 ** -8 * np.abs(want[:, ~none]) + 2.0 ** -16 * 9).all()


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("dtype,m,inter", [(torch.bfloat16, 3, 32), (torch.bfloat16, 100, 64), (torch.bfloat16, 300, 256),
                                           (torch.float32, 3, 32)])
def test_the_same_of_weights_that_are_stored(ops, dtype, m, inter, act):
    k = 256
    w = torch.zeros((2 * inter, k))
    w[:inter, 0], w[inter:, 1] = -1.0, 2.0
    w[5, 200], w[inter + 7, 40] = float("nan"), float("nan")
    x = torch.zeros((m, k))
    x[:, 0], x[:, 1] = 1.0, 1.5
    got = ops.linear_swiglu(x.to(dtype).cuda(), w.to(dtype).cuda(), dtype, act).cpu()
    assert torch.isnan(got[:, [5, 7]]).all() and int(torch.isnan(got).sum()) == 2 * m


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kernel", ["few", "many", "many, small", "joined"])
def test_silu_of_gates_far_from_zero(ops, monkeypatch, kernel, out):
    """Gates of -170 to 170 with ups of any size: the result is right wherever 32 bits hold it, though e^-g
    overflows below -88 and its reciprocal is no normal number from -87 on."""
    by_one_kernel(ops, monkeypatch, kernel)
    inter, k = 48, 1024
    w = torch.zeros((2 * inter, k))
    w[:inter, 0] = 1.0
    ups = [2.0 ** 100, 1.0, -2.0 ** -20]
    for i in range(inter):
        w[inter + i, 32 * (1 + i % 3)] = 1.0                    # (a block of its own each)
    x = torch.zeros((341, k), dtype=torch.bfloat16)
    x[:, 0] = torch.linspace(-170, 170, 341)
    for i, up in enumerate(ups):
        x[:, 32 * (1 + i)] = up
    got = ops.linear_swiglu(x.cuda(), ops.quantize_mx4(w.cuda()), out).double().cpu().numpy()
    g = x[:, :1].double().numpy()
    want = g / (1 + np.exp(-g)) * np.array([ups[i % 3] for i in range(inter)])
    # e^(-|g| / 2), twice: its argument, up to 0.73 |g|, is rounded twice where the instruction takes powers of
    # two, |g| 2^-24 each time it is used; the rest are a dozen roundings of 2^-24 (an instruction's last bit is
    # two of them).  Then the result's own; below 2^-126 it may be taken for zero.
    half = 2.0 ** -8 if out == torch.bfloat16 else 2.0 ** -24
    lim = (half + (2 * np.abs(g) + 16) * 2.0 ** -24) * np.abs(want) + 2.0 ** -126
    assert (np.abs(got - want) <= lim).all(), np.abs(got - want).max()
