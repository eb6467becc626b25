"""Products with MXFP4 weights at sizes for which every kernel and every variant of it is chosen: each test
looks at what was launched, so that a change of the choice does not leave one untested.  The operands of most
are whole numbers and halves, whose sums 32 bits hold: those results have to be equal."""
import numpy as np
import pytest
import torch

import test_gpu_mx4 as mx4
from test_gpu_mx4 import normal, ops  # noqa: F401

pytestmark = pytest.mark.gpu

FEW, MANY, JOIN = "llm_gemm_mx4_rows", "llm_gemm_mx4_many", "llm_mx4_join"


@pytest.fixture
def launched(ops, monkeypatch):
    """What was launched, in order: (entry point, form and slices of K where it is the product for many rows)."""
    names, real = [], ops._launch

    def launch(name, *args):
        names.append((name, args[-2:] if name == MANY else None))
        real(name, *args)
    monkeypatch.setattr(ops, "_launch", launch)
    monkeypatch.setattr(ops, "_mx4_plans", {})
    return names


def forms(launched):
    return {how[0] for name, how in launched if name == MANY}


def whole(shape, seed, most=4):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(torch.bfloat16)


def held(ops, n, k, seed):
    """A weight of codes drawn evenly under scales of 1, and its numbers in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda").to(torch.uint8)
    even = torch.nn.functional.pad(codes, (0, k % 2))
    packed = (even[:, 0::2] | (even[:, 1::2] << 4)).contiguous()
    scales = torch.full((n, -(-k // 32)), 127, dtype=torch.uint8, device="cuda")
    grid = torch.tensor(mx4.GRID, device="cuda")
    return ops.mx4_from_codes(packed, scales, k), torch.cat([grid, -grid])[codes.int()]


def rows_for(ops, x, four):
    """Whole numbers up to 4 are MXFP4's own: both kinds of rows are the same numbers."""
    if not four:
        return x
    q = ops.quantize_mx4(x)
    assert torch.equal(ops.dequantize_mx4(q), x)
    return q


# sizes that the choice sends to every form of the product for many rows, by kind of rows
MANY_SIZES = [(0, False, 1000, 12304, 2056), (1, False, 200, 28688, 2056), (2, False, 130, 6160, 72),
              (2, False, 70, 12400, 200), (3, False, 130, 6160, 264), (3, False, 70, 2048, 5000),
              (4, False, 256, 1040, 72), (4, False, 200, 2080, 520), (0, True, 1000, 8208, 72),
              (1, True, 200, 16400, 72), (2, True, 130, 6160, 72), (3, True, 130, 6160, 1032),
              (3, True, 130, 6160, 1033), (4, True, 130, 2064, 72), (4, True, 64, 4096, 14336)]


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form,four,m,n,k", MANY_SIZES)
def test_many_rows(ops, launched, form, four, m, n, k, out):
    x, (w, wd) = whole((m, k), m + k), held(ops, n, k, n)
    bias = whole((n,), 3).float()
    want = x.double() @ wd.t()
    rows = rows_for(ops, x, four)
    del launched[:]
    assert torch.equal(ops.linear(rows, w, None, out), want.to(out))
    assert torch.equal(ops.linear(rows, w, bias, out), (want + bias.double()).to(out))
    assert forms(launched) == {form}


# the same for gated products, gate and up in whole tiles; and one whose up rows begin inside a tile
GATED_SIZES = [(0, False, 1000, 12320, 2056), (1, False, 200, 28704, 2056), (2, False, 130, 6176, 72),
               (2, False, 70, 12416, 200), (3, False, 130, 6176, 264), (3, False, 70, 2048, 5000),
               (4, False, 256, 1056, 72), (4, False, 200, 2080, 520), (0, True, 1000, 8224, 72),
               (1, True, 200, 16416, 72), (2, True, 130, 6176, 72), (3, True, 130, 6176, 1032),
               (4, True, 130, 2080, 72), (4, True, 64, 4096, 14336), (4, False, 256, 1042, 72)]


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("form,four,m,n,k", GATED_SIZES)
def test_many_rows_gated(ops, launched, form, four, m, n, k, act):
    x, (w, wd) = whole((m, k), m + k), held(ops, n, k, n)
    x = x * 2.0 ** -5                                            # gates of some tens: some of them small
    rows = rows_for(ops, x, four)
    y = (x.double() @ wd.t()).cpu().numpy()
    g, u = y[:, :n // 2], y[:, n // 2:]
    del launched[:]
    got = ops.linear_swiglu(rows, w, None, act).double().cpu().numpy()
    assert forms(launched) == {form}
    sliced = any(how[1] > 1 for name, how in launched if name == MANY)
    assert (JOIN in dict(launched)) == (sliced or n // 2 % 16 != 0)
    want = mx4.gate(act, np.maximum(g, -700.0), u)
    # the sums are exact; 2^-16 of |g| |u| for the device's exp and tanh and the cancellation in 1 + tanh
    lim = 2.0 ** -16 * np.abs(g * u)
    assert (np.abs(got - want) <= lim + 2.0 ** -8 * (np.abs(want) + lim)).all()


@pytest.mark.parametrize("form,four,m,n,k", [(3, False, 70, 2048, 5000), (4, True, 64, 4096, 14336), (3, False, 33, 8192, 4200)])
def test_slices_of_k_are_added_by_the_norm(ops, launched, form, four, m, n, k):
    """With ``residual`` the slices come back unadded, and the norm adds them to the stream in 32 bits."""
    x, (w, wd) = whole((m, k), m), held(ops, n, k, n)
    res, nw = whole((m, n), 5).float(), (1 + 0.25 * whole((n,), 6).float() / 4)
    rows = rows_for(ops, x, four)
    del launched[:]
    got = ops.linear(rows, w, None, torch.bfloat16, residual=res)
    assert forms(launched) == {form} and JOIN not in dict(launched)
    assert got.dim() == 3 and got.shape[0] > 1 and got.dtype == torch.float32
    want = res.double() + x.double() @ wd.t()
    normed = ops.add_rmsnorm(res, got, nw, 1e-5, torch.float32)
    assert torch.equal(res.double(), want)
    want = want / (want.square().mean(1, keepdim=True) + 1e-5).sqrt() * nw.double()
    # a sum of n squares in 32 bits (any order: at most n roundings of positive numbers), rsqrt, two products
    assert ((normed.double() - want).abs() <= (n / 2 + 8) * 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("bias,write,rot_half", [(True, True, True), (False, True, False), (True, False, True)])
@pytest.mark.parametrize("n_heads,n_kv,hd,k,seqs", [(28, 2, 64, 96, [(0, 3, 170), (2, 0, 130)]),
                                                    (56, 4, 64, 72, [(1, 0, 140)])])
def test_stacked_projection_of_many_rows(ops, launched, n_heads, n_kv, hd, k, seqs, bias, write, rot_half):
    mx4.test_stacked_projection(ops, n_heads, n_kv, hd, k, seqs, bias, write, rot_half)
    assert forms(launched) and FEW not in dict(launched)


@pytest.mark.parametrize("far", [1 << 22, (1 << 22) + 512, (1 << 22) + 8])
@pytest.mark.parametrize("m,form", [(70, None), (256, 0)])
def test_rows_that_lie_far_apart(ops, launched, monkeypatch, m, form, far):
    """As far as the offsets of a block of rows reach, and beyond, where they are copied."""
    n, k = (12400, 200) if form is None else (64, 384)
    if form is not None:
        monkeypatch.setattr(ops, "_mx4_plan", lambda *sizes: (form, 1))
    x = torch.empty((m, far), dtype=torch.bfloat16, device="cuda")[:, :k]
    x.copy_(whole((m, k), m))
    w, wd = held(ops, n, k, n)
    del launched[:]
    got = ops.linear(x, w, None, torch.float32)
    assert len(forms(launched)) == 1 and ("llm_pad_rows" in dict(launched)) == (far > 1 << 22 or k % 128 != 0)
    assert torch.equal(got.double(), x.double() @ wd.t())


@pytest.mark.parametrize("four,form", [(f, i) for f in (False, True) for i in range(5)])
@pytest.mark.parametrize("m,n,k,ks", [(2200, 2144, 72, 1), (2049, 2432, 584, 2), (600, 4640, 40, 1)])
def test_bands_of_blocks(ops, monkeypatch, m, n, k, ks, four, form):
    """More than eight blocks along the rows of X and along those of W, in no whole bands."""
    monkeypatch.setattr(ops, "_mx4_plan", lambda *sizes: (form, ks))
    monkeypatch.setattr(ops, "_mx4_plans", {})
    x, (w, wd) = whole((m, k), m + k), held(ops, n, k, n)
    rows = rows_for(ops, x, four)
    want = x.double() @ wd.t()
    assert torch.equal(ops.linear(rows, w, None, torch.float32).double(), want)
    assert torch.equal(ops.linear(rows, w, None, torch.bfloat16), want.to(torch.bfloat16))
    relu = (want[:, :n // 2].clamp(min=0) * want[:, n // 2:]).to(torch.bfloat16)
    # (the product of two sums is rounded to 32 bits before it is to 16)
    got = ops.linear_swiglu(rows, w, None, "relu")
    assert ((got.double() - relu.double()).abs() <= 2.0 ** -7 * relu.double().abs()).all()


# outputs of the product for few rows: tiles for half of 256 units at most, up to one a unit, up to three, and
# more, odd numbers of them, and a last one that is not whole
FEW_OUTPUTS = [1000, 2504, 4200, 12392]
FEW_ROWS = [1, 4, 6, 12, 16, 20, 32, 40]


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("k", [64, 300, 2100])
@pytest.mark.parametrize("n", FEW_OUTPUTS)
def test_few_rows(ops, launched, monkeypatch, n, k, four):
    monkeypatch.setattr(ops, "_mx4_plan", lambda *sizes: (-1, 1))
    w, wd = held(ops, n, k, n)
    bias = whole((n,), 3).float()
    for m in FEW_ROWS:
        x = whole((m, k), m)
        rows, want = rows_for(ops, x, four), x.double() @ wd.t()
        for out in (torch.float32, torch.bfloat16):
            assert torch.equal(ops.linear(rows, w, None, out), want.to(out)), (m, out)
        assert torch.equal(ops.linear(rows, w, bias, torch.float32).double(), want + bias.double()), m
    assert FEW in dict(launched) and not forms(launched)


@pytest.mark.parametrize("act", ["silu", "relu"])
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("k", [64, 300, 2100])
@pytest.mark.parametrize("inter", [1008, 2512, 4208, 12400])
def test_few_rows_gated(ops, launched, monkeypatch, inter, k, four, act):
    monkeypatch.setattr(ops, "_mx4_plan", lambda *sizes: (-1, 1))
    w, wd = held(ops, 2 * inter, k, inter)
    for m in FEW_ROWS:
        x = whole((m, k), m) * 2.0 ** -5
        y = x.double() @ wd.t()
        g, u = y[:, :inter], y[:, inter:]
        want = g.clamp(min=0) * u if act == "relu" else g * torch.sigmoid(g) * u
        got = ops.linear_swiglu(rows_for(ops, x, four), w, None, act).double()
        lim = 2.0 ** -16 * (g * u).abs()                         # as for many rows
        assert ((got - want).abs() <= lim + 2.0 ** -8 * (want.abs() + lim)).all(), m
    assert FEW in dict(launched) and not forms(launched) and JOIN not in dict(launched)


@pytest.mark.parametrize("n,k", [(2504, 1056), (4200, 1056), (12392, 520)])
def test_a_row_is_the_same_whatever_the_batch(ops, n, k):
    """The same bits, whichever variant of the product for few rows the sizes choose."""
    x = normal((32, k), 8, dtype=torch.bfloat16).cuda()
    q = ops.quantize_mx4(normal((n, k), 9, dtype=torch.bfloat16).cuda())
    both = ops.quantize_mx4(normal((2 * 2512, k), 9, dtype=torch.bfloat16).cuda())
    product, gated = ops.linear(x, q, None, torch.float32), ops.linear_swiglu(x, both)
    for m0, m in ((0, 1), (3, 4), (5, 7), (16, 16), (10, 9), (10, 22), (1, 31)):
        assert torch.equal(ops.linear(x[m0:m0 + m], q, None, torch.float32), product[m0:m0 + m])
        assert torch.equal(ops.linear_swiglu(x[m0:m0 + m], both), gated[m0:m0 + m])
    for m in (1, 16, 17, 31):                                    # (rows in MXFP4 begin at whole tiles)
        assert torch.equal(ops.linear(ops.quantize_mx4(x[:m]), q, None, torch.float32),
                           ops.linear(ops.quantize_mx4(x), q, None, torch.float32)[:m])


@pytest.mark.parametrize("m", [1, 6, 12, 16, 30])
@pytest.mark.parametrize("n,k", [(2512, 96), (4208, 200), (12400, 300)])
def test_few_rows_added_into_the_stream(ops, launched, m, n, k):
    x, (w, wd), res = whole((m, k), m), held(ops, n, k, n), whole((m, n), 5).float()
    want = res.double() + x.double() @ wd.t()
    del launched[:]
    assert ops.linear(x, w, None, torch.bfloat16, residual=res) is None
    assert FEW in dict(launched) and not forms(launched) and torch.equal(res.double(), want)


@pytest.mark.parametrize("m", [1, 6, 12, 16])
@pytest.mark.parametrize("n,k,inter", [(2512, 96, 528), (4208, 96, 528), (12400, 200, 528), (96, 64, 2512),
                                       (96, 64, 4208), (96, 64, 12400)])
def test_norm_between_two_wide_products(ops, m, n, k, inter):
    mx4.test_norm_between_two_products(ops, m, n, k, inter)


@pytest.mark.parametrize("bias,write,rot_half", [(True, True, True), (False, False, False)])
@pytest.mark.parametrize("n_heads,n_kv,hd", [(153, 2, 16), (259, 2, 16), (96, 2, 48), (771, 2, 16)])
@pytest.mark.parametrize("seqs", [[(0, 0, 1)], [(i, 7 * i, 1) for i in range(12)], [(1, 60, 9), (0, 5, 15)]])
def test_wide_stacked_projection_of_few_rows(ops, launched, n_heads, n_kv, hd, seqs, bias, write, rot_half):
    mx4.test_stacked_projection(ops, n_heads, n_kv, hd, 96, seqs, bias, write, rot_half)
    assert "llm_gemm_mx4_rows_rope" in dict(launched) and not forms(launched)


def run_of(ops, weights, nw, h, res):
    """A run of a layer's products: into the stream in slices of K, its norm, gate and up, and down."""
    down, gate_up = weights
    delta = ops.linear(h, down, None, torch.bfloat16, residual=res)
    rows = ops.add_rmsnorm(res, delta, nw, 1e-5, torch.bfloat16)
    act = ops.linear_swiglu(rows, gate_up)
    return res, act, ops.linear(act, down, None, torch.float32), ops.linear(ops.quantize_mx4(act), down, None, torch.bfloat16)


def layer(ops):
    down = ops.quantize_mx4(normal((2048, 5008), 1, 0.02).cuda())
    gate_up = ops.quantize_mx4(normal((2 * 5008, 2048), 2, 0.02).cuda())
    return (down, gate_up), (1 + 0.1 * normal((2048,), 3)).cuda()


def test_many_rows_replayed_from_a_graph(ops, launched):
    m, held_out = 70, {}
    weights, nw = layer(ops)
    h, res = torch.empty((m, 5008), dtype=torch.bfloat16, device="cuda"), torch.empty((m, 2048), device="cuda")
    stream = torch.empty_like(res)

    def step():
        stream.copy_(res)
        held_out["out"] = run_of(ops, weights, nw, h, stream)
    h.normal_(), res.normal_()
    del launched[:]
    graph = ops.capture(step)
    assert any(how[1] > 1 for name, how in launched if name == MANY) and JOIN in dict(launched)
    replayed = held_out["out"]
    for i in range(4):
        h.copy_(normal((m, 5008), 50 + i)), res.copy_(normal((m, 2048), 60 + i))
        graph.replay()
        got = [t.clone() for t in replayed]
        step()
        assert all(torch.equal(a, b) for a, b in zip(got, held_out["out"]))
        torch.cuda.synchronize()


def test_many_rows_from_two_threads(ops, launched):
    """Two host threads with a stream each: every result as it is alone."""
    import threading
    weights, nw = layer(ops)
    sizes = (70, 130, 300, 520)
    inputs = [(normal((m, 5008), m, dtype=torch.bfloat16).cuda(), normal((m, 2048), m + 1).cuda()) for m in sizes]
    work = lambda: [run_of(ops, weights, nw, h, res.clone()) for h, res in inputs]
    want = work()
    torch.cuda.synchronize()
    assert len(forms(launched)) > 1 and JOIN in dict(launched)
    got, failed = {}, []

    def run(name):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got[name] = work()
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", [(131090, 16400), (131089, 16403)])
def test_conversions_of_more_elements_than_32_bits_count(ops, rows, width, dtype):
    """Offsets of elements, of codes and of what is read back pass 2^31; the last rows are what they are alone."""
    assert rows * width > 1 << 31
    x = torch.empty((rows, width), dtype=dtype, device="cuda")
    x.copy_(whole((rows, 1), 1).to(dtype) * torch.arange(1, width + 1, device="cuda").remainder(7).to(dtype) * 0.25)
    q = ops.quantize_mx4(x)
    back = ops.dequantize_mx4(q, dtype)
    at = rows // 16 * 16
    for first, last in ((0, 48), (at - 48, rows)):
        part = ops.quantize_mx4(x[first:last].contiguous())
        assert torch.equal(ops.dequantize_mx4(part, dtype), back[first:last])
    codes, scales = ops.quantize_mx4(x[at - 16:at].contiguous()), q.leading_rows(at)
    assert torch.equal(scales.codes[-codes.codes.numel():], codes.codes)
    assert torch.equal(scales.scales[-codes.scales.numel():], codes.scales)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(33000, 65600), (33001, 65603)])
def test_results_of_more_elements_than_32_bits_count(ops, launched, m, n, out, four):
    assert m * n > 1 << 31
    k = 64
    x, (w, wd) = whole((m, k), 1), held(ops, n, k, 2)
    rows = rows_for(ops, x, four)
    got = ops.linear(rows, w, None, out)
    assert forms(launched)
    for first in list(range(0, m - 500, 4096)) + [m - 500]:
        want = (x[first:first + 500].double() @ wd.t()).to(out)
        assert torch.equal(got[first:first + 500], want), first
