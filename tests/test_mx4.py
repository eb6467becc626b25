"""MXFP4 matrices on the host: sizes, checks and launch plans.  (What runs on the device:
test_gpu_mx4.py.)"""
import random

import pytest
import torch

from libllm_amd.errors import ConfigError, KernelError
from libllm_amd.hip.mx4 import Mx4Matrix, Mx4Ops, tiled_sizes


def test_tiled_sizes():
    assert tiled_sizes(1, 1) == (4096, 256)
    assert tiled_sizes(16, 512) == (4096, 256)
    assert tiled_sizes(17, 513) == (4 * 4096, 4 * 256)
    assert tiled_sizes(28672, 4096) == (28672 * 4096 // 2, 28672 * 4096 // 32)


def test_matrix_checks_its_storage():
    codes, scales = torch.zeros(8192, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    q = Mx4Matrix((20, 100), codes, scales)
    assert q.shape == (20, 100) and q.codes is codes and q.scales is scales
    top = q.leading_rows(16)
    assert top.shape == (16, 100) and top.codes.shape == (4096,) and top.codes.data_ptr() == codes.data_ptr()
    for rows in (0, 8, 17, 32):
        with pytest.raises(KernelError):
            q.leading_rows(rows)
    for bad in (((20, 513), codes, scales), ((33, 100), codes, scales), ((20, 100), codes.int(), scales),
                ((20, 100), codes, scales[:256]), ((20, 100), codes.view(2, 4096), scales),
                ((20, 100), torch.zeros(8193, dtype=torch.uint8)[1:], scales)):
        with pytest.raises(KernelError):
            Mx4Matrix(*bad)
    room = Mx4Matrix._new(20, 100, codes.device, codes[:0])
    assert room.codes.shape == (8192,) and room.scales.shape == (512,)
    assert room.codes_ptr == room.codes.data_ptr() and room.scales_ptr == room.scales.data_ptr()


class Host(Mx4Ops):
    def __init__(self, units=256):
        self.units, self._mx4_plans = units, {}


def test_plans_are_launches_the_kernels_take():
    """Every slice of K has quads of its own, a form exists, and the number of plans kept is bounded."""
    ops, rng = Host(), random.Random(1)
    ops.MX4_PLANS = 50
    for _ in range(3000):
        m, n, k = (int(2 ** rng.uniform(0, top)) for top in (14, 17, 16))
        four = rng.random() < 0.5
        gated = n % 2 == 0 and rng.random() < 0.5
        form, ks = ops._mx4_plan(m, n, n // 2 if gated else n, k, four)
        assert len(ops._mx4_plans) <= 50
        assert (form, ks) == ops._mx4_plan(m, n, n // 2 if gated else n, k, four)
        if form < 0:
            assert ks == 1 and (m <= 2 * ops.MX4_ROWS or -(-m // 32) * -(-n // 16) <= 3 * ops.units)
            continue
        assert form in (0, 1, 2, 3, 4)
        quads = -(-k // 512)
        per = -(-quads // ks)
        assert -(-quads // per) == ks                    # no slice is empty


def test_engine_refuses_formats_it_cannot_hold(tmp_path):
    from libllm_amd.config import config_from_dict
    from libllm_amd.runtime import random_engine
    from tiny import TINY_A

    class Ops:
        device = torch.device("cpu")
        supports_graphs = False
    cfg = config_from_dict(TINY_A)
    for kw in ({"weights": "fp4"}, {"weights": "mxfp4", "dtype": "float32"}, {"weights": "mxfp4"}):
        with pytest.raises(ConfigError):
            random_engine(cfg, ops=Ops(), max_tokens=64, **kw)


def test_a_matrix_is_bound_once_whatever_its_order():
    """Rows in a row for the quantiser, a transposed matrix too; the leading rows in the same storage where
    they are whole tiles."""
    from libllm_amd.parts.linear import Linear

    class Quantised:
        def __init__(self, w):
            assert w.stride(-1) == 1
            self.w = w

        def leading_rows(self, rows):
            return ("leading", rows)

    class Ops:
        weight_format = "mxfp4"
        quantize_mx4 = staticmethod(Quantised)
    w = torch.arange(12 * 40).reshape(12, 40).float()
    whole = Linear(12, 40, low_bit=True)
    whole.bind(w.t(), ops=Ops())
    assert whole.weight is None and torch.equal(whole.prepared.w, w.t())
    part = Linear(12, 32, low_bit=True)
    part.bind(w.t()[:32], ops=Ops(), like=whole.prepared)
    assert part.prepared == ("leading", 32)
    part = Linear(12, 24, low_bit=True)
    part.bind(w.t()[:24], ops=Ops(), like=whole.prepared)
    assert torch.equal(part.prepared.w, w.t()[:24])


@pytest.mark.parametrize("stored", ["float32", "float16", "bfloat16", "float64"])
def test_matrices_come_to_the_quantiser_as_the_file_stores_them(tmp_path, stored):
    """Rounded to bfloat16 first they would be rounded twice; what is held in the model's type is so as ever."""
    import os

    from libllm_amd.config import config_from_dict
    from libllm_amd.engine import DecoderModel
    from libllm_amd.runtime import _bind, load_tensors
    from plain import files
    from tiny import TINY_A, make_model

    class Held:
        def leading_rows(self, rows):
            return self

    class Ops:
        device = torch.device("cpu")

        def __init__(self):
            self.given = []

        def quantize_mx4(self, w):
            self.given.append(w)
            return Held()
    path = make_model(tmp_path, TINY_A, seed=3, stored=stored)
    held = files.read_safetensors(os.path.join(path, "model.safetensors"))
    model, ops = DecoderModel(config_from_dict(TINY_A).to_spec()), Ops()
    tensors = load_tensors(path, model.declared(), model.spec.optional_tensors, torch.bfloat16, ops.device,
                           weights="mxfp4")
    _bind(model, tensors, ops, torch.bfloat16, "mxfp4")
    for i in range(len(model.blocks)):
        at = "model.layers.%d." % i
        for names in (("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"), ("self_attn.o_proj",),
                      ("mlp.gate_proj", "mlp.up_proj"), ("mlp.down_proj",)):
            w = torch.cat([torch.from_numpy(held[at + n + ".weight"]).double() for n in names])
            if stored == "float64":
                w = w.float().double()
            match = [g for g in ops.given if g.shape == w.shape and torch.equal(g.double(), w)]
            assert len(match) == 1 and match[0].dtype == (torch.bfloat16 if stored == "bfloat16" else torch.float32)
    assert len(ops.given) == 4 * len(model.blocks)
    assert tensors["model.embed_tokens.weight"].dtype == torch.bfloat16
    assert tensors["model.norm.weight"].dtype == torch.float32


def test_two_models_bound_at_once_over_the_same_operations(tmp_path):
    """Each in its own format, whatever the other asks for between the two's matrices."""
    import threading

    from libllm_amd.config import config_from_dict
    from libllm_amd.engine import DecoderModel
    from libllm_amd.runtime import _bind, load_tensors
    from tiny import TINY_A, make_model

    class Held:
        def leading_rows(self, rows):
            return self

    class Ops:
        device = torch.device("cpu")
        turns = threading.Barrier(2, timeout=60)

        def wait(self):                     # the two threads take every matrix of a layer in step
            try:
                self.turns.wait()
            except threading.BrokenBarrierError:
                pass

        def quantize_mx4(self, w):
            self.wait()
            return Held()

        def prepare_weight(self, w, like=None):
            if like is None and w.shape[0] != 256:
                self.wait()
            return w
    path, ops, models = make_model(tmp_path, TINY_A, seed=3), Ops(), {}

    def load(weights):
        try:
            model = DecoderModel(config_from_dict(TINY_A).to_spec())
            _bind(model, load_tensors(path, model.declared(), model.spec.optional_tensors, torch.bfloat16, ops.device,
                                      weights=weights), ops, torch.bfloat16, weights)
            models[weights] = model
        finally:
            ops.turns.abort()
    threads = [threading.Thread(target=load, args=(w,)) for w in ("mxfp4", "stored")]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for weights in ("mxfp4", "stored"):
        for block in models[weights].blocks:
            for linear in (block.mixer.qkv, block.mixer.out, block.feed_forward.gate_up, block.feed_forward.down):
                assert isinstance(linear.prepared, Held) == (weights == "mxfp4")
    assert not hasattr(ops, "weight_format")


@pytest.mark.parametrize("mode", [["--workload", "batch64"], ["--sweep"], ["--unequal"], ["--requests", "8"]])
def test_bench_measures_mxfp4_in_the_default_run_only(mode):
    """The other runs build engines with stored weights: they do not pass for what was asked."""
    import os
    import subprocess
    import sys
    bench = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bench.py")
    got = subprocess.run([sys.executable, bench, "--weights", "mxfp4"] + mode, capture_output=True, text=True, timeout=100)
    assert got.returncode == 2 and "--weights mxfp4" in got.stderr and not got.stdout
