"""Models whose layers are in MXFP4, beside those of test_gpu_mx4.py."""
import os

import numpy as np
import pytest
import torch

from test_gpu_mx4 import quantise, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stored", ["float32", "float16"])
def test_a_file_of_more_bits_is_rounded_once(tmp_path, stored):
    """The codes that a model holds are those of the file's numbers, not of their rounding to bfloat16."""
    from libllm_amd.runtime import load_engine
    from plain import files
    from tiny import TINY_B, make_model
    path = make_model(tmp_path, TINY_B, seed=17, stored=stored)
    held = files.read_safetensors(os.path.join(path, "model.safetensors"))
    engine = load_engine(path, max_tokens=256, weights="mxfp4")
    twice = 0
    for i, block in enumerate(engine.model.blocks):
        at = "model.layers.%d." % i
        for linear, names in ((block.mixer.out, ["self_attn.o_proj"]), (block.feed_forward.down, ["mlp.down_proj"]),
                              (block.feed_forward.gate_up, ["mlp.gate_proj", "mlp.up_proj"])):
            w = np.concatenate([held[at + n + ".weight"] for n in names]).astype(np.float64)
            codes, scales = quantise(w)
            got_codes, got_scales = rows_of(linear.prepared)
            n, k = w.shape
            assert np.array_equal(got_codes[:n, :k], codes) and np.array_equal(got_scales[:n, :scales.shape[1]], scales)
            coarse = quantise(torch.from_numpy(w).to(torch.bfloat16).double().numpy())
            twice += int((coarse[0] != codes).sum())
    assert twice > 0                                            # the numbers tell the two apart


def test_two_layers_of_the_1b_shape(monkeypatch):
    """Layers of the measured shape with its whole vocabulary: prompts of 247 rows, of 100 more in short ones, and
    decode steps of all 37 sequences, against the plain implementation on the rounded weights; the products for
    few rows and for many, whole and in slices of K, all take part."""
    import bench
    from helpers import assert_logits_close
    from libllm_amd.config import config_from_dict
    from libllm_amd.engine import StepEntry
    from libllm_amd.hip import HipOps
    from libllm_amd.runtime import random_engine
    from libllm_amd.weights import random_tensors
    from plain import llama
    from test_gpu_mx4 import LAYER_MATRICES, values
    launched, real = set(), HipOps._launch

    def launch(ops, name, *args):
        launched.add((name, args[-1] > 1 if name == "llm_gemm_mx4_many" else None))
        real(ops, name, *args)
    monkeypatch.setattr(HipOps, "_launch", launch)
    config = config_from_dict(dict(bench.FULL, num_hidden_layers=2, max_position_embeddings=4096))
    cfg = llama.PlainConfig(config.to_dict())
    engine = random_engine(config, seed=3, max_tokens=37 * 64 + 1024, weights="mxfp4")
    declared = engine.model.declared()
    # the random-weights mode draws every tensor from (seed, name): the same draw here, rounded by the quantiser
    weights = {name: random_tensors({name: declared[name]}, 3, std=0.02, dtype=torch.bfloat16,
                                    device="cuda")[name].double().cpu().numpy() for name in declared}
    weights = {name: values(*quantise(w)) if name.split(".")[-2] in LAYER_MATRICES else w for name, w in weights.items()}
    rng = np.random.default_rng(78)
    lengths, more = [200, 40, 7] + [2 + i % 3 for i in range(34)], 3
    toks = [rng.integers(0, cfg.vocab, size=n + more).tolist() for n in lengths]
    got = [[] for _ in toks]
    for part in (range(3), range(3, 37)):
        out = engine.step([StepEntry(i, toks[i][:-more], [lengths[i] - 1]) for i in part])
        for j, i in enumerate(part):
            got[i].append(out[j].double().cpu().numpy())
    for k in range(more):
        out = engine.step([StepEntry(i, [t[lengths[i] + k]], [0]) for i, t in enumerate(toks)])
        for i in range(37):
            got[i].append(out[i].double().cpu().numpy())
    assert {("llm_gemm_mx4_rows", None), ("llm_gemm_mx4_many", False), ("llm_gemm_mx4_many", True)} <= launched
    for i, t in enumerate(toks):
        rows = list(range(lengths[i] - 1, len(t)))
        exact, rounded = (llama.lm_head(cfg, weights, llama.hidden_states(cfg, weights, t, **kw)[rows])
                          for kw in ({}, {"store": llama.to_bfloat16}))
        assert_logits_close(np.stack(got[i]), exact, "bfloat16", "request %d" % i, rounded)
