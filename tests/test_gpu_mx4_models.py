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
