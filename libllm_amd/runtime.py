"""From a model folder to an engine: configuration, model as data, weights, cache, step function."""
from typing import Optional

import torch

from .config import config_from_dir
from .engine.model import DecoderModel
from .engine.step import Engine
from .errors import ConfigError
from .weights import load_tensors, random_tensors
from .weights.loader import Tensors, place

_DTYPES = {"bfloat16": torch.bfloat16, "bf16": torch.bfloat16,
           "float32": torch.float32, "fp32": torch.float32}


def parse_dtype(name) -> torch.dtype:
    if isinstance(name, torch.dtype):
        if name not in (torch.bfloat16, torch.float32):
            raise ConfigError("dtype must be bfloat16 or float32")
        return name
    if name not in _DTYPES:
        raise ConfigError("dtype must be bfloat16 or float32, got %r" % (name,))
    return _DTYPES[name]


def default_ops():
    """The kernels of the product path.  Raises KernelError without a GPU or the built library."""
    from .hip import HipOps
    return HipOps()


WEIGHT_FORMATS = ("stored", "mxfp4")


def _check_format(weights, ops, dtype):
    if weights not in WEIGHT_FORMATS:
        raise ConfigError("weights are %s, not %r" % (" or ".join(WEIGHT_FORMATS), weights))
    if weights == "mxfp4":
        if dtype != torch.bfloat16:
            raise ConfigError("weights in MXFP4 need bfloat16 activations")
        if not hasattr(ops, "quantize_mx4"):
            raise ConfigError("these operations know no weights in MXFP4")


class _Binding:
    """The operations as a model's parts see them while they are bound: with the format of this
    model's weights, which another model that is bound over them at the same time does not share."""

    def __init__(self, ops, weights):
        self._ops, self.weight_format = ops, weights

    def __getattr__(self, name):
        return getattr(self._ops, name)


def _bind(model, tensors, ops, dtype, weights):
    """Binds the tensors, the layers' matrices in the format asked for."""
    model.bind(tensors, ops if weights == "stored" else _Binding(ops, weights), dtype)


def load_engine(model_dir: str, dtype="bfloat16", max_tokens: int = 8192, ops=None,
                max_slots: Optional[int] = None, use_graphs: bool = True,
                keep_float32: bool = False, tiled_weights: bool = True, weights: str = "stored") -> Engine:
    """Reads config.json, chooses the architecture by its ``model_type``, loads the tensors by
    name and returns an engine whose cache holds ``max_tokens`` tokens.  ``keep_float32``: in
    bfloat16 mode a matrix that the file stores in 32-bit stays float32 (true 32-bit products
    for it) instead of becoming bfloat16.  ``tiled_weights=False``: no second, tiled copy of the
    bfloat16 matrices (half the weight memory; decoding is 5 to 11 % slower).  ``weights="mxfp4"``:
    the matrices of attention and feed-forwards are rounded to MXFP4 when they are bound, from what the
    file stores (4.25 bits an element, held once; the embedding and the output matrix are as without)."""
    config = config_from_dir(model_dir)
    tdtype = parse_dtype(dtype)
    spec = config.to_spec()
    model = DecoderModel(spec)
    ops = ops if ops is not None else default_ops()
    _check_format(weights, ops, tdtype)
    if not tiled_weights:
        ops.pack_weights = False
    tensors = load_tensors(model_dir, model.declared(), spec.optional_tensors, tdtype, ops.device,
                           keep_float32, weights)
    _bind(model, tensors, ops, tdtype, weights)
    engine = Engine(model, ops, tdtype, max_tokens, max_slots=max_slots, use_graphs=use_graphs)
    engine.config = config
    return engine


def random_engine(config, seed: int = 0, dtype="bfloat16", max_tokens: int = 8192, ops=None,
                  max_slots: Optional[int] = None, use_graphs: bool = True, std: float = 0.02,
                  stored: torch.dtype = torch.bfloat16, tiled_weights: bool = True,
                  weights: str = "stored") -> Engine:
    """The random-weights mode without a file: every tensor the model declares is drawn on the
    device from ``seed`` (matrices normal with ``std``, norm scales 1) and bound as a loaded file
    would be that stores ``stored`` (float32: full significands for the 32-bit path).  ``config``
    is a typed configuration; ``weights`` as for ``load_engine``."""
    tdtype = parse_dtype(dtype)
    spec = config.to_spec()
    model = DecoderModel(spec)
    ops = ops if ops is not None else default_ops()
    _check_format(weights, ops, tdtype)
    if not tiled_weights:
        ops.pack_weights = False
    declared = model.declared()
    tensors = Tensors()
    for name in sorted(declared):
        def draw(name=name, decl=declared[name]):
            t = random_tensors({name: decl}, seed, std=std, dtype=stored, device=ops.device)[name]
            return place(t, decl, tdtype, ops.device, weights=weights)
        tensors[name] = draw if weights != "stored" and declared[name].low_bit else draw()
    _bind(model, tensors, ops, tdtype, weights)
    engine = Engine(model, ops, tdtype, max_tokens, max_slots=max_slots, use_graphs=use_graphs)
    engine.config = config
    return engine
