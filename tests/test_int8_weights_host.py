"""Models whose weights become 8-bit integers: what needs no GPU."""
from types import SimpleNamespace

import pytest
import torch

from tinyllama_c_b200.engine.decode_graph import DecodeGraph
from tinyllama_c_b200.weights import load_model

import configs
from helpers import make_model_dir


def test_a_captured_step_is_stale_once_the_model_has_other_weights(tmp_path):
    """The graph holds addresses of weights: bind() and to_int8() replace them."""
    folder = make_model_dir(tmp_path, configs.TINY_A, seed=3)
    model = load_model(folder, "bfloat16", "cpu")
    captured = SimpleNamespace(model=model, graph=None, weights_version=-1)
    stale = lambda: DecodeGraph.stale.fget(captured)  # noqa: E731
    assert stale()
    captured.graph, captured.weights_version = object(), model.weights_version
    assert not stale()
    for layer in model.layers:                            # (the kernels that round weights need a GPU)
        layer.to_int8 = lambda: 1
    model.to_int8()
    assert stale()
    captured.weights_version = model.weights_version
    assert not stale()
    tensors = {s.name: torch.zeros(s.shape) for s in model.weight_specs()}
    model.bind(tensors, torch.float32, "cpu")
    assert stale()


def test_a_model_stored_in_32_bits_is_refused(tmp_path):
    """Its matrices keep their 32 bits: asked for 8, it would run unchanged."""
    folder = make_model_dir(tmp_path, configs.TINY_A, seed=3, dtype="float32")
    with pytest.raises(ValueError, match="32 bits"):
        load_model(folder, "bfloat16", "cpu", weights="int8")
    model = load_model(folder, "bfloat16", "cpu")
    with pytest.raises(ValueError, match="32 bits"):
        model.to_int8()
