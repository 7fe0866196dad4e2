"""Models whose weights become 8-bit integers: what needs no GPU."""
from types import SimpleNamespace

import pytest
import torch

from tinyllama_c_b200 import ops
from tinyllama_c_b200.engine.decode_graph import DecodeGraph
from tinyllama_c_b200.parts.feed_forward import MoEFeedForward
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


def test_experts_are_converted_as_a_whole_or_not_at_all(monkeypatch):
    """The second of an expert's two tables may find no memory; the layer then still runs as it was, and can be asked again."""
    moe = MoEFeedForward(64, 3, 2, 40, "router", dict(gate="e{e}.g", up="e{e}.u", down="e{e}.d"))
    moe.bind({s.name: torch.ones(s.shape, dtype=torch.bfloat16) for s in moe.weight_specs()}, torch.bfloat16, "cpu")
    calls = []

    def weight_int8(w):
        calls.append(w)
        if len(calls) == 2:
            raise torch.OutOfMemoryError("no room")
        return w.to(torch.int8), w.float()[..., 0]

    monkeypatch.setattr(ops, "weight_int8", weight_int8)
    with pytest.raises(torch.OutOfMemoryError):
        moe.to_int8()
    assert moe.w_gate_up.dtype == moe.w_down.dtype == torch.bfloat16 and moe.gate_up_scale is None and moe.down_scale is None
    assert moe.to_int8() == 2 and moe.w_gate_up.dtype == moe.w_down.dtype == torch.int8
