"""Models whose layers multiply in 8-bit integers.

Parts are compared with the formula in 64 bits on the integers that the part itself holds (allowances as in test_gpu_int8.py).  Whole
models are compared with the same model in bfloat16: rounding a row or a channel of some hundred values with a largest magnitude of
3 to 4.5 times the root mean square moves a product by 1 to 1.5 % of its size, a dozen products on the way to a logit by 5 %, norms and
gates a few times that: 25 % of the logits' size is allowed, where a lost scale, bias or interleaving gives 100 %."""
import copy

import pytest
import torch

import tinyllama_c_b200 as tlc
from tinyllama_c_b200 import ops
from tinyllama_c_b200.engine import StepEntry
from tinyllama_c_b200.parts.feed_forward import MoEFeedForward, SwiGLU
from tinyllama_c_b200.parts.linear import StackedLinear

import configs
import __graft_entry__ as entry
from helpers import make_model_dir, random_tokens

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
MODELS = {"A": configs.TINY_A, "B": configs.TINY_B, "C": configs.TINY_C, "D": dict(configs.TINY_D, num_hidden_layers=4), "turevik": entry.SMOKE_TUREVIK,
          "porarax": entry.SMOKE_PORARAX, "sogazen": entry.SMOKE_SOGAZEN, "kimutar": entry.SMOKE_KIMUTAR, "kefetar": entry.SMOKE_KEFETAR,
          "fobatar": entry.SMOKE_FOBATAR}


def _tensors(specs, seed):
    g = torch.Generator().manual_seed(seed)
    return {s.name: (torch.randn(s.shape, generator=g) * 0.2).bfloat16() for s in specs}


def _dequantised(q, scale):
    return q.double() * scale.double()[..., None]


def test_a_projection_with_scales_biases_padded_heads_and_gathered_rows():
    lin = StackedLinear(64)
    lin.add("a", 48, "a.b", in_scale=1.5, out_scale=0.7)
    lin.add("b", 32, None, out_scale=[0.1 * i for i in range(32)], heads=(2, 11, 16))
    lin.add("c", 5, "c.b", gather=(4, (3, 0, 0, 2, 1)))
    t = _tensors(lin.weight_specs(), 0)
    lin.bind(t, torch.bfloat16, DEV)
    full = lin.weight.double() * (lin.colscale.double()[:, None] if lin.colscale is not None else 1.0)
    lin.to_int8()
    assert lin.weight.dtype == torch.int8 and lin.colscale is None
    # a channel's integers stand for its weights to half a step
    assert bool(((_dequantised(lin.weight, lin.int8_scale) - full).abs() <= 0.501 * lin.int8_scale.double().abs()[:, None] + 1e-12).all())
    x = torch.randn(7, 64, device=DEV).bfloat16()
    q, s = ops.rows_int8(x)
    want = _dequantised(q, s) @ _dequantised(lin.weight, lin.int8_scale).T + lin.colbias.double()
    for given in (x, (q, s)):
        out = torch.empty(7, lin.out_features, device=DEV)
        lin.forward(given, out)
        assert float((out.double() - want).abs().max()) <= 1e-6 * float(want.abs().max())
        lin.forward(given, out, accumulate=True)
        assert float((out.double() - 2 * want).abs().max()) <= 2e-6 * float(want.abs().max())


@pytest.mark.parametrize("F", [96, 52])
def test_a_gated_feed_forward(F):
    ffn = SwiGLU(64, F, "", bias=True, gate_scale=0.8, down_scale=1.3)
    ffn.bind(_tensors(ffn.weight_specs(), 1), torch.bfloat16, DEV)
    x, base = torch.randn(9, 64, device=DEV).bfloat16(), torch.randn(9, 64, device=DEV)
    before, after = base.clone(), base.clone()
    ffn.forward(x, before)
    ffn.to_int8()
    assert ffn.takes_int8
    ffn.forward(x, after)
    again = base.clone()
    ffn.forward(ops.rows_int8(x), again)
    assert torch.equal(after, again)
    y = _dequantised(*ops.rows_int8(x)) @ _dequantised(ffn.gate_up.weight, ffn.gate_up.int8_scale).T + ffn.gate_up.colbias.double()
    act = (torch.nn.functional.silu(y[:, :F]) * y[:, F:]).bfloat16()
    want = base.double() + _dequantised(*ops.rows_int8(act)) @ _dequantised(ffn.down.weight, ffn.down.int8_scale).T + ffn.down.colbias.double()
    # (an activation that rounds to another 16-bit value, 2^-8 of it, or to another integer, 1/127 of the row's largest)
    assert float((after.double() - want).abs().max()) <= 0.02 * float((want - base.double()).abs().max())
    assert float((after - before).norm()) <= 0.06 * float((before - base).norm())


@pytest.mark.parametrize("weights,act,shared", [("sigmoid", "silu", False), ("softmax", "silu", True), ("softmax_all", "relu_squared", False)])
def test_experts(weights, act, shared):
    from tinyllama_c_b200.parts.base import PartSpec
    names = dict(gate="e{e}.g", up="e{e}.u", down="e{e}.d")
    moe = MoEFeedForward(64, 6, 2, 40, "router", names, weights=weights, weight_on="output" if act == "relu_squared" else "input", act=act,
                         shared=PartSpec("feed_forward", "swiglu", dict(hidden=64, intermediate=48, prefix="s.")) if shared else None,
                         shared_gate_name="sg" if shared else None, n_identity=1 if weights == "softmax_all" else 0)
    moe.bind(_tensors(moe.weight_specs(), 2), torch.bfloat16, DEV)
    int8 = copy.deepcopy(moe)
    int8.to_int8()
    assert int8.w_gate_up.dtype == torch.int8 and moe.w_gate_up.dtype == torch.bfloat16
    for T in (1, 3, 50):
        x = torch.randn(T, 64, device=DEV).bfloat16()
        before, after = torch.zeros(T, 64, device=DEV), torch.zeros(T, 64, device=DEV)
        moe.forward(x, before)
        int8.forward(x, after)
        assert bool(torch.isfinite(after).all()) and float((after - before).norm()) <= 0.08 * float(before.norm())
    ops.check_errors()


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("models")
    # (weights that neither wash the layers out nor let one layer's rounding decide the next one's tokens)
    return {name: make_model_dir(root, cfg, seed=7, name=name, std=0.1) for name, cfg in MODELS.items()}


@pytest.mark.parametrize("name", list(MODELS))
def test_whole_models_are_near_their_16_bit_selves(folders, name):
    logits = []
    for weights in (None, "int8"):
        llm = tlc.LLM(folders[name], max_tokens=1024, max_seqs=4, weights=weights)
        toks = [random_tokens(llm.model.vocab, n, 3 + n) for n in (70, 9, 1)]
        slots = [llm.cache.acquire() for _ in toks]
        out = [llm.step([StepEntry(s, t, [len(t) - 1]) for s, t in zip(slots, toks)])]
        for i in range(3):
            out.append(llm.step([StepEntry(s, [(5 * i + 1) % llm.model.vocab], [0]) for s in slots]))
        logits.append(torch.cat(out).float())
        ops.check_errors()
    plain, int8 = logits
    assert bool(torch.isfinite(int8).all())
    assert float((int8 - plain).norm()) <= 0.25 * float(plain.norm()), float((int8 - plain).norm() / plain.norm())
    assert not torch.equal(int8, plain)


def test_generation_through_the_entry_point_and_decoding_as_in_the_prompt(folders):
    llm = tlc.LLM(folders["D"], max_tokens=1024, max_seqs=4, weights="int8")
    prompts = [random_tokens(llm.model.vocab, n, n) for n in (33, 5)]
    res = llm.generate(prompts, tlc.GREEDY, max_new_tokens=8, ignore_eos=True)
    eager = tlc.LLM(llm.model, max_tokens=1024, max_seqs=4, use_graphs=False)
    for r, e in zip(res, eager.generate(prompts, tlc.GREEDY, max_new_tokens=8, ignore_eos=True)):
        assert r.tokens == e.tokens and len(r.tokens) == 8


def test_layers_repeated_from_a_table_give_the_same_bits(folders):
    llm = tlc.LLM(folders["D"], max_tokens=1024, max_seqs=4, weights="int8")
    assert llm.model.repeated is not None
    got = []
    calls = []
    for repeat in (True, False):
        if not repeat:
            llm.model.repeated = None
        slot = llm.cache.acquire()
        replayed, real = [], ops.replay
        ops.replay = lambda f, w, n: (replayed.append(n), real(f, w, n))
        try:
            got.append(llm.step([StepEntry(slot, random_tokens(llm.model.vocab, 60, 1), list(range(60)))]))
        finally:
            ops.replay = real
        calls.append(sum(replayed))
        llm.cache.release(slot)
    assert torch.equal(*got)
    assert calls == [3, 0]


def test_a_bound_model_and_what_it_holds(folders):
    model = tlc.load_model(folders["B"])
    held = sum(t.numel() * t.element_size() for t in (model.layers[0].fused_in.weight, model.layers[0].ffn.down.weight))
    llm = tlc.LLM(model, max_tokens=256, max_seqs=2, weights="int8")
    block = llm.model.layers[0]
    assert block.fused_in.weight.dtype == torch.int8 and block.ffn.down.weight.dtype == torch.int8
    assert 2 * sum(t.numel() for t in (block.fused_in.weight, block.ffn.down.weight)) == held
    for m in block.mixers:                                # the mixers' own are ranges of the fused ones
        assert m.input_projection().weight.untyped_storage().data_ptr() == block.fused_in.weight.untyped_storage().data_ptr()
    before = [p.weight for p in (block.fused_in, block.ffn.gate_up)]
    llm.model.to_int8()                                   # a second time changes nothing
    assert all(a is b for a, b in zip(before, (block.fused_in.weight, block.ffn.gate_up.weight)))


@pytest.mark.parametrize("name", ["linear_int8", "linear_swiglu_int8", "rmsnorm_int8", "_call_packed"])
def test_a_function_around_a_product_is_called_for_every_layer(folders, name, monkeypatch):
    llm = tlc.LLM(folders["D"], max_tokens=1024, max_seqs=4, weights="int8")
    tokens = random_tokens(llm.model.vocab, 60, 1)
    layers = len(llm.model.layers)

    def step():
        slot = llm.cache.acquire()
        out = llm.step([StepEntry(slot, tokens, [59])])
        llm.cache.release(slot)
        return out

    want = step()
    real, calls = getattr(ops, name), []
    monkeypatch.setattr(ops, name, lambda *a, **k: (calls.append(name), real(*a, **k))[1])
    assert torch.equal(step(), want)
    assert len(calls) % layers == 0 and len(calls) >= layers
