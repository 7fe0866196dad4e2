"""What the parts of a model hold and compute once their weights are 8-bit integers, against the formulas in 64 bits on those integers.

Allowances: a weight stands half a step (its channel's scale) off at most, a 16-bit weight's step being exact in 32 bits up to 1e-6 of
it.  A product of given integers is off by a few units in the last place of 32 bits (1e-6 of the largest term's size).  An activation
between two products that lies next to a half may go either way: a hundredth of the result's size (test_gpu_int8_model.py).  Decoding and
the prompt differ by the 16-bit rounding of what other kernels make, which moves integers next to a half: less than the rounding to
integers itself, which is 5 % of a logit; 10 % are allowed, where a wrong position, scale or weight gives 100 %."""
import pytest
import torch

import tinyllama_c_b200 as tlc
from tinyllama_c_b200 import ops
from tinyllama_c_b200.engine import StepEntry
from tinyllama_c_b200.parts.feed_forward import MoEFeedForward

import configs
import __graft_entry__ as entry
from helpers import make_model_dir, random_tokens

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
MODELS = {"A": configs.TINY_A, "B": configs.TINY_B, "C": configs.TINY_C, "D": dict(configs.TINY_D, num_hidden_layers=4), "turevik": entry.SMOKE_TUREVIK,
          "kefetar": entry.SMOKE_KEFETAR}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("models")
    return {name: make_model_dir(root, cfg, seed=7, name=name, std=0.1) for name, cfg in MODELS.items()}


def _columns(weight, scale):
    return weight.double() * (scale.double()[:, None] if scale is not None else 1.0)


@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_mixers_own_projections_are_their_16_bit_selves_to_half_a_step(folders, name):
    """Behind shared input and output products a mixer's own projection is a range of the shared matrix, with scales of its own."""
    model = tlc.load_model(folders[name])
    block = model.layers[0]
    assert block.fused_in is not None
    projections = [(kind, getattr(m, kind)()) for m in block.mixers for kind in ("input_projection", "output_projection")]
    before = [_columns(p.weight, p.colscale) for _, p in projections]
    model.to_int8()
    for (kind, p), w in zip(projections, before):
        assert p.weight.dtype == torch.int8 and p.colscale is None and p.int8_scale.shape == (p.out_features,)
        off = (_columns(p.weight, p.int8_scale) - w).abs()
        assert bool((off <= 0.5 * (1 + 1e-5) * p.int8_scale.double().abs()[:, None] + 1e-12).all()), kind
        # ... and by itself it multiplies with them
        x = torch.randn(5, p.in_features, device=DEV).bfloat16()
        q, s = ops.rows_int8(x)
        want = _columns(q, s) @ _columns(p.weight, p.int8_scale).T + (p.colbias.double() if p.colbias is not None else 0)
        out = torch.empty(5, p.out_features, device=DEV)
        p.forward(x, out)
        assert float((out.double() - want).abs().max()) <= 1e-6 * float(want.abs().max())
    if block.fused_out is None:
        return
    # the shared product of inputs that lie side by side, scaled as the layer scales them, is the sum of the mixers' own
    outs = [p for kind, p in projections if kind == "output_projection"]
    rows = [torch.randint(-127, 128, (5, p.in_features), device=DEV, dtype=torch.int8) for p in outs]
    want = sum(_columns(r, torch.ones(5, device=DEV)) @ _columns(p.weight, p.int8_scale).T for r, p in zip(rows, outs))
    got = torch.zeros(5, outs[0].out_features, dtype=torch.float64, device=DEV)
    for r, (off, n), factor in zip(rows, block.out_offsets, block.out_scales):
        joint = ops.int8_empty(5, block.fused_out.in_features, DEV).zero_()
        joint[:, off:off + n] = r
        part = torch.empty(5, outs[0].out_features, device=DEV)
        ops.linear_int8(joint, block.fused_out.weight, block.fused_out.int8_scale, part, torch.full((5,), factor, device=DEV))
        got += part.double()
    assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max())


def _silu(z):
    return z * torch.sigmoid(z)


@pytest.mark.parametrize("weights,weight_on,act", [("sigmoid", "input", "silu"), ("softmax", "output", "silu"), ("softmax_all", "output", "relu_squared")])
@pytest.mark.parametrize("T", [1, 3, 50])
def test_a_layer_of_experts(T, weights, weight_on, act):
    """Against the experts one by one in 64 bits, chosen from the part's own router in 64 bits."""
    names = dict(gate="e{e}.g", up="e{e}.u", down="e{e}.d")
    moe = MoEFeedForward(64, 6, 2, 40, "router", names, weights=weights, weight_on=weight_on, act=act)
    g = torch.Generator().manual_seed(5)
    moe.bind({s.name: (torch.randn(s.shape, generator=g) * 0.2).bfloat16() for s in moe.weight_specs()}, torch.bfloat16, DEV)
    assert moe.to_int8() == 2
    x = torch.randn(T, 64, generator=g).to(DEV).bfloat16()
    got = torch.zeros(T, 64, device=DEV)
    moe.forward(x, got)
    ops.check_errors()
    z = x.double() @ moe.router.double().T
    best = z.topk(2)
    share = torch.sigmoid(best.values) if weights == "sigmoid" else torch.softmax(best.values, -1) if weights == "softmax" \
        else torch.softmax(z, -1).gather(1, best.indices)
    q, s = ops.rows_int8(x)
    want = torch.zeros(T, 64, dtype=torch.float64, device=DEV)
    for t in range(T):
        for k in range(2):
            e, f = int(best.indices[t, k]), share[t, k]
            y = _columns(q[t:t + 1], s[t:t + 1]) @ _columns(moe.w_gate_up[e], moe.gate_up_scale[e]).T
            y = y * f if weight_on == "input" else y
            a = y.clamp(min=0).square() if act == "relu_squared" else _silu(y[:, :40]) * y[:, 40:]
            step = a.abs().max() / 127
            y = torch.round(a / step) * step @ _columns(moe.w_down[e], moe.down_scale[e]).T
            want[t] += y[0] * (f if weight_on == "output" else 1.0)
    assert float((got.double() - want).abs().max()) <= 0.01 * float(want.abs().max())


@pytest.mark.parametrize("name", list(MODELS))
def test_decoding_as_in_the_prompt(folders, name):
    """The logits of a prompt's last tokens, brought one by one and all at once."""
    llm = tlc.LLM(folders[name], max_tokens=1024, max_seqs=2, weights="int8")
    tokens = random_tokens(llm.model.vocab, 40, 3)
    whole, apart = llm.cache.acquire(), llm.cache.acquire()
    want = llm.step([StepEntry(whole, tokens, [36, 37, 38, 39])]).float()
    llm.step([StepEntry(apart, tokens[:36], [])])
    got = torch.cat([llm.step([StepEntry(apart, tokens[i:i + 1], [0])]) for i in range(36, 40)]).float()
    ops.check_errors()
    assert float((got - want).norm()) <= 0.1 * float(want.norm()), float((got - want).norm() / want.norm())


@pytest.mark.parametrize("M", [1, 2, 7, 12, 24, 200])
def test_weights_that_pass_32_bits(M):
    """More than 2^32 bytes of weights: their last rows, by every kernel that these numbers of rows take."""
    K, N = 8208, 530_000
    w = torch.empty(N, K, dtype=torch.int8, device=DEV)
    assert w.numel() > 1 << 32
    w[:64].random_(-127, 128)
    w[-64:].random_(-127, 128)
    sw = torch.full((N,), 0.01, device=DEV)
    for k in (8208, 2048):
        a, sa = ops.rows_int8(torch.randn(M, k, device=DEV))
        out, ends = torch.empty(M, N, device=DEV), torch.empty(M, 128, device=DEV)
        ops.linear_int8(a, w[:, :k], sw, out, a_scale=sa)
        ops.linear_int8(a, torch.cat([w[:64, :k], w[-64:, :k]]), sw[:128], ends, a_scale=sa)
        assert torch.equal(torch.cat([out[:, :64], out[:, -64:]], 1), ends)
    ops.check_errors()
