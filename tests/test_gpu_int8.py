"""Products in 8-bit integers against their formulas in 64 bits.

Allowances, with u = 2^-24 (half a unit in the last place of 32 bits):
  rows      the scale is a quotient: u of it (3u are allowed).  An integer differs from the quotient in 64 bits
            by 1/2 and what the division and the scale are off: 127 * 4u.  Behind the norm the products x w add 2u to both, and the
            scale has the root of a mean of squares: at most 42 sums in a row (21u after the root), rsqrt 4u, products 4u.
  products  the sum is exact; conversion, two scales: 3u of the result; a bias, an old value: u of each sum's size.  A 16-bit result
            is rounded once, to 8 bits: 2^-8 of it at most.
  gated     gate and up 4u each, which silu turns into (1 + |gate|) 4u, the exponential (2 + 1.2 |gate|) 2u, division 4u,
            product u: below 2e-6 (1 + |gate|) of the result.
  experts   the activation between the products is rounded to integers: one that lies within 127 * (its own relative error) of a half may
            go to either side, and each that does moves a result by at most 127 * both scales.  The reference counts them.
"""
import numpy as np
import pytest
import torch

import tinyllama_c_b200 as tlc
from tinyllama_c_b200 import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.empty(*shape, device=DEV).normal_(generator=g) * std).to(dtype)


def integers(g, *shape):
    """-127..127, rows on 16-byte boundaries."""
    k = shape[-1]
    full = torch.randint(-127, 128, (*shape[:-1], (k + 15) // 16 * 16), generator=g, device=DEV, dtype=torch.int8)
    return full[..., :k]


def scales(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV) * 0.02 + 1e-4


def rows_64(v):
    """(quotients, integers, scale) in 64 bits."""
    v = v.double()
    scale = v.abs().amax(-1) / 127
    quotient = v / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    return quotient, torch.round(quotient), scale


def product_64(a, sa, w, sw):
    return (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()[None, :]


def near(out, ref, size=None, rel=4 * U):
    """out against ref, allowed rel of `size` (default: of the result) and one rounding to out's type."""
    size = ref.abs() if size is None else size
    allowed = rel * size + (2.0 ** -8 * 1.001 * ref.abs() if out.dtype == torch.bfloat16 else 0) + 1e-37
    off = (out.double() - ref).abs()
    assert bool((off <= allowed).all()), f"largest error / allowance {float((off / allowed).max()):.3f}"


# ---- rows ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K", [(1, 1), (3, 7), (1, 2048), (5, 1023), (64, 2560), (2, 4097), (3, 8192), (2, 16384), (2, 20001)])
def test_rows(T, K, dtype):
    x = normal(gen(T + K), T, K, dtype=dtype)
    x[:, 0] *= 9
    q, scale = ops.rows_int8(x)
    quotient, _, ref = rows_64(x)
    assert q.dtype == torch.int8 and tuple(q.shape) == (T, K) and q.stride(0) % 16 == 0
    assert bool(((scale.double() - ref).abs() <= 3 * U * ref).all())
    assert float((q.double() - quotient).abs().max()) <= 0.5 + 127 * 4 * U
    assert bool((q.abs().amax(1) == 127).all())


@pytest.mark.parametrize("T,K", [(1, 64), (7, 2048), (33, 2560), (2, 8193), (2, 16392)])
def test_rows_behind_the_norm(T, K):
    g = gen(T * K)
    x, w = normal(g, T, K, std=3.0), normal(g, K) * 0.1 + 1
    q, scale = ops.rmsnorm_int8(x, w, 1e-5)
    v = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    quotient, _, ref = rows_64(v)
    assert bool(((scale.double() - ref).abs() <= 34 * U * ref).all())
    assert float((q.double() - quotient).abs().max()) <= 0.5 + 127 * 8 * U


def test_rows_with_nothing_or_nonsense_in_them():
    x = normal(gen(0), 8, 300)
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 299] = float("nan")
    x[4] *= 1e-42                                      # below what a scale can hold
    x[5, 11] = -float("inf")
    x[6] *= 1e30
    x[7] *= 1e-30
    q, scale = ops.rows_int8(x)
    assert scale[1] == 0 and scale[4] == 0 and not q[1].any() and not q[4].any()
    for r in (2, 3, 5):
        assert torch.isnan(scale[r]) and not q[r].any()
    for r in (0, 6, 7):
        assert float((q[r].double() - x[r].double() / (x[r].double().abs().max() / 127)).abs().max()) <= 0.5 + 127 * 4 * U
    # what is multiplied by them: nothing, or NaN, and the other rows are as they are alone
    w, sw = integers(gen(1), 96, 300), scales(gen(2), 96)
    out, alone = torch.empty(8, 96, device=DEV), torch.empty(1, 96, device=DEV)
    ops.linear_int8(x, w, sw, out)
    assert not out[1].any() and not out[4].any() and bool(torch.isnan(out[[2, 3, 5]]).all())
    for r in (0, 6, 7):
        ops.linear_int8(x[r:r + 1], w, sw, alone)
        assert torch.equal(out[r], alone[0])


def test_halves_go_to_the_even_integer_and_the_lowest_integer_is_minus_127():
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, -127.0]], device=DEV)
    q, scale = ops.rows_int8(x)
    assert q[0].tolist() == [127, 0, 2, 2, 0, -2, -126, -127] and float(scale) == 1.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_integers_are_those_of_the_quotients(dtype):
    """Integer by integer what dividing in 32 bits and rounding gives, over many magnitudes (one row in 128 of 16-bit rows is full of
    quotients that are halves exactly)."""
    g = gen(11)
    for K in (8, 64, 2048):
        x = normal(g, (1 << 22) // K, K) * torch.empty((1 << 22) // K, 1, device=DEV).uniform_(-30, 30, generator=g).exp2()
        x = x.to(dtype)
        q, scale = ops.rows_int8(x)
        largest = x.float().abs().amax(1)
        s = largest / torch.full((), 127.0, device=DEV)
        assert torch.equal(scale, s) and torch.equal(q, torch.round(x.float() / s[:, None]).to(torch.int8))


def test_rows_of_strided_and_unaligned_views():
    g = gen(3)
    big = normal(g, 9, 700, dtype=torch.bfloat16)
    for view in (big[:, 3:515], big[::2, 8:520], big[1:2, 1:]):
        q, scale = ops.rows_int8(view)
        q2, scale2 = ops.rows_int8(view.contiguous())
        assert torch.equal(q, q2) and torch.equal(scale, scale2)


def test_weight_scales_are_per_output_channel():
    w = normal(gen(4), 3, 40, 72, std=0.02, dtype=torch.bfloat16)
    q, scale = ops.weight_int8(w)
    assert tuple(q.shape) == (3, 40, 72) and tuple(scale.shape) == (3, 40) and q.stride() == (40 * 80, 80, 1)
    quotient, _, ref = rows_64(w)
    assert float((q.double() - quotient).abs().max()) <= 0.5 + 127 * 4 * U and bool(((scale.double() - ref).abs() <= 3 * U * ref).all())
    q2, scale2 = ops.weight_int8(w[1])
    assert torch.equal(q2, q[1]) and torch.equal(scale2, scale[1])


# ---- products --------------------------------------------------------------------------------------------
ROWS = [1, 2, 4, 5, 8, 9, 16, 17, 24, 32, 33, 64, 65, 100, 128, 129, 200, 256, 257, 300, 513]
SHAPES = [(64, 128), (128, 2048), (130, 80), (1000, 272), (2048, 4096), (8240, 512), (37, 2560), (1, 64), (257, 1040), (2560, 8192)]


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("N,K", SHAPES[:7])
def test_product(M, N, K):
    g = gen(M * N + K)
    a, sa, w, sw = integers(g, M, K), scales(g, M), integers(g, N, K), scales(g, N)
    ref = product_64(a, sa, w, sw)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((M, N), float("nan"), dtype=dtype, device=DEV)
        ops.linear_int8(a, w, sw, out, a_scale=sa)
        near(out, ref)
    ops.check_errors()


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 5, 7), (2, 300, 33), (40, 70, 1001), (130, 129, 15), (300, 33, 130), (1, 2048, 2049),
                                   (600, 2000, 96), (1024, 1536, 640), (2049, 300, 128), (5, 17, 131071), (200, 16, 131071), (16, 40000, 64)])
def test_product_of_odd_and_extreme_sizes(M, N, K):
    g = gen(M + N + K)
    a, sa, w, sw = integers(g, M, K), scales(g, M), integers(g, N, K), scales(g, N)
    bias = normal(g, N)
    ref = product_64(a, sa, w, sw)
    out = torch.empty(M, N, device=DEV)
    ops.linear_int8(a, w, sw, out, a_scale=sa, colbias=bias)
    near(out, ref + bias.double(), ref.abs() + bias.double().abs())
    ops.check_errors()


@pytest.mark.parametrize("M", [1, 3, 20, 130, 600])
def test_sums_at_the_edge_of_32_bits_are_exact(M):
    K = 131071
    a = torch.full((M, K), -128, dtype=torch.int8, device=DEV)
    w = torch.full((48, K + 1), -128, dtype=torch.int8, device=DEV)[:, :K]
    w[1::2] = 127
    one = torch.ones(max(M, 48), device=DEV)
    out = torch.empty(M, 48, device=DEV)
    ops.linear_int8(a, w, one[:48], out, a_scale=one[:M])
    assert bool((out[:, ::2] == float(np.float32(128 * 128 * K))).all()) and bool((out[:, 1::2] == float(np.float32(-128 * 127 * K))).all())


@pytest.mark.parametrize("M", [1, 7, 24, 90, 260])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K", [(96, 320), (1040, 2048)])
def test_product_added_to_what_is_there(M, N, K, dtype):
    g = gen(M + N)
    a, sa, w, sw, bias = integers(g, M, K), scales(g, M), integers(g, N, K), scales(g, N), normal(g, N)
    old = normal(g, M, N, std=30.0, dtype=dtype)
    out = old.clone()
    ops.linear_int8(a, w, sw, out, a_scale=sa, colbias=bias, accumulate=True)
    ref = product_64(a, sa, w, sw)
    near(out, ref + bias.double() + old.double(), ref.abs() + bias.double().abs() + old.double().abs(), 5 * U)


@pytest.mark.parametrize("M", [3, 40, 150])
def test_views_with_strides_and_off_the_boundaries(M):
    g = gen(M)
    N, K = 200, 384
    a, sa, w, sw = integers(g, M, K), scales(g, M), integers(g, N, K), scales(g, N)
    ref = product_64(a, sa, w, sw)
    room_a = torch.zeros(2 * M, 1024, dtype=torch.int8, device=DEV)
    room_w = torch.zeros(N, 3 * K + 5, dtype=torch.int8, device=DEV)
    for off_a in (0, 16, 3):
        for off_w in (0, 1):
            va, vw = room_a[::2, off_a:off_a + K], room_w[:, off_w:off_w + K]
            va.copy_(a)
            vw.copy_(w)
            room = torch.full((M, N + 8), 7.0, device=DEV)
            ops.linear_int8(va, vw, sw, room[:, 3:3 + N], a_scale=sa)
            near(room[:, 3:3 + N], ref)
            assert bool((room[:, :3] == 7).all()) and bool((room[:, 3 + N:] == 7).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(1, 512, 2048), (8, 100, 1001), (23, 2560, 640), (140, 300, 2050), (700, 520, 256)])
def test_rows_are_rounded_within_the_call(M, N, K, dtype):
    """The call that rounds its rows gives the bits of the two calls."""
    g = gen(M + K)
    x, w, sw = normal(g, M, K, dtype=dtype), integers(g, N, K), scales(g, N)
    q, sa = ops.rows_int8(x)
    for odt in (torch.float32, torch.bfloat16):
        one, two = torch.empty(M, N, dtype=odt, device=DEV), torch.empty(M, N, dtype=odt, device=DEV)
        ops.linear_int8(x, w, sw, one)
        ops.linear_int8(q, w, sw, two, a_scale=sa)
        assert torch.equal(one, two)
    near(two, product_64(q, sa, w, sw))


def gated_64(act, y, limit, alpha):
    F = y.shape[1] // 2
    g, u = y[:, :F], y[:, F:]
    if act == "swish_clamped":
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        return g, g * torch.sigmoid(alpha * g) * (u + 1)
    if act == "gelu_tanh":
        return g, torch.nn.functional.gelu(g, approximate="tanh") * u
    return g, g * torch.sigmoid(g) * u


@pytest.mark.parametrize("M", [1, 2, 8, 16, 17, 40, 65, 128, 129, 300])
@pytest.mark.parametrize("F,K", [(64, 256), (688, 2048), (100, 144), (33, 65), (1024, 512), (4096, 128)])
def test_gated(M, F, K):
    g = gen(M + F + K)
    a, sa, w, sw = integers(g, M, K), scales(g, M) * 0.05, integers(g, 2 * F, K), scales(g, 2 * F) * (30 / K ** 0.5)
    bias = normal(g, 2 * F)
    y = product_64(a, sa, w, sw) + bias.double()
    size = product_64(a, sa, w, sw).abs() + bias.double().abs()
    gate, ref = gated_64("silu", y, 0, 1)
    # gate and up are off by 4u of `size`, which counts through silu's slope (at most 1.1) and through up
    allowed = 2e-6 * (1 + gate.abs()) * ref.abs() + 6 * U * (1.1 * size[:, :F] * y[:, F:].abs() + size[:, F:] * gate.abs())
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((M, F), float("nan"), dtype=dtype, device=DEV)
        ops.linear_swiglu_int8(a, w, sw, out, a_scale=sa, colbias=bias)
        near(out, ref, allowed, 1.0)
    ops.check_errors()


@pytest.mark.parametrize("act,limit,alpha", [("gelu_tanh", 0.0, 1.0), ("swish_clamped", 1.5, 1.7)])
@pytest.mark.parametrize("M,F,K", [(3, 64, 256), (50, 200, 512), (200, 136, 272)])
def test_other_activations(act, limit, alpha, M, F, K):
    g = gen(M + F)
    a, sa, w, sw = integers(g, M, K), scales(g, M) * 0.02, integers(g, 2 * F, K), scales(g, 2 * F) * (30 / K ** 0.5)
    y = product_64(a, sa, w, sw)
    _, ref = gated_64(act, y, limit, alpha)
    out = torch.empty(M, F, device=DEV)
    ops.linear_swiglu_int8(a, w, sw, out, a_scale=sa, act=act, limit=limit, alpha=alpha)
    # (gelu's cube and tanh: 1 - tanh is off by its argument's error times 2)
    assert float((out.double() - ref).abs().max()) <= 1e-5 * float((1 + y.abs()).square().max())


# ---- experts ---------------------------------------------------------------------------------------------
def make_routing(expert, weight, E):
    """ids, weights, order, offsets of chosen experts [T, top], as moe_route leaves them."""
    ids = expert.flatten().to(torch.int32)
    order = torch.argsort(ids, stable=True).to(torch.int32)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
    offsets[1:] = torch.bincount(ids.long(), minlength=E).cumsum(0)
    return ids, weight.flatten().contiguous(), order, offsets, None, 0


def experts_64(x, wgu, sgu, wd, sd, expert, weight, act, weight_on, limit, alpha):
    """(results [T, top, D], allowance for integers next to a half)."""
    T, top = expert.shape
    D, F = wd.shape[1], wd.shape[2]
    y = torch.zeros(T, top, D, dtype=torch.float64, device=DEV)
    slack = torch.zeros_like(y)
    qx, sx = ops.rows_int8(x)                          # (what test_rows is about)
    for t in range(T):
        q, s = qx[t:t + 1], sx[t:t + 1]
        for k in range(top):
            e, wt = int(expert[t, k]), float(weight[t, k])
            h = product_64(q, s, wgu[e], sgu[e])
            if weight_on == "input":
                h = h * wt
            if act == "relu_squared":
                gate = h
                v = h.clamp(min=0).square()
            else:
                gate, v = gated_64(act, h, limit, alpha)
            quotient, q2, s2 = rows_64(v)
            # the activation's own error, relative to the row's largest: both gate's and up's through the product
            err = 127 * (4e-6 * (1 + gate.abs().max()))
            close = ((quotient - torch.floor(quotient) - 0.5).abs() <= err).sum()
            f = wt if weight_on == "output" else 1.0
            y[t, k] = product_64(q2, s2, wd[e], sd[e])[0] * f
            slack[t, k] = float(close) * 127 * float(s2) * abs(f) * sd[e].double()
            slack[t, k] += 4e-6 * (1 + gate.abs().max()) * (q2.abs().sum() * 127 * float(s2) * abs(f) * sd[e].double() * 0.05 + y[t, k].abs())
    return y, slack


@pytest.mark.parametrize("T,E,top,F,D,act,weight_on", [
    (1, 4, 2, 64, 128, "silu", "input"), (5, 8, 3, 96, 256, "silu", "output"), (40, 3, 2, 72, 80, "gelu_tanh", "output"),
    (23, 6, 2, 33, 65, "silu", "input"), (70, 2, 1, 128, 272, "swish_clamped", "output"), (30, 5, 2, 144, 128, "relu_squared", "output"),
    (9, 40, 4, 64, 144, "silu", "output"), (150, 2, 2, 200, 128, "silu", "input"), (3, 1, 1, 1024, 2048, "silu", "output")])
def test_experts(T, E, top, F, D, act, weight_on):
    g = gen(T + E + F)
    x = normal(g, T, D, dtype=torch.bfloat16)
    wgu, sgu = integers(g, E, F if act == "relu_squared" else 2 * F, D), scales(g, E, F if act == "relu_squared" else 2 * F) * (3 / D ** 0.5)
    wd, sd = integers(g, E, D, F), scales(g, E, D)
    logits = normal(g, T, E)
    best = logits.topk(top)
    weight = torch.softmax(best.values, -1)
    ref, slack = experts_64(x, wgu, sgu, wd, sd, best.indices, weight, act, weight_on, 2.0, 1.3)
    for routing in (ops.moe_route(logits, E, top, weights="softmax"), make_routing(best.indices, weight, E)):
        for dtype in (torch.float32, torch.bfloat16):
            y = torch.full((T, top, D), float("nan"), dtype=dtype, device=DEV)
            ops.moe_experts_int8(x, wgu, sgu, wd, sd, routing, top, y, act_fn=act, weight_on=weight_on, limit=2.0, alpha=1.3)
            near(y, ref, 12 * U * ref.abs() + slack, 1.0)
    ops.check_errors()


@pytest.mark.parametrize("T,E", [(1, 300), (33, 7), (260, 3), (520, 64)])
def test_every_row_to_one_expert_or_each_to_its_own(T, E):
    g = gen(T)
    F, D = 64, 128
    x = normal(g, T, D)
    wgu, sgu, wd, sd = integers(g, E, 2 * F, D), scales(g, E, 2 * F) * 0.2, integers(g, E, D, F), scales(g, E, D)
    w = torch.rand(T, 1, generator=g, device=DEV) + 0.1
    alone = torch.empty(T, F, device=DEV)
    for expert in (torch.full((T, 1), E - 1, device=DEV), torch.arange(T, device=DEV)[:, None] % E):
        y = torch.empty(T, 1, D, device=DEV)
        ops.moe_experts_int8(x, wgu, sgu, wd, sd, make_routing(expert, w, E), 1, y, weight_on="output")
        for e in expert.unique().tolist():                     # the same as the expert's own two products
            rows = (expert[:, 0] == e).nonzero()[:, 0]
            act, back = torch.empty(len(rows), F, device=DEV), torch.empty(len(rows), D, device=DEV)
            ops.linear_swiglu_int8(x[rows], wgu[e], sgu[e], act)
            ops.linear_int8(act, wd[e], sd[e], back)
            near(y[rows, 0], back.double() * w[rows].double(), rel=6 * U)


def test_an_expert_result_does_not_depend_on_the_others_in_the_batch():
    g = gen(77)
    T, E, top, F, D = 45, 6, 2, 80, 160
    x, logits = normal(g, T, D, dtype=torch.bfloat16), normal(g, T, E)
    wgu, sgu, wd, sd = integers(g, E, 2 * F, D), scales(g, E, 2 * F) * 0.2, integers(g, E, D, F), scales(g, E, D)
    y = torch.empty(T, top, D, device=DEV)
    ops.moe_experts_int8(x, wgu, sgu, wd, sd, ops.moe_route(logits, E, top), top, y)
    one = torch.empty(1, top, D, device=DEV)
    for t in (0, 7, T - 1):
        ops.moe_experts_int8(x[t:t + 1], wgu, sgu, wd, sd, ops.moe_route(logits[t:t + 1].contiguous(), E, top), top, one)
        assert torch.equal(one[0], y[t])


# ---- calls -----------------------------------------------------------------------------------------------
def test_nothing_to_do():
    w, sw = integers(gen(1), 64, 128), scales(gen(1), 64)
    q, scale = ops.rows_int8(torch.empty(0, 128, device=DEV))
    assert tuple(q.shape) == (0, 128) and scale.numel() == 0
    ops.linear_int8(torch.empty(0, 128, device=DEV), w, sw, torch.empty(0, 64, device=DEV))
    ops.linear_int8(q, w, sw, torch.empty(0, 64, device=DEV), a_scale=scale)
    ops.linear_swiglu_int8(q, w, sw, torch.empty(0, 32, device=DEV), a_scale=scale)
    ids = torch.empty(0, 1, dtype=torch.long, device=DEV)
    ops.moe_experts_int8(torch.empty(0, 128, device=DEV), w[None], sw[None], integers(gen(1), 1, 128, 32), scales(gen(1), 1, 128),
                         make_routing(ids, torch.empty(0, 1, device=DEV), 1), 1, torch.empty(0, 1, 128, device=DEV))
    torch.cuda.synchronize()


def test_refusals():
    E = ops.KernelError
    x, w, sw = normal(gen(1), 4, 128), integers(gen(1), 64, 128), scales(gen(1), 64)
    q, sa = ops.rows_int8(x)
    out = torch.empty(4, 64, device=DEV)
    for bad in (lambda: ops.linear_int8(x.cpu(), w, sw, out), lambda: ops.linear_int8(x, w.float(), sw, out),
                lambda: ops.linear_int8(x[:, :64], w, sw, out), lambda: ops.linear_int8(x, w, sw, out[:, :32]),
                lambda: ops.linear_int8(x, w, sw[:32], out), lambda: ops.linear_int8(x, w, sw.double(), out),
                lambda: ops.linear_int8(q, w, sw, out), lambda: ops.linear_int8(x, w, sw, out, a_scale=sa),
                lambda: ops.linear_int8(x.half(), w, sw, out), lambda: ops.linear_int8(x, w, sw, out.half()),
                lambda: ops.linear_int8(x.T.contiguous().T, w, sw, out), lambda: ops.linear_int8(x, w, sw, out, colbias=sw[:5]),
                lambda: ops.linear_int8(q, w, sw, out, a_scale=sa[:2]),
                lambda: ops.linear_int8(torch.zeros(1, ops.INT8_MAX_K + 1, device=DEV), torch.zeros(1, ops.INT8_MAX_K + 1, dtype=torch.int8, device=DEV),
                                        sw[:1], torch.empty(1, 1, device=DEV)),
                lambda: ops.linear_swiglu_int8(x, w[:63], sw[:63], out[:, :31]), lambda: ops.linear_swiglu_int8(x, w, sw, out[:, :32], act="tanh"),
                lambda: ops.rows_int8(x[0]), lambda: ops.rows_int8(x.half()), lambda: ops.rows_int8(torch.empty(3, 0, device=DEV)),
                lambda: ops.rmsnorm_int8(x, sw, 1e-5), lambda: ops.weight_int8(x[0])):
        with pytest.raises(E):
            bad()
    wgu, wd, logits = w[None].expand(2, 64, 128).contiguous(), integers(gen(1), 2, 128, 32), normal(gen(2), 4, 2)
    sgu, sd, y = scales(gen(1), 2, 64), scales(gen(1), 2, 128), torch.empty(4, 1, 128, device=DEV)
    r = ops.moe_route(logits, 2, 1)
    ops.moe_experts_int8(x, wgu, sgu, wd, sd, r, 1, y)
    for bad in (lambda: ops.moe_experts_int8(x, wgu, sgu, wd, sd, r, 2, torch.empty(4, 2, 128, device=DEV)),
                lambda: ops.moe_experts_int8(x, wgu, sgu, wd, sd, r, 1, y, act_fn="tanh"),
                lambda: ops.moe_experts_int8(x, wgu, sgu, wd, sd, r, 1, y, weight_on="both"),
                lambda: ops.moe_experts_int8(x, wgu[:, :62], sgu, wd, sd, r, 1, y),
                lambda: ops.moe_experts_int8(x, wgu, sgu, wd.float(), sd, r, 1, y),
                lambda: ops.moe_experts_int8(x, wgu, sgu[:1], wd, sd, r, 1, y),
                lambda: ops.moe_experts_int8(x[:, ::2], wgu, sgu, wd, sd, r, 1, y),
                lambda: ops.moe_experts_int8(x, wgu[:, :32].contiguous(), sgu[:, :32].contiguous(), wd, sd, r, 1, y, act_fn="relu_squared"),
                lambda: ops.moe_experts_int8(x, wgu, sgu, wd, sd, r, 1, y.transpose(0, 2))):
        with pytest.raises(E):
            bad()
    torch.cuda.synchronize()


def test_calls_in_a_graph_and_on_another_stream():
    g = gen(5)
    x, w, sw = normal(g, 6, 256, dtype=torch.bfloat16), integers(g, 192, 256), scales(g, 192)
    wg, sg = integers(g, 128, 192), scales(g, 128)
    out, mid = torch.empty(6, 64, device=DEV), torch.empty(6, 192, dtype=torch.bfloat16, device=DEV)

    def calls():
        ops.linear_int8(x, w, sw, mid)
        ops.linear_swiglu_int8(mid, wg, sg, out)

    calls()
    ref = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out.zero_()
        calls()
    side.synchronize()
    assert torch.equal(out, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    x2 = normal(g, 6, 256, dtype=torch.bfloat16)
    x.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    again = out.clone()
    calls()
    assert torch.equal(out, again) and not torch.equal(out, ref)


def test_weights_may_follow_at_once():
    """weight_int8 and, right behind it, products that fetch those weights ahead of their wait."""
    g = gen(6)
    for i in range(20):
        w = normal(g, 2048, 1024, dtype=torch.bfloat16)
        x = normal(g, 8, 1024)
        torch.cuda.synchronize()
        q, s = ops.weight_int8(w)
        out = torch.empty(8, 2048, device=DEV)
        ops.linear_int8(x, q, s, out)
        torch.cuda.synchronize()
        again = torch.empty(8, 2048, device=DEV)
        ops.linear_int8(x, q, s, again)
        assert torch.equal(out, again)


KERNELS = [(4, 0), (2, 16), (2, 32), (2, 64), (2, 128), (3, 128), (3, 256)]


@pytest.mark.parametrize("kernel", KERNELS)
def test_every_kernel_gives_the_same_bits(kernel):
    """The sums are exact, so a result does not depend on which kernel made it; it is compared with the CUDA cores'."""
    g = gen(9)
    for M, N, K in [(1, 200, 384), (3, 77, 2049), (8, 300, 4096), (40, 1000, 272), (129, 2050, 130), (515, 520, 1024), (300, 2048, 64)]:
        a, sa, w, sw = integers(g, M, K), scales(g, M), integers(g, N, K), scales(g, N)
        bias = normal(g, N)
        w2, sw2 = integers(g, 2 * 136, K), scales(g, 2 * 136) * 0.1
        for dtype in (torch.float32, torch.bfloat16):
            old = normal(g, M, N, dtype=dtype)
            got = []
            for k in ((1, 0), kernel):
                ops.linear_int8_kernel(*k)
                try:
                    outs = [torch.full((M, N), float("nan"), dtype=dtype, device=DEV), old.clone(), torch.full((M, 136), float("nan"), dtype=dtype, device=DEV)]
                    ops.linear_int8(a, w, sw, outs[0], a_scale=sa, colbias=bias)
                    ops.linear_int8(a, w, sw, outs[1], a_scale=sa, accumulate=True)
                    ops.linear_swiglu_int8(a, w2, sw2, outs[2], a_scale=sa)
                    got.append(outs)
                finally:
                    ops.linear_int8_kernel()
            for x, y in zip(*got):
                assert torch.equal(x, y)
    ops.check_errors()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("T,E,top,F,D,act,weight_on", [(1, 4, 2, 64, 128, "silu", "input"), (2, 9, 4, 129, 400, "silu", "output"),
                                                       (5, 3, 3, 65, 80, "relu_squared", "output"), (200, 5, 3, 136, 272, "silu", "output"),
                                                       (700, 3, 2, 72, 400, "silu", "input"), (33, 70, 4, 200, 128, "relu_squared", "output")])
def test_every_kernel_gives_the_same_experts(kernel, T, E, top, F, D, act, weight_on):
    g = gen(T)
    x, logits = normal(g, T, D, dtype=torch.bfloat16), normal(g, T, E)
    rows = F if act == "relu_squared" else 2 * F
    wgu, sgu, wd, sd = integers(g, E, rows, D), scales(g, E, rows) * 0.2, integers(g, E, D, F), scales(g, E, D)
    routing = ops.moe_route(logits, E, top, weights="softmax")
    for dtype in (torch.float32, torch.bfloat16):
        got = []
        for k in ((1, 0), kernel):
            ops.linear_int8_kernel(*k)
            try:
                y = torch.full((T, top, D), float("nan"), dtype=dtype, device=DEV)
                ops.moe_experts_int8(x, wgu, sgu, wd, sd, routing, top, y, act_fn=act, weight_on=weight_on)
                got.append(y)
            finally:
                ops.linear_int8_kernel()
        assert torch.equal(*got)
    ops.check_errors()


@pytest.mark.parametrize("M,N,K", [(1, 200, 384), (3, 77, 2049), (8, 300, 4096), (8, 1000, 272), (6, 2050, 130), (7, 2048, 64), (2, 33, 3001), (4, 16, 4095),
                                   (5, 9, 17), (8, 40, 4097)])
def test_few_rows_give_the_same_bits(M, N, K):
    """The kernel of up to 8 rows against the CUDA cores', at column counts and lengths that end inside a tile; rows of the activations on
    16-byte boundaries and off them."""
    g = gen(M * K)
    a, sa, w, sw = integers(g, M, K), scales(g, M), integers(g, N, K), scales(g, N)
    off = torch.empty(M, K + 37, dtype=torch.int8, device=DEV)[:, 3:3 + K]
    off.copy_(a)
    bias, w2, sw2 = normal(g, N), integers(g, 2 * 132, K), scales(g, 2 * 132) * 0.1
    for dtype in (torch.float32, torch.bfloat16):
        old = normal(g, M, N, dtype=dtype)
        got = []
        for k, rows in (((1, 0), a), ((5, 0), a), ((5, 0), off)):
            ops.linear_int8_kernel(*k)
            try:
                outs = [torch.full((M, N), float("nan"), dtype=dtype, device=DEV), old.clone(), torch.full((M, 132), float("nan"), dtype=dtype, device=DEV)]
                ops.linear_int8(rows, w, sw, outs[0], a_scale=sa, colbias=bias)
                ops.linear_int8(rows, w, sw, outs[1], a_scale=sa, accumulate=True)
                ops.linear_swiglu_int8(rows, w2, sw2, outs[2], a_scale=sa)
                got.append(outs)
            finally:
                ops.linear_int8_kernel()
        for other in got[1:]:
            assert all(torch.equal(x, y) for x, y in zip(got[0], other))
    ops.check_errors()


@pytest.mark.parametrize("N,K", [(2048, 2048), (8240, 2048), (4738, 2041), (2368, 4096), (2369, 4096), (2048, 2064), (40, 8192), (9472, 2048), (9480, 100)])
def test_one_row_rounded_within_gives_the_same_bits(N, K):
    """One row in 16 or 32 bits, rounded where it is multiplied, at both sides of the rules that say how many weight rows a warp takes."""
    g = gen(N + K)
    w, sw, bias = integers(g, N, K), scales(g, N), normal(g, N)
    for xt, dtype in ((torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)):
        x = normal(g, 1, K, dtype=xt)
        got = []
        for k in ((1, 0), (4, 0)):
            ops.linear_int8_kernel(*k)
            try:
                outs = [torch.full((1, N), float("nan"), dtype=dtype, device=DEV), torch.ones(1, N, dtype=dtype, device=DEV)]
                ops.linear_int8(x, w, sw, outs[0], colbias=bias)
                ops.linear_int8(x, w, sw, outs[1], accumulate=True)
                if N % 2 == 0:
                    outs.append(torch.full((1, N // 2), float("nan"), dtype=dtype, device=DEV))
                    ops.linear_swiglu_int8(x, w, sw * 0.1, outs[2])
                got.append(outs)
            finally:
                ops.linear_int8_kernel()
        assert all(torch.equal(x, y) for x, y in zip(*got))
    ops.check_errors()


@pytest.mark.parametrize("M,N,K", [(9, 100, 4096), (16, 2050, 2048), (13, 77, 1001), (15, 2048, 333), (12, 17, 16), (16, 8, 4081)])
def test_up_to_sixteen_rows_give_the_same_bits(M, N, K):
    test_few_rows_give_the_same_bits(M, N, K)


@pytest.mark.parametrize("N,K", [(2048, 2048), (8240, 2048), (4738, 2041), (9480, 100), (33, 17), (8, 2049)])
def test_two_rows_rounded_within_give_the_same_bits(N, K):
    """Two rows in 16 or 32 bits, on 16-byte boundaries and off them, one with a NaN, rounded where they are multiplied."""
    g = gen(N + 2 * K)
    w, sw, bias = integers(g, N, K), scales(g, N), normal(g, N)
    for xt, dtype, first in ((torch.bfloat16, torch.float32, 0), (torch.float32, torch.bfloat16, 0), (torch.bfloat16, torch.bfloat16, 3)):
        x = normal(g, 2, K + 5, dtype=xt)[:, first:first + K]
        if first:
            x[1, K // 2] = float("nan")
        got = []
        for k in ((1, 0), (4, 0)):
            ops.linear_int8_kernel(*k)
            try:
                outs = [torch.full((2, N), 3.0, dtype=dtype, device=DEV), torch.ones(2, N, dtype=dtype, device=DEV)]
                ops.linear_int8(x, w, sw, outs[0], colbias=bias)
                ops.linear_int8(x, w, sw, outs[1], accumulate=True)
                if N % 2 == 0:
                    outs.append(torch.full((2, N // 2), 3.0, dtype=dtype, device=DEV))
                    ops.linear_swiglu_int8(x, w, sw * 0.1, outs[2])
                got.append(outs)
            finally:
                ops.linear_int8_kernel()
        assert all(torch.equal(a.nan_to_num(7e30), b.nan_to_num(7e30)) for a, b in zip(*got))
        assert not first or bool(got[0][0][1].isnan().all())
    ops.check_errors()
