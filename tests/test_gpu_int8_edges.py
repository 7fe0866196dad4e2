"""Products in 8-bit integers where operands are at the edge of what they can be."""
import numpy as np
import pytest
import torch

from tinyllama_c_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _next_to_halves(exponent, K, seed):
    """Rows [64, K] (numpy float32) whose scales are 2^exponent to 2^(exponent + 1) and whose quotients by them lie next to a half; with
    them their scales and the integers nearest to the quotients, both by IEEE divisions."""
    r = np.random.RandomState(seed)
    largest = (np.float32(127) * np.ldexp(r.uniform(1.01, 1.99, (64, 1)).astype(np.float32), exponent)).astype(np.float32)
    s = (largest / np.float32(127)).astype(np.float32)
    half = r.randint(-126, 126, (64, K)) + 0.5
    x = (half * s.astype(np.float64)).astype(np.float32)
    up = np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(-np.inf)), x
    x = np.choose(r.randint(0, 3, x.shape), up).astype(np.float32)
    x[:, :1] = largest
    return x, s, np.rint((x / s).astype(np.float32)).astype(np.int8)


@pytest.mark.parametrize("K", [64, 2048, 77])
@pytest.mark.parametrize("exponent", [-126, -125, -122, -118, -103, -102, -101, -100, -99, -90, -30, 100, 119])
def test_integers_of_small_and_large_rows_are_those_of_the_quotients(exponent, K):
    """Down to the smallest scale that a row can have (2^-126): equal to the nearest integer of the IEEE quotient."""
    x, s, q = _next_to_halves(exponent, K, K)
    rows = torch.from_numpy(x).to(DEV)
    got, scale = ops.rows_int8(rows)
    assert np.array_equal(scale.cpu().numpy(), s[:, 0]) and np.array_equal(got.cpu().numpy(), q)
    if exponent < 0:                                     # (the sum of squares of larger rows is infinite)
        got, _ = ops.rmsnorm_int8(rows, torch.ones(K, device=DEV), 1e-5)
        assert np.array_equal(got.cpu().numpy(), q)
    # one row and two, rounded by the product itself: times the unit matrix and a power of two that brings them into range
    w = ops.int8_empty(K, K, DEV)
    w.copy_(torch.eye(K, dtype=torch.int8))
    power = 2.0 ** (-exponent if exponent < 0 else 0)
    for M in (1, 2):
        out = torch.empty(M, K, device=DEV)
        ops.linear_int8(rows[:M], w, torch.full((K,), power, device=DEV), out)
        want = (q[:M].astype(np.float32) * s[:M]) * np.float32(power)
        assert np.array_equal(out.cpu().numpy(), want)
    ops.check_errors()


def _operands(M, N, K, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = torch.empty(M, K, device=DEV).normal_(generator=g)
    return x, *ops.weight_int8(torch.empty(N, K, device=DEV).normal_(0.0, 0.1, generator=g)), g


def test_numbers_beyond_32_bits_are_infinities_as_in_the_16_bit_products():
    """A clamp that does nothing, given as a number that only 64 bits hold."""
    x, w, sw, g = _operands(5, 128, 64, 1)
    outs = []
    for limit in (1e300, float("inf"), 1e30):
        outs.append(torch.empty(5, 64, device=DEV))
        ops.linear_swiglu_int8(x, w, sw, outs[-1], act="swish_clamped", limit=limit, alpha=1.5)
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    logits = torch.empty(5, 2, device=DEV).normal_(generator=g)
    wd, sd = ops.weight_int8(torch.empty(2, 64, 64, device=DEV).normal_(generator=g))
    wgu, sgu = torch.stack([w, w]), torch.stack([sw, sw])
    outs = []
    for limit in (1e300, float("inf")):
        outs.append(torch.empty(5, 1, 64, device=DEV))
        ops.moe_experts_int8(x, wgu, sgu, wd, sd, ops.moe_route(logits, 2, 1), 1, outs[-1], act_fn="swish_clamped", limit=limit, alpha=1.5)
    assert torch.equal(*outs)
    weights = [ops.moe_route(logits, 2, 1, weights="softmax_all", sum_to=s)[1] for s in (1e300, float("inf"))]
    assert torch.equal(*weights) and bool(torch.isinf(weights[0]).all())
    ops.check_errors()


def test_rows_further_apart_than_32_bits_count_are_refused():
    """Strides of 2^32 + 64 elements, which as 32-bit numbers would be 64."""
    far = (1 << 32) + 64
    room = torch.zeros(far + 4096, dtype=torch.int8, device=DEV)
    a, sa = room.as_strided((2, 64), (far, 1)), torch.ones(2, device=DEV)
    x, w, sw, g = _operands(2, 128, 64, 2)
    out = torch.empty(2, 128, device=DEV)
    with pytest.raises(ops.KernelError):
        ops.linear_int8(a, w, sw, out, a_scale=sa)
    with pytest.raises(ops.KernelError):
        ops.linear_int8(x, a, sa, torch.empty(2, 2, device=DEV))
    with pytest.raises(ops.KernelError):
        ops.rows_int8(x, (a, sa))
    ops.linear_int8(x, w, sw, out)                       # and nothing is left of it
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("kernel", [(0, 0), (3, 128), (3, 256)])
def test_results_whose_rows_lie_far_apart(kernel):
    """Rows of the result 310,000,000 values apart: the sixteenth begins beyond 2^32."""
    M, N, K, far = 16, 64, 256, 310_000_000
    x, w, sw, g = _operands(M, N, K, 3)
    a, sa = ops.rows_int8(x)
    room = torch.empty((M - 1) * far + N, dtype=torch.bfloat16, device=DEV)
    for product, n in ((ops.linear_int8, N), (ops.linear_swiglu_int8, N // 2)):
        want = torch.empty(M, n, dtype=torch.bfloat16, device=DEV)
        product(a, w, sw, want, a_scale=sa)
        out = room.as_strided((M, n), (far, 1))
        out.fill_(float("nan"))
        ops.linear_int8_kernel(*kernel)
        try:
            product(a, w, sw, out, a_scale=sa)
            if product is ops.linear_int8:
                product(a, w, sw, out, a_scale=sa, accumulate=True)
                product(a, w, sw, want, a_scale=sa, accumulate=True)
        finally:
            ops.linear_int8_kernel()
        assert torch.equal(out, want)
    ops.check_errors()
