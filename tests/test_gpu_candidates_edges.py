"""Calls of the operators for several candidates at the ends of their ranges, against what the formulas say."""
import random

import pytest
import torch

from tinyllama_c_b200 import ops

import candidates_plain as plain
from test_gpu_candidates import DEV, HALF, PAGE, TYPES, U, DevicePool, attention_case, attention_check, attention_run, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.float32, 16)])
@pytest.mark.parametrize("context", [2 ** 31 - 1, 2 ** 31 - 64, 2 ** 30 + 5])
def test_tree_attention_longest_contexts(dtype, hd, context):
    """A context of up to 2^31 - 1 positions, every page of it the same one.  With queries of 0 every weight is 1: sums of whole numbers, exact in every
    block, and the result the mean of the page's values (what the last, partly filled page lacks is less than 2^-24 of it), off by the additions of the
    parts' sums (296 at most, of sums and of results) and its own rounding."""
    table = torch.zeros(1, 2 ** 25, dtype=torch.int32, device=DEV)
    k = torch.ones(1, 1, PAGE, hd, dtype=dtype, device=DEV)
    v = torch.randint(-4, 5, (1, 1, PAGE, hd), device=DEV).to(dtype)
    zero = torch.zeros(1, hd, dtype=dtype, device=DEV)
    out = torch.full((1, hd), 7.0, dtype=dtype, device=DEV)
    ops.tree_attention(zero, zero, zero, k, v, table, ints([0]), ints([context]), ints([0, 1]), ints([context]), out, 1, 1, hd, 0.5, max_context=2 ** 31 - 1, max_new=1)
    want = v[0, 0].double().mean(0)
    allow = (2 * 296 + 8) * U * v[0, 0].double().abs().mean(0) + (HALF if dtype == torch.bfloat16 else U) * want.abs() + 1e-30
    assert bool(((out[0].double() - want).abs() <= allow).all())
    # a window that only the last positions are in
    ops.tree_attention(zero, zero, zero, k, v, table, ints([0]), ints([context]), ints([0, 1]), ints([context]), out, 1, 1, hd, 0.5, max_context=2 ** 31 - 1, max_new=1,
                       window=PAGE + 1)
    at = torch.arange(context - PAGE, context, device=DEV) % PAGE
    want = v[0, 0][at].double().sum(0) / (PAGE + 1)
    assert bool(((out[0].double() - want).abs() <= 8 * U * v[0, 0].double().abs().sum(0) + (HALF if dtype == torch.bfloat16 else U) * want.abs() + 1e-30).all())
    ops.check_errors()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("scale", [0.0, -0.2, -1e-30, 1e-30, 1e-50])
@pytest.mark.parametrize("window,softcap,sink", [(0, 0.0, False), (50, 0.0, True), (0, 3.0, False)])
def test_tree_attention_scales(dtype, hd, scale, window, softcap, sink):
    """Scales that are not positive, and tiny ones: hidden keys stay hidden, the scores' order is what the scale makes it."""
    if softcap and scale == 0:
        pytest.skip("refused")
    c = dict(attention_case(dtype, [300, 0, 64, 129], [20, 9, 70, 1], 4, 2, hd, seed=21), scale=scale)
    values = torch.linspace(-1.0, 1.0, 4) if sink else None
    out = attention_run(c, window=window, softcap=softcap, sink_values=values.to(DEV) if sink else None)
    attention_check(c, out, window, softcap, values)
    ops.check_errors()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("softcap,scale", [(0.01, 1.0), (1024.0, 0.3), (1025.0, 0.3), (1e5, 0.3), (1e30, 0.1), (50.0, 1e-37), (1e4, -0.3), (1e-35, 0.3)])
def test_tree_attention_caps(dtype, hd, softcap, scale):
    """Caps far above and below the scores, and scales that a cap cannot be divided by in 32 bits."""
    c = dict(attention_case(dtype, [300, 0, 64, 129], [20, 9, 70, 1], 4, 2, hd, seed=22), scale=scale)
    attention_check(c, attention_run(c, softcap=softcap), 0, softcap)
    ops.check_errors()


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 24)])
@pytest.mark.parametrize("drafts", [True, False])
def test_tree_attention_more_rows_than_said(dtype, hd, drafts):
    """Requests of 70, 3 and 33 rows where 33 were announced: what is within is right, rows beyond stay as they were, and it is reported."""
    c = attention_case(dtype, [100, 5, 64], [70, 3, 33], 4, 2, hd, drafts=drafts, seed=31)
    full = attention_run(c)
    ops.check_errors()
    cut = attention_run(dict(c, new=[33, 3, 33], mask=c["mask"]))
    with pytest.raises(ops.KernelError, match="code 60"):
        torch.cuda.synchronize()
        ops.check_errors()
    ops.check_errors()                                                   # (said once)
    rows = torch.zeros(c["T"], dtype=torch.bool, device=DEV)
    for b, n in enumerate([33, 3, 33]):
        rows[c["cu"][b]:c["cu"][b] + n] = True
    assert bool((cut[~rows] == 3.0).all())
    # (the rows within see none beyond: their own results, which other shares may have added up in another order)
    assert float((cut[rows].float() - full[rows].float()).abs().max()) <= 4 * (HALF if dtype == torch.bfloat16 else 2000 * U) * float(c["v"][:c["cu"][-1]].float().abs().max().clamp(min=6.0))


def test_row_maps_of_more_rows_than_the_mask_has_bits():
    parents = [-1] + list(range(39))
    maps = ops.row_maps(ints([[0, 1], [2, 3]]), ints([0, 1]), ints([10, 20]), ints([40, 2]), 42, ints(parents + [-1, 0]), torch.ones(42, dtype=torch.bool, device=DEV), 32)
    assert maps.mask.shape == (42, 1) and maps.mask[32:40].tolist() == [[0]] * 8 and maps.row_map[32:40].tolist() == [-1] * 8
    assert maps.positions[32:40].tolist() == [10] * 8 and maps.positions[:32].tolist() == list(range(10, 42))
    assert [v & 0xFFFFFFFF for v in maps.mask[:32, 0].tolist()] == [(2 << i) - 1 for i in range(32)] and maps.row_map[:32].tolist() == list(range(10, 42))
    assert maps.row_map[40:].tolist() == [2 * 64 + 20, 2 * 64 + 21] and maps.mask[40:].tolist() == [[1], [3]]


@pytest.mark.parametrize("R,K,V,n", [(1, 4, 65536, 4), (5, 8, 130048, 3), (0, 2, 9, 2)])
def test_beam_select_results_keep_little_else(R, K, V, n):
    """Tokens and parents are kept for every step of a search: with them their own bytes and 16 KB at most."""
    got = ops.beam_select(torch.randn(R * K, V, device=DEV), torch.zeros(R, K, device=DEV), n)
    assert all(t.untyped_storage().nbytes() <= 12 * R * n + 12 + 16384 and t.shape == (R, n) for t in got)
