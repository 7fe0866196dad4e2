"""Routing of few rows (one launch up to 8 rows and 128 experts, else two) and of more choices than a warp has lanes, all weightings, against the
definition in 64 bits.

The weights' allowance, u = 2^-24: an exponential's argument is a difference of two logits of at most 6 each (12u), the exponential itself
2u, a sum of positive terms one u a term along a warp's tree or, of the chosen ones, one after the other (at most 70), quotient and
products 4u: below 100u."""
import numpy as np
import pytest
import torch

from tinyllama_c_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _inputs(T, n, seed):
    """Logits [T, n + 3] (three columns more than outputs) with no two of a row nearer than 1e-4, within -6..6, and a correction that keeps
    the corrected scores apart too."""
    r = np.random.RandomState(seed)
    z = np.stack([r.permutation(n) for _ in range(T)]) * (11.0 / max(n - 1, 1)) - 5.5 + r.uniform(0, 1e-3, (T, n))
    bias = r.uniform(-0.2, 0.2, n)
    return np.concatenate([z, np.full((T, 3), 50.0)], 1).astype(np.float32), bias.astype(np.float32)


def _route_64(z, top, weights, bias, sum_to):
    z = z.astype(np.float64)
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    score = p + bias.astype(np.float64) if weights == "softmax_all" and bias is not None else p if weights == "softmax_all" else z
    ids = np.argsort(-score, axis=1, kind="stable")[:, :top]
    ranked = np.take_along_axis(score, ids, 1)
    apart = top < 2 or np.diff(ranked, axis=1).max() < -1e-7                    # (nothing for 32 bits to decide)
    chosen = np.take_along_axis(z, ids, 1)
    if weights == "sigmoid":
        w = 1 / (1 + np.exp(-chosen))
    elif weights == "softmax":
        w = np.exp(chosen - chosen[:, :1])
        w /= w.sum(1, keepdims=True)
    else:
        w = np.take_along_axis(p, ids, 1)
        if sum_to:
            w = w / (w.sum(1, keepdims=True) + 1e-20) * sum_to
    return ids, w, apart


@pytest.mark.parametrize("T", [1, 3, 4, 5, 8, 9, 40])
@pytest.mark.parametrize("n,ident,top", [(1, 0, 1), (7, 0, 3), (8, 2, 5), (33, 0, 32), (64, 0, 33), (64, 5, 64), (100, 3, 70), (300, 0, 8)])
def test_choices_weights_and_lists(T, n, ident, top):
    z, bias = _inputs(T, n, 31 * n + top)
    logits, correction = torch.from_numpy(z).to(DEV), torch.from_numpy(bias).to(DEV)
    for weights, choice_bias, sum_to in (("sigmoid", None, 0.0), ("softmax", None, 0.0), ("softmax_all", None, 0.0), ("softmax_all", bias, 0.0),
                                         ("softmax_all", bias, 2.5)):
        want_ids, want_w, apart = _route_64(z[:, :n], top, weights, choice_bias, sum_to)
        for tile_rows in (32, 64):
            ids, wts, order, offsets, tile_off, rows = ops.moe_route(logits, n, top, tile_rows, weights, correction if choice_bias is not None else None,
                                                                     ident, sum_to)
            got, w, order, offsets, tile_off = (t.cpu().numpy() for t in (ids, wts, order, offsets, tile_off))
            assert rows == tile_rows and sorted(order.tolist()) == list(range(T * top)) and offsets[0] == tile_off[0] == 0
            got = got.reshape(T, top)
            if apart:
                assert (got == want_ids).all()
            else:                                          # near ties: distinct choices all the same
                assert all(len(set(row)) == top for row in got.tolist())
                want_w = None
            if want_w is not None:
                assert np.abs(w.reshape(T, top) / want_w - 1).max() <= 100 * U
            flat = got.reshape(-1)
            for e in range(n):
                mine = order[offsets[e]:offsets[e + 1]]
                assert (flat[mine] == e).all() and len(mine) == (flat == e).sum()
                assert tile_off[e + 1] - tile_off[e] == ((len(mine) + tile_rows - 1) // tile_rows if e < n - ident else 0)


@pytest.mark.parametrize("weights,sum_to", [("sigmoid", 0.0), ("softmax", 0.0), ("softmax_all", 0.0), ("softmax_all", 1.7)])
@pytest.mark.parametrize("n,top", [(7, 3), (64, 33), (256, 8)])
def test_one_launch_and_two_choose_and_weigh_alike(n, top, weights, sum_to):
    """Rows by themselves, five at a time and all together: the same bits."""
    g = torch.Generator(device=DEV)
    g.manual_seed(n)
    logits = torch.empty(20, n, device=DEV).normal_(0.0, 2.0, generator=g)
    logits[3] = logits[3].round()                          # ties: the lowest index first
    logits[4, 1:] = -float("inf")
    logits[5] = 0
    more = dict(weights=weights, sum_to=sum_to, choice_bias=torch.empty(n, device=DEV).uniform_(-0.1, 0.1, generator=g) if weights == "softmax_all" else None)
    ids, wts = ops.moe_route(logits, n, top, **more)[:2]
    for size in (1, 5):
        parts = [ops.moe_route(logits[i:i + size], n, top, **more)[:2] for i in range(0, 20, size)]
        assert torch.equal(torch.cat([p[0] for p in parts]), ids)
        assert torch.equal(torch.cat([p[1] for p in parts]).nan_to_num(9.0), wts.nan_to_num(9.0))
    if weights == "sigmoid":
        assert (ids.view(20, top)[5].cpu() == torch.arange(top)).all()


@pytest.mark.parametrize("T,n,launches", [(1, 32, 1), (8, 128, 1), (9, 32, 2), (4, 4096, 2), (8, 129, 2)])
def test_many_experts_are_chosen_from_in_a_launch_of_its_own(T, n, launches):
    """Beside the lists' shared memory the rows of many experts do not stay in the L1."""
    logits = torch.randn(T, n, device=DEV)
    before = ops.launch_count()
    ops.moe_route(logits, n, 2)
    assert ops.launch_count() - before == launches
