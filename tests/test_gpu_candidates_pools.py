"""The pool's operators by what they leave behind: what a beam's table row reads after a reordering, whose pages a step writes."""
import random

import pytest
import torch

from tinyllama_c_b200 import ops

import candidates_plain as plain
from test_gpu_candidates import DEV, PAGE, DevicePool, ints

pytestmark = pytest.mark.gpu


def histories(dev, slots, pages):
    """What each slot's row reads: [L, KV, length, hd] of pages [L, n, KV, 64, hd]."""
    out = []
    for s in slots:
        n = int(dev.lengths[s])
        row = dev.table[s, :plain.pages_of(n)].long()
        out.append(pages[:, row].transpose(1, 2).flatten(2, 3)[:, :, :n].clone())
    return out


def reordered(dev, slots, parents, pages):
    """One call of all requests; its code.  With code 0 every beam reads what its parent read, else what it read before; the counts are those of the table."""
    before = [[histories(dev, row, p) for row in slots] for p in pages]
    ops.beam_reorder_pages(dev.table, dev.refs, dev.lengths, ints(slots), ints(parents), pages[0], pages[1], dev.status)
    code = int(dev.status)
    dev.status.zero_()
    for p, old in zip(pages, before):
        for r, row in enumerate(slots):
            now = histories(dev, row, p)
            same = [all(torch.equal(a, b) for a, b in zip(now, want)) for want in ([old[r][k] for k in parents[r]], old[r])]
            assert same[0] or (code and same[1]), (r, code)
    counts = torch.zeros_like(dev.refs)
    for s, n in enumerate(dev.lengths.tolist()):
        row = dev.table[s, :plain.pages_of(n)].long()
        counts.index_add_(0, row, torch.ones_like(row, dtype=torch.int32))
    assert torch.equal(counts, dev.refs)
    return code


@pytest.mark.parametrize("lengths,parents", [([64, 100], [1, 0]), ([100, 64], [1, 0]), ([64, 100, 100], [1, 0, 2]), ([128, 70, 64], [1, 2, 0]), ([64, 64, 100], [2, 0, 2]),
                                             ([64, 128, 100, 5], [2, 0, 1, 1]), ([64, 64, 64, 90], [3, 0, 0, 1]), ([128, 128, 70, 71], [2, 3, 0, 1])])
def test_whole_last_pages_that_a_child_takes_over(lengths, parents):
    K = len(lengths)
    pool = plain.Pool(2 * K, 4, 8 * K)
    slots = [list(range(K)), list(range(K, 2 * K))[::-1]]
    for row in slots:
        assert pool.resize(row, lengths) == 0
    dev = DevicePool(pool)
    pages = [torch.randint(0, 250, (2, 8 * K, 2, PAGE, 9), device=DEV).bfloat16() for _ in range(2)]
    assert reordered(dev, slots, [parents, list(range(K))], pages) == 0
    for row, up in zip(slots, [parents, list(range(K))]):
        assert pool.reorder(row, up)[0] == 0
    dev.equals(pool)
    # every beam may go on
    dev.resize([s for row in slots for s in row], [n + 1 for row in slots for n in dev.lengths[ints(row).long()].tolist()])
    assert dev.status.tolist() == [0]


@pytest.mark.parametrize("K,hd,dtype", [(2, 128, torch.bfloat16), (4, 5, torch.float32), (7, 16, torch.bfloat16), (20, 7, torch.bfloat16)])
def test_histories_of_random_lengths(K, hd, dtype):
    rng, R, codes = random.Random(K), 3, []
    for _ in range(8):
        n_slots = R * K + 1
        pool = plain.Pool(n_slots, 5, 5 * n_slots)
        taken = rng.sample(range(n_slots), R * K)
        slots = [taken[r * K:(r + 1) * K] for r in range(R)]
        assert pool.resize(taken, [rng.choice([64, 128, 320, rng.randint(1, 320)]) for _ in taken]) == 0
        dev = DevicePool(pool)
        pages = [torch.randint(0, 250, (1, 5 * n_slots, 2, PAGE, hd), device=DEV).to(dtype) for _ in range(2)]
        for _ in range(3):
            parents = [[rng.randrange(K) for _ in range(K)] for _ in range(R)]
            want = max(pool.reorder(row, up)[0] for row, up in zip(slots, parents))
            codes.append(reordered(dev, slots, parents, pages))
            assert codes[-1] == want
            dev.equals(pool)
    assert 0 in codes


def test_no_page_to_spare():
    """The only page that the beams give back is another slot's too: refused, nothing changes."""
    pool = plain.Pool(4, 4, 16)
    assert pool.resize([0, 1, 2], [64, 64, 100]) == 0
    pool.table[3], pool.lengths[3] = list(pool.table[1]), 64
    pool.refs[pool.table[1][0]] = 2
    dev = DevicePool(pool)
    pages = [torch.randn(1, 16, 1, PAGE, 8, device=DEV) for _ in range(2)]
    before = [p.clone() for p in pages]
    assert reordered(dev, [[0, 1, 2]], [[2, 0, 2]], pages) == 5
    dev.equals(pool)
    assert all(torch.equal(a, b) for a, b in zip(before, pages))


def test_requests_that_share_whole_pages():
    """Two requests over one whole prompt page, whose beams give it back and take it over at once: nobody fills it."""
    pool = plain.Pool(6, 4, 24)
    assert pool.resize([0, 2, 3, 5], [64, 100, 64, 100]) == 0
    for s in (1, 4):
        assert pool.resize([s], [64]) == 0
    prompt = pool.table[1][0]
    for s in (3, 4):                                                     # slots 1, 3 and 4 name one page
        pool.refs[pool.table[s][0]] = 0
        pool.table[s][0] = prompt
    pool.refs[prompt] = 3
    dev = DevicePool(pool)
    pages = [torch.randn(2, 24, 1, PAGE, 8, device=DEV) for _ in range(2)]
    # request 0: beam 0 fills a page that its child, beam 1, takes over, and beam 1's page is the prompt's; request 1 moves the prompt's page about
    assert reordered(dev, [[0, 1, 2], [3, 4, 5]], [[2, 0, 2], [1, 0, 2]], pages) == 5
    assert int(dev.refs[prompt]) == 3


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 63, 2 ** 31 - 64, 4 * 64 + 1, -1, -2 ** 31])
def test_lengths_that_no_row_can_hold(length):
    """The largest numbers too (63 more than they are is beyond 32 bits): code 2, the request stays as it is."""
    pool = plain.Pool(4, 4, 16)
    assert pool.resize([0, 1, 2, 3], [100, 100, 70, 70]) == 0
    for parents in ([1, 0], [1, 1], [0, 0]):
        mine = pool.copy()
        mine.lengths[0] = length
        dev = DevicePool(mine)
        pages = torch.randn(16, 1, PAGE, 8, device=DEV)
        before = pages.clone()
        ops.beam_reorder_pages(dev.table, dev.refs, dev.lengths, ints([[0, 1], [2, 3]]), ints([parents, [0, 1]]), pages, None, dev.status)
        dev.equals(mine)
        assert dev.status.tolist() == [2] and torch.equal(pages, before)


@pytest.mark.parametrize("bad", [5, 2 ** 25 - 2])
def test_entries_of_the_longest_rows(bad):
    """64 beams, two of them with 2^25 pages each: an entry that names no page is found wherever it is."""
    n = 2 ** 31 - 1
    table = torch.zeros(2, 2 ** 25, dtype=torch.int32, device=DEV)
    table[0, -1], table[1, -1], table[1, bad] = 1, 2, 3
    refs, lengths, status = ints([2 ** 26 - 3, 1, 1]), ints([n, n]), ints([0])
    before = table.clone()
    pages = torch.zeros(3, 1, PAGE, 1, dtype=torch.bfloat16, device=DEV)
    ops.beam_reorder_pages(table, refs, lengths, ints([[0, 1] + [-1] * 62]), ints([[1] + list(range(1, 64))]), pages, None, status)
    assert status.tolist() == [4] and torch.equal(table, before) and refs.tolist() == [2 ** 26 - 3, 1, 1] and lengths.tolist() == [n, n]


# ---- whose pages a step writes ------------------------------------------------------------------------------------
def step(dev, slots, start, new, pages):
    """Room for a step's rows, their places, their values stored; the places."""
    dev.resize(slots, [a + n for a, n in zip(start, new)])
    T = sum(new)
    rows = torch.randn(T, pages.shape[1] * pages.shape[3], device=DEV)
    maps = ops.row_maps(dev.table, ints(slots), ints(start), ints(new), T, lengths=dev.lengths)
    ops.kv_store(rows, rows, maps.row_map, pages, pages.clone())
    return maps.row_map.tolist()


def test_a_refused_step_stores_nothing():
    """The pool is full (1), or a request would grow in a page that it shares (5): no row beyond what the slots hold has a place."""
    pool = plain.Pool(3, 4, 4)
    assert pool.resize([0, 1, 2], [62, 100, 20]) == 0                    # four pages of four
    pages = torch.randn(4, 2, PAGE, 8, device=DEV)
    before, dev = pages.clone(), DevicePool(pool)
    assert step(dev, [0, 1], [62, 100], [4, 1], pages) == [-1] * 5
    assert dev.status.tolist() == [1] and torch.equal(pages, before)
    dev.equals(pool)
    assert step(dev, [0, 1], [62, 100], [2, 1], pages) == [pool.table[0][0] * 64 + 62, pool.table[0][0] * 64 + 63, pool.table[1][1] * 64 + 36]
    pool = plain.Pool(3, 4, 9)
    assert pool.resize([0, 2], [100, 64]) == 0
    pool.table[1], pool.lengths[1] = list(pool.table[0]), 100            # both pages shared
    for p in pool.table[0][:2]:
        pool.refs[p] = 2
    pages = torch.randn(9, 2, PAGE, 8, device=DEV)
    before, dev = pages.clone(), DevicePool(pool)
    assert step(dev, [1, 2], [100, 64], [1, 3], pages) == [-1] * 4
    assert dev.status.tolist() == [5] and torch.equal(pages, before)
    # rows that the slot does hold have places all the same, whatever has become of the step
    maps = ops.row_maps(dev.table, ints([1, -1, 0]), ints([98, 0, 99]), ints([4, 1, 2]), 7, lengths=dev.lengths)
    last = pool.table[0][1] * 64
    assert maps.row_map.tolist() == [last + 34, last + 35, -1, -1, -1, last + 35, -1]
    assert maps.positions.tolist() == [98, 99, 100, 101, 0, 99, 100]


@pytest.mark.parametrize("seed", range(6))
def test_places_of_what_slots_hold(seed):
    """Random lengths, slots and drafts: the plain form's places, but for positions that the slot does not hold."""
    rng = random.Random(seed)
    B, width = rng.randint(1, 40), rng.randint(1, 6)
    pool = plain.Pool(B + 2, width, (B + 2) * width)
    assert pool.resize(list(range(B + 2)), [rng.randint(0, width * PAGE) for _ in range(B + 2)]) == 0
    slots = [rng.choice([-1, rng.randrange(B + 2), B + 2]) if rng.random() < 0.2 else s for s in rng.sample(range(B + 2), B)]
    start = [rng.randint(0, width * PAGE) if not 0 <= s < B + 2 or rng.random() < 0.3 else max(0, pool.lengths[s] - rng.randint(0, 9)) for s in slots]
    new = [rng.randint(0, 20) for _ in slots]
    T = sum(new) + 2
    dev = DevicePool(pool)
    for drafts in (False, True):
        parents = [p for n in new for p in plain.draft(rng, n)] + [-1, -1] if drafts else None
        keep = [rng.random() < 0.6 for _ in range(T)] if drafts or seed % 2 else None
        got = ops.row_maps(dev.table, ints(slots), ints(start), ints(new), T, ints(parents) if drafts else None,
                           None if keep is None else torch.tensor(keep, device=DEV), 20, lengths=dev.lengths)
        cu, seq, pos, place, mask = plain.row_maps(pool.table, slots, start, new, T, parents, keep, 1)
        place = [-1 if b < 0 or p < 0 or at >= pool.lengths[slots[b]] else p for b, p, at in zip(seq, place, pos)]
        assert (got.cu_seqlens.tolist(), got.row_seq.tolist(), got.positions.tolist(), got.row_map.tolist()) == (cu, seq, pos, place)
        assert not drafts or got.mask.tolist() == mask


def test_room_comes_before_places():
    """Accepted rows that cross into a new page: after page_resize they have places there; asked before it they have none, and are not stored into page 0."""
    pool = plain.Pool(2, 3, 6)
    assert pool.resize([1, 0], [64, 62]) == 0                            # page 0 is slot 1's
    parents, keep, slots, start, new = ints([-1, 0, 1, 2]), torch.tensor([True] * 4, device=DEV), ints([0]), ints([62]), ints([4])
    rows = torch.randn(4, 2 * 8, device=DEV)
    for early in (False, True):
        dev, pages = DevicePool(pool), torch.zeros(6, 2, PAGE, 8, device=DEV)
        if not early:
            dev.resize([0], [66])
        maps = ops.row_maps(dev.table, slots, start, new, 4, parents, keep, 4, lengths=dev.lengths)
        if early:
            dev.resize([0], [66])
        ops.kv_store(rows, None, maps.row_map, pages, None)
        assert dev.status.tolist() == [0] and dev.table.tolist() == [[1, 2, 0], [0, 0, 0]]
        assert maps.row_map.tolist() == ([-1] * 4 if early else [64 + 62, 64 + 63, 128, 129])
        assert not bool(pages[0].any()) and bool(pages[1:].any()) != early
        assert maps.mask.tolist() == [[1], [3], [7], [15]] and maps.positions.tolist() == [62, 63, 64, 65]
