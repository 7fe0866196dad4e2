"""The plain form of reordering pages, by what a beam's table row reads after the move (no GPU)."""
import random

import pytest

import candidates_plain as plain

PAGE = 64


def histories(pool, slots, memory):
    """What each slot's row reads, position by position: memory [page][offset]."""
    return [[memory[pool.table[s][j // PAGE]][j % PAGE] for j in range(pool.lengths[s])] for s in slots]


def moved(pool, slots, parents, memory):
    """Reorders a pool and its memory; with code 0 every beam reads what its parent read, and nothing that is shared was written."""
    before = histories(pool, slots, memory)
    counts = lambda: [sum(p in row[:plain.pages_of(n)] for row, n in zip(pool.table, pool.lengths)) for p in range(len(pool.refs))]
    code, copies = pool.reorder(slots, parents)
    old = [list(page) for page in memory]
    for a, b, used in copies.values():
        memory[b][:used] = old[a][:used]
    after = histories(pool, slots, memory)
    assert after == ([before[p] for p in parents] if code == 0 else before)
    assert counts() == pool.refs and all(pool.refs[b] == 1 for _, b, _ in copies.values())
    return code


@pytest.mark.parametrize("lengths,parents", [([64, 100], [1, 0]), ([100, 64], [1, 0]), ([64, 100, 100], [1, 0, 2]), ([128, 70, 64], [1, 2, 0]), ([64, 64, 100], [2, 0, 2]),
                                             ([64, 128, 100, 5], [2, 0, 1, 1]), ([64, 64, 64, 90], [3, 0, 0, 1]), ([128, 128, 70, 71], [2, 3, 0, 1])])
def test_whole_last_pages_that_a_child_takes_over(lengths, parents):
    K = len(lengths)
    pool = plain.Pool(K, 4, 4 * K)
    assert pool.resize(list(range(K)), lengths) == 0
    memory = [[(p, i) for i in range(PAGE)] for p in range(4 * K)]
    assert moved(pool, list(range(K)), parents, memory) == 0


def test_histories_of_random_lengths():
    rng, codes = random.Random(2), []
    for _ in range(400):
        K = rng.randint(2, 5)
        pool = plain.Pool(K + 1, 4, 4 * K + 4)
        slots = rng.sample(range(K + 1), K)
        assert pool.resize(slots, [rng.choice([64, 128, 192, rng.randint(1, 256)]) for _ in slots]) == 0
        memory = [[(p, i) for i in range(PAGE)] for p in range(4 * K + 4)]
        for _ in range(3):
            codes.append(moved(pool, slots, [rng.randrange(K) for _ in slots], memory))
    assert codes.count(0) > len(codes) // 2 and set(codes) == {0, 5}


def test_no_page_to_spare():
    """The only page that the beams give back is another slot's too: refused, nothing changes."""
    pool = plain.Pool(4, 4, 16)
    assert pool.resize([0, 1, 2], [64, 64, 100]) == 0
    pool.table[3], pool.lengths[3] = list(pool.table[1]), 64
    pool.refs[pool.table[1][0]] = 2
    memory = [[(p, i) for i in range(PAGE)] for p in range(16)]
    before = pool.copy()
    assert moved(pool, [0, 1, 2], [2, 0, 2], memory) == 5
    assert pool.__dict__ == before.__dict__
