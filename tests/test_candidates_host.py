"""What the operators for several candidates of a request refuse, and the plain forms that their tests compare with (no GPU)."""
import random

import pytest
import torch

from tinyllama_c_b200 import ops

import candidates_plain as plain

I = torch.int32


def ints(*shape):
    return torch.zeros(shape, dtype=I)


def resize(**kw):
    a = dict(block_table=ints(3, 4), refs=ints(9), lengths=ints(3), slots=ints(2), want=ints(2), status=ints(1))
    a.update(kw)
    ops.page_resize(**a)


def maps(**kw):
    a = dict(block_table=ints(3, 4), slots=ints(2), start=ints(2), new=ints(2), n_rows=5)
    a.update(kw)
    ops.row_maps(**a)


def store(**kw):
    a = dict(k=torch.zeros(5, 16), v=torch.zeros(5, 16), row_map=ints(5), k_pages=torch.zeros(3, 2, 64, 8), v_pages=torch.zeros(3, 2, 64, 8))
    a.update(kw)
    ops.kv_store(**a)


def attend(**kw):
    a = dict(q=torch.zeros(5, 32), k_new=torch.zeros(5, 16), v_new=torch.zeros(5, 16), k_pages=torch.zeros(3, 2, 64, 8), v_pages=torch.zeros(3, 2, 64, 8),
             block_table=ints(3, 4), slots=ints(2), start=ints(2), cu_seqlens=ints(3), positions=ints(5), out=torch.zeros(5, 32), H=4, KV=2, hd=8,
             scale=1.0, max_context=64, max_new=5, mask=ints(5, 1))
    a.update(kw)
    ops.tree_attention(**a)


def select(**kw):
    a = dict(logits=torch.zeros(6, 50), scores=torch.zeros(2, 3), n=4)
    a.update(kw)
    ops.beam_select(**a)


def states(**kw):
    a = dict(state=torch.zeros(2, 7, 4, 5), slots=ints(2, 3), parents=ints(2, 3))
    a.update(kw)
    ops.beam_reorder_states(**a)


def pages(**kw):
    a = dict(block_table=ints(3, 4), refs=ints(9), lengths=ints(3), slots=ints(1, 3), parents=ints(1, 3), k_pages=torch.zeros(9, 2, 64, 8),
             v_pages=torch.zeros(9, 2, 64, 8), status=ints(1))
    a.update(kw)
    ops.beam_reorder_pages(**a)


REFUSED = [
    (resize, dict(block_table=ints(12))), (resize, dict(block_table=ints(4, 3).t())), (resize, dict(block_table=torch.zeros(3, 4))), (resize, dict(block_table=ints(3, 0))),
    (resize, dict(refs=ints(3, 3))), (resize, dict(refs=ints(18)[::2])), (resize, dict(refs=ints(0))), (resize, dict(lengths=ints(4))),
    (resize, dict(lengths=torch.zeros(3, dtype=torch.int64))), (resize, dict(want=ints(3))), (resize, dict(want=torch.zeros(2))), (resize, dict(status=ints(0))),
    (resize, dict(slots=ints(8193), want=ints(8193))),
    (maps, dict(start=ints(3))), (maps, dict(new=ints(1))), (maps, dict(n_rows=-1)), (maps, dict(parents=ints(4), max_new=3)), (maps, dict(parents=ints(5))),
    (maps, dict(keep=ints(5))), (maps, dict(keep=torch.zeros(4, dtype=torch.bool))), (maps, dict(slots=ints(8193), start=ints(8193), new=ints(8193))),
    (store, dict(v=None)), (store, dict(v_pages=None)), (store, dict(k=torch.zeros(5, 15), v=torch.zeros(5, 15))), (store, dict(row_map=ints(4))),
    (store, dict(v=torch.zeros(5, 16).bfloat16())), (store, dict(k=torch.zeros(16, 5).t(), v=torch.zeros(16, 5).t())), (store, dict(k=torch.zeros(1, 5, 16), v=torch.zeros(1, 5, 16))),
    (store, dict(k_pages=torch.zeros(3, 2, 32, 8), v_pages=torch.zeros(3, 2, 32, 8))), (store, dict(v_pages=torch.zeros(3, 2, 64, 8).bfloat16())),
    (store, dict(v=torch.zeros(4, 16))),
    (attend, dict(H=3)), (attend, dict(hd=257)), (attend, dict(KV=0)), (attend, dict(q=torch.zeros(5, 31))), (attend, dict(k_new=torch.zeros(4, 16))),
    (attend, dict(out=torch.zeros(5, 32).bfloat16())), (attend, dict(out=torch.zeros(4, 32))), (attend, dict(v_pages=torch.zeros(2, 2, 64, 8))),
    (attend, dict(k_pages=torch.zeros(3, 64, 2, 8).transpose(1, 2))), (attend, dict(start=ints(3))), (attend, dict(cu_seqlens=ints(2))), (attend, dict(positions=ints(4))),
    (attend, dict(mask=ints(5))), (attend, dict(mask=ints(4, 1))), (attend, dict(mask=ints(5, 1), max_new=33)), (attend, dict(mask=ints(5, 2)[:, :1])),
    (attend, dict(sink_values=torch.zeros(3))), (attend, dict(window=-1)), (attend, dict(softcap=-1.0)), (attend, dict(softcap=1.0, scale=0.0)), (attend, dict(max_context=-1)),
    (attend, dict(q=torch.zeros(32, 5).t())),
    (select, dict(n=0)), (select, dict(n=65)), (select, dict(n=4, placed=True)), (select, dict(logits=torch.zeros(5, 50))), (select, dict(logits=torch.zeros(6, 50).bfloat16())),
    (select, dict(scores=torch.zeros(2, 3, dtype=torch.float64))), (select, dict(pad=50)), (select, dict(pad=-1)), (select, dict(ended=torch.zeros(2, 3))),
    (select, dict(ended=torch.zeros(2, 2, dtype=torch.bool))), (select, dict(logits=torch.zeros(6, 1))), (select, dict(logits=torch.zeros(65, 9), scores=torch.zeros(1, 65))),
    (states, dict(parents=ints(3, 2))), (states, dict(slots=ints(6), parents=ints(6))), (states, dict(state=torch.zeros(7))), (states, dict(state=torch.zeros(2, 7, 5, 4).transpose(2, 3))),
    (states, dict(state=torch.zeros(7, 2, 4, 5).expand(7, 2, 4, 5)[:, :1].expand(7, 3, 4, 5))), (states, dict(slots=ints(1, 65), parents=ints(1, 65))),
    (states, dict(slots=torch.zeros(2, 3), parents=torch.zeros(2, 3))),
    (pages, dict(refs=ints(8))), (pages, dict(v_pages=torch.zeros(9, 2, 64, 8).bfloat16())), (pages, dict(k_pages=torch.zeros(9, 2, 64, 4))), (pages, dict(lengths=ints(2))),
    (pages, dict(slots=ints(1, 2))), (pages, dict(k_pages=torch.zeros(2, 9, 64, 8), v_pages=None)),
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_refused(i):
    call, change = REFUSED[i]
    with pytest.raises(ops.KernelError) as e:
        call(**change)
    assert "CUDA device" not in str(e.value)             # refused for what is wrong with it, not for where it runs


@pytest.mark.parametrize("call", [resize, maps, store, attend, select, states, pages])
def test_there_is_no_cpu_path(call):
    with pytest.raises(ops.KernelError, match="CUDA device"):
        call()


def test_plain_pool_loses_no_page():
    rng = random.Random(0)
    pool = plain.Pool(6, 5, 22)
    for _ in range(300):
        if rng.random() < 0.6:
            slots = rng.sample(range(6), rng.randint(1, 6))
            pool.resize(slots, [rng.randint(0, 5 * 64) for _ in slots])
        else:
            pool.reorder(rng.sample(range(6), 4), [rng.randrange(4) for _ in range(4)])
        counts = [0] * 22
        for row, n in zip(pool.table, pool.lengths):
            for page in row[:plain.pages_of(n)]:
                counts[page] += 1
        assert counts == pool.refs


def test_plain_masks_and_positions():
    cu, seq, pos, place, mask = plain.row_maps([[5, 9]], [0], [62], [4], 5, [-1, 0, 0, 2], [True, False, True, True, False], 1)
    assert (cu, seq, pos) == ([0, 4], [0, 0, 0, 0, -1], [62, 63, 63, 64, 0])
    assert place == [5 * 64 + 62, -1, 5 * 64 + 63, 9 * 64, -1]
    assert mask == [[1], [3], [5], [13], [0]]
