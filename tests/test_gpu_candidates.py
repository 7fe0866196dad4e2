"""The operators for several candidates of a request (drafted tokens, beams) over the paged cache, against plain forms: pools and maps
value by value, attention and search against 64 bits.

Allowances of tree_attention, u = 2^-24, b = 2^-8 (half a step of bfloat16, relative): a score is a sum of hd products in 32 bits, off by at most
(hd + 4) u S with S = scale * sum |q| |k| (its scale and a cap's tanh among the 4), which moves a weight p by twice that relative to itself (numerator and
denominator); an exponential of 32 bits is off by 2^-21 or less at arguments up to 100 (their own rounding, 100 u, and the unit's
4u), sums of `keys` terms, joined over blocks, by (keys + 64) u.  So |o - o_64| <= E * A + rounding of the output, A = sum p |v|,
E = 2 (hd + 4) u S + 2 (104 + keys + 64) u.  bfloat16 adds b |o| for the output, and where weights are rounded to 16 bits for the tensor
cores b A more.
Allowance of beam scores: rounding to 32 bits (u |score|) and what 32-bit exponentials of values that are not among a piece's largest
leave in a logarithm of a sum, 2^-21 at most (an exponential's 2^-22, sums of 16)."""
import random

import pytest
import torch

from tinyllama_c_b200 import ops

import candidates_plain as plain

pytestmark = pytest.mark.gpu
DEV, PAGE = "cuda", 64
U, HALF = 2.0 ** -24, 2.0 ** -8
TYPES = [torch.float32, torch.bfloat16]


def ints(x, **kw):
    return torch.tensor(x, dtype=torch.int32, device=DEV, **kw)


class DevicePool:
    def __init__(self, pool, shift=0):
        self.table, self.lengths, self.status = ints(pool.table), ints(pool.lengths), ints([0])
        self.refs = ints([7] * shift + pool.refs)[shift:]          # (off 16-byte boundaries with a shift)

    def resize(self, slots, want):
        ops.page_resize(self.table, self.refs, self.lengths, ints(slots), ints(want), self.status)

    def equals(self, pool):
        assert self.lengths.tolist() == pool.lengths
        assert self.refs.tolist() == pool.refs
        assert self.table.tolist() == pool.table


# ---- pages -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n_slots,max_pages,n_pages,shift", [(1, 1, 1, 0), (5, 7, 20, 1), (40, 9, 200, 0), (300, 30, 20011, 3)])
def test_page_resize_walk(n_slots, max_pages, n_pages, shift):
    rng = random.Random(n_slots)
    pool = plain.Pool(n_slots, max_pages, n_pages)
    for p in rng.sample(range(n_pages), n_pages // 3):
        pool.refs[p] = 1                                              # somebody else's
    dev, worst, codes = DevicePool(pool, shift), 0, set()
    for step in range(25):
        B = rng.randint(1, n_slots)
        slots = rng.sample(range(n_slots), B)
        want = [rng.choice([0, pool.lengths[s], min(max_pages * PAGE, pool.lengths[s] + rng.choice([1, 1, 3, 64, 500])),
                            rng.randint(0, max_pages * PAGE)]) for s in slots]
        if step % 5 == 3:
            slots[rng.randrange(B)] = -1
        if step % 7 == 6:
            want[rng.randrange(B)] = rng.choice([-1, max_pages * PAGE + 1])
        if step % 11 == 10:
            slots[rng.randrange(B)] = rng.choice([slots[0], n_slots, n_slots + 5])
        code = pool.resize(slots, want)
        codes.add(code)
        worst = max(worst, code)
        dev.resize(slots, want)
        dev.equals(pool)
        assert dev.status.tolist() == [worst]
        if step % 8 == 7:
            dev.status.zero_()
            worst = 0
    assert 0 in codes


def test_page_resize_all_or_nothing():
    pool = plain.Pool(4, 6, 8)
    dev = DevicePool(pool)
    for slots, want, code in [([0, 1], [200, 130], 0), ([0, 1, 2], [10, 300, 380], 1), ([2], [64 * 1], 0), ([2, 0, 3], [129, 0, 64], 0)]:
        assert pool.resize(slots, want) == code
        dev.resize(slots, want)
        dev.equals(pool)
        assert dev.status.tolist() == [code]
        dev.status.zero_()


def test_page_resize_shared_pages():
    pool = plain.Pool(3, 4, 9)
    assert pool.resize([0], [100]) == 0
    pool.table[1], pool.lengths[1] = list(pool.table[0]), 100                # both pages shared
    for p in pool.table[0][:2]:
        pool.refs[p] = 2
    dev = DevicePool(pool)
    for slots, want, code in [([1], [101], 5), ([0, 1], [101, 64], 0), ([1], [0], 0), ([0], [0], 0)]:
        assert pool.resize(slots, want) == code
        dev.resize(slots, want)
        dev.equals(pool)
        assert dev.status.tolist() == [code]
        dev.status.zero_()
    assert pool.refs == [0] * 9


def test_page_resize_that_cannot_be():
    """Entries and counts that no pool has: a code, no access outside."""
    for entry, refs in ((9, 1), (-1, 1), (2, 0)):
        table, lengths, status = ints([[entry, 0], [0, 0]]), ints([5, 0]), ints([0])
        counts = ints([1, 1, refs, 0])
        before = [t.clone() for t in (table, counts, lengths)]
        ops.page_resize(table, counts, lengths, ints([0]), ints([0]), status)
        ops.page_resize(table, counts, lengths, ints([0]), ints([6]), status)
        assert status.tolist() == [4]
        assert all(torch.equal(a, b) for a, b in zip(before, (table, counts, lengths)))


def test_page_resize_many_requests():
    B = ops.MAX_TABLE_REQUESTS
    pool = plain.Pool(B, 2, 2 * B + 5)
    dev = DevicePool(pool)
    want = [(s * 37) % 129 for s in range(B)]
    dev.resize(list(range(B)), want)
    at = 0
    for s, w in enumerate(want):                              # (the plain form looks for each page from the start: too slow here)
        for c in range(plain.pages_of(w)):
            pool.table[s][c], pool.refs[at] = at, 1
            at += 1
        pool.lengths[s] = w
    dev.equals(pool)
    with pytest.raises(ops.KernelError):
        ops.page_resize(dev.table, dev.refs, dev.lengths, ints([0] * (B + 1)), ints([0] * (B + 1)), dev.status)


@pytest.mark.parametrize("B,most,room,drafts,keep", [(1, 1, 0, False, False), (3, 5, 4, False, True), (7, 40, -11, True, True),
                                                     (5, 130, 9, True, False), (600, 3, 0, False, False), (33, 64, 70, True, True)])
def test_row_maps(B, most, room, drafts, keep):
    rng = random.Random(B * most)
    table = [[rng.randint(0, 5000) for _ in range(9)] for _ in range(B + 2)]
    slots = rng.sample(range(B + 2), B)
    start, new = [rng.randint(0, 8 * PAGE) for _ in range(B)], [rng.randint(0, most) for _ in range(B)]
    new[0] = most
    if B > 4:
        slots[2], new[2], new[3] = -1, 1, -4
    T = max(1, sum(max(0, n) for n in new) + room)
    parents = None
    if drafts:
        parents = []
        for n in new:
            parents += plain.draft(rng, max(0, n))
        parents = (parents + [0] * T)[:T]
        if B > 4:
            parents[most // 2], parents[most - 1] = -2, most          # no parents that could be
    kept = [rng.random() < 0.4 for _ in range(T)] if keep else None
    words = (most + 31) // 32 if drafts else 0
    got = ops.row_maps(ints(table), ints(slots), ints(start), ints(new), T, ints(parents) if drafts else None,
                       torch.tensor(kept, device=DEV) if keep else None, most if drafts else 0)
    cu, seq, pos, place, mask = plain.row_maps(table, slots, start, new, T, parents, kept, words)
    assert got.cu_seqlens.tolist() == cu
    assert got.row_seq.tolist() == seq
    assert got.positions.tolist() == pos
    assert got.row_map.tolist() == place
    if drafts:
        assert got.mask.tolist() == mask


def test_row_maps_of_nothing():
    got = ops.row_maps(ints([[3]]), ints([]), ints([]), ints([]), 2)
    assert (got.cu_seqlens.tolist(), got.row_seq.tolist(), got.row_map.tolist()) == ([0], [-1, -1], [-1, -1])
    got = ops.row_maps(ints([[3]]), ints([0]), ints([5]), ints([4]), 0)
    assert got.cu_seqlens.tolist() == [0, 0]
    got = ops.row_maps(ints([[3]]), ints([0]), ints([5]), ints([0]), 0, ints([]), torch.zeros(0, dtype=torch.bool, device=DEV), 40)
    assert got.cu_seqlens.tolist() == [0, 0] and got.mask.shape == (0, 2)


# ---- rows to their places -----------------------------------------------------------------------------
@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("dst", TYPES)
@pytest.mark.parametrize("L,T,KV,hd,pad,values", [(1, 1, 1, 1, 0, True), (3, 17, 2, 128, 16, True), (2, 40, 3, 7, 1, True), (1, 9, 2, 64, 4, False),
                                                  (0, 33, 5, 80, 0, True)])
def test_kv_store(src, dst, L, T, KV, hd, pad, values):
    g = torch.Generator(device=DEV).manual_seed(1)
    rng, n = random.Random(T), 3
    lead = (L,) if L else ()
    rows = [torch.randn(*lead, T, KV * hd + pad, device=DEV, generator=g).to(src)[..., :KV * hd] for _ in range(2)]
    pages = [torch.randn(*lead, n, KV, PAGE, hd, device=DEV, generator=g).to(dst) for _ in range(2)]
    place = rng.sample(range(n * PAGE), T)
    for t in range(0, T, 4):
        place[t] = rng.choice([-1, -7, n * PAGE, 2 ** 31 - 1])
    want = [p.clone() for p in pages]
    for t, at in enumerate(place):
        if 0 <= at < n * PAGE:
            for p, r in zip(want, rows):
                p[..., at // PAGE, :, at % PAGE, :] = r[..., t, :].reshape(*lead, KV, hd).to(dst)
    ops.kv_store(rows[0], rows[1] if values else None, ints(place), pages[0], pages[1] if values else None)
    assert torch.equal(pages[0], want[0])
    if values:
        assert torch.equal(pages[1], want[1])


# ---- attention ----------------------------------------------------------------------------------------
def attention_case(dtype, context, new, H, KV, hd, drafts=True, pad=0, seed=0, slots=None):
    """Inputs of a call, on pages in any order; the context's last page and the rows behind the last request hold NaN where no
    row may look."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    B, T = len(context), sum(new) + 3
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    n_pages = sum(plain.pages_of(c) for c in context) + 2
    order = rng.sample(range(n_pages), n_pages)
    width = max([plain.pages_of(c) for c in context] + [1]) + 1
    table = [[0] * width for _ in range(B + 1)]
    slots = slots or rng.sample(range(B + 1), B)
    for s, c in zip(slots, context):
        if s >= 0:
            table[s][:plain.pages_of(c)] = [order.pop() for _ in range(plain.pages_of(c))]
    q = torch.randn(T, H * hd + pad, generator=g).to(dtype)[:, :H * hd]
    rows = [torch.randn(T, KV * hd + pad, generator=g).to(dtype)[:, :KV * hd] for _ in range(2)]
    pages = [torch.randn(n_pages, KV, PAGE, hd, generator=g).to(dtype) for _ in range(2)]
    for r in rows + [q]:
        r[cu[-1]:] = float("nan")
    for p in pages:
        for s, c in zip(slots, context):
            if s >= 0 and c % PAGE:
                p[table[s][c // PAGE], :, c % PAGE:] = float("nan")
        for left in order:
            p[left] = float("nan")
    parents = [p for n in new for p in plain.draft(rng, n)] if drafts else None
    depth = []
    for b in range(B):
        here = []
        for i in range(new[b]):
            p = parents[cu[b] + i] if drafts else i - 1
            here.append(context[b] if p < 0 else here[p] + 1)
        depth += here
    words = (max(new + [1]) + 31) // 32
    mask = None
    if drafts:
        mask = ints(plain.row_maps([[0] * 1], [0] * B, context, new, T, parents + [-1] * 3, None, words)[4]).view(T, words)
    return dict(dtype=dtype, context=context, new=new, cu=cu, H=H, KV=KV, hd=hd, q=q, k=rows[0], v=rows[1], kp=pages[0], vp=pages[1], table=table,
                slots=slots, parents=parents, positions=depth + [0] * 3, mask=mask, T=T, scale=hd ** -0.5)


def attention_run(c, out=None, **kw):
    dev = lambda t, w: torch.cat([t.contiguous().to(DEV), torch.zeros(len(t), w, dtype=t.dtype, device=DEV)], 1)[:, :t.shape[1]] if w else t.contiguous().to(DEV)
    pad = kw.pop("row_pad", 0)
    if out is None:
        out = torch.full((c["T"], c["H"] * c["hd"]), 3.0, dtype=c["dtype"], device=DEV)
    ops.tree_attention(dev(c["q"], pad), dev(c["k"], pad), dev(c["v"], pad), c["kp"].to(DEV), c["vp"].to(DEV), ints(c["table"]), ints(c["slots"]),
                       ints(c["context"]), ints(c["cu"]), ints(c["positions"]), out, c["H"], c["KV"], c["hd"], c["scale"],
                       max_context=max(c["context"]), max_new=max(c["new"]), mask=c["mask"], **kw)
    return out


def attention_check(c, out, window=0, softcap=0.0, sink=None, cores=True):
    """cores: weights may have been rounded to 16 bits."""
    H, KV, hd, cu = c["H"], c["KV"], c["hd"], c["cu"]
    got = out.float().cpu().double().view(c["T"], H, hd)
    assert bool((got[cu[-1]:] == 3.0).all())                          # behind the last request: as it was
    sees = plain.tree_sees(cu, c["context"], c["positions"], c["parents"], [n if s >= 0 else 0 for n, s in zip(c["context"], c["slots"])], window, c["T"])
    for b, n in enumerate(c["new"]):
        if not n:
            continue
        rows, ctx = slice(cu[b], cu[b + 1]), c["context"][b] if c["slots"][b] >= 0 else 0
        at = [c["table"][c["slots"][b]][j // PAGE] * PAGE + j % PAGE for j in range(ctx)]
        k, v = (torch.cat([p.transpose(1, 2).reshape(-1, KV, hd)[at], r[rows].reshape(n, KV, hd)]) for p, r in ((c["kp"], c["k"]), (c["vp"], c["v"])))
        o, A, S = plain.tree_attention(c["q"][rows].reshape(n, H, hd), k, v, sees[b], c["scale"], softcap, sink)
        E = 2 * (hd + 4) * U * S[..., None] + 2 * (104 + len(k) + 64) * U
        allow = E * A + (HALF * o.abs() + (HALF * A if cores else 0.0) if c["dtype"] == torch.bfloat16 else U * o.abs()) + 1e-30
        bad = ~((got[rows] - o).abs() <= allow)
        assert not bool(bad.any()), (b, bad.nonzero()[0].tolist(), float(((got[rows] - o).abs() / allow).nan_to_num(1e9).max()))


SHAPES = [  # context, new, H, KV, hd
    ([0], [1], 1, 1, 64),
    ([5], [3], 4, 2, 128),
    ([64, 63, 65], [1, 2, 33], 8, 2, 128),
    ([0, 200, 1, 128], [17, 0, 64, 5], 10, 2, 128),
    ([300, 700], [65, 130], 6, 1, 64),
    ([130, 5], [9, 20], 3, 3, 64),
    ([1000, 40], [12, 7], 12, 2, 128),
    ([70], [4], 4, 4, 16),
    ([129, 64], [21, 3], 6, 3, 80),
    ([90, 33], [6, 40], 5, 1, 256),
    ([100], [5], 2, 1, 1),
    ([77], [30], 9, 3, 37),
    ([257], [3], 40, 1, 64),
    ([66], [2], 256, 1, 16),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_tree_attention(shape, dtype):
    c = attention_case(dtype, *shape)
    attention_check(c, attention_run(c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 24])
@pytest.mark.parametrize("window,softcap,sink", [(50, 0.0, None), (1, 0.0, "zero"), (130, 5.0, "values"), (0, 2.0, None), (0, 0.0, "values"), (64, 0.0, None)])
def test_tree_attention_windows_caps_sinks(dtype, hd, window, softcap, sink):
    c = attention_case(dtype, [300, 0, 64, 129], [20, 9, 70, 1], 4, 2, hd, seed=3)
    values = torch.linspace(-2.0, 3.0, 4) if sink == "values" else torch.zeros(4) if sink else None
    out = attention_run(c, window=window, softcap=softcap, sink=sink == "zero", sink_values=values.to(DEV) if sink == "values" else None)
    attention_check(c, out, window, softcap, values)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_tree_attention_strides_and_chains(dtype, pad):
    """Rows of wider buffers (on 16-byte boundaries and off them), no mask: each row sees the rows up to itself."""
    c = attention_case(dtype, [100, 7], [40, 66], 4, 2, 64, drafts=False, seed=5)
    wide = torch.full((c["T"], 4 * 64 + 16), 3.0, dtype=dtype, device=DEV)
    out = wide[:, 8:8 + 256]
    attention_run(c, out, row_pad=pad)
    attention_check(c, out)
    assert bool((wide[:, :8] == 3.0).all()) and bool((wide[:, 264:] == 3.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 40])
def test_tree_attention_rows_that_see_nothing(dtype, hd):
    c = attention_case(dtype, [0, 0, 70], [5, 40, 3], 4, 2, hd, seed=6, slots=[1, 0, -1])
    c["mask"][:] = 0
    for sink in (False, True):
        out = attention_run(c, sink=sink)
        assert bool((out[:c["cu"][-1]] == 0).all()) and bool((out[c["cu"][-1]:] == 3.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_tree_attention_bad_values_stay_where_they_are_seen(dtype, hd, bad):
    """A draft whose key or value is no number, and one in the context behind a window's edge: rows that do not see it are as without it, the
    others are not numbers (where a value is infinite: infinite in its column)."""
    window = 40
    c = attention_case(dtype, [100, 64], [30, 70], 4, 2, hd, seed=7)
    clean = attention_run(c, window=window)
    j, col = 11, 2
    c["v"][c["cu"][1] + j, hd + col] = bad                                # second request, second key/value head
    c["vp"][c["table"][c["slots"][0]][0], 0, 61, 5] = bad                # first request: position 61 is behind the edge of most rows
    got = attention_run(c, window=window)
    sees = plain.tree_sees(c["cu"], c["context"], c["positions"], c["parents"], c["context"], window, c["T"])
    same, T0 = torch.ones(c["T"], 4, hd, dtype=torch.bool), c["cu"][1]
    same[T0:c["cu"][2], 2:, col] = ~sees[1][:, c["context"][1] + j][:, None]
    same[:T0, :2, 5] = ~sees[0][:, 61][:, None]
    assert int(same.sum()) < same.numel()
    got, clean = got.float().cpu().view(same.shape), clean.float().cpu().view(same.shape)
    assert bool((got[same] == clean[same]).all())
    assert bool((got[~same] == bad).all() if bad == float("inf") else got[~same].isnan().all())
    c["k"][c["cu"][1] + j, hd + col] = float("nan")
    got = attention_run(c, window=window).float().cpu().view(same.shape)
    hit = sees[1][:, c["context"][1] + j]
    assert bool(got[T0:c["cu"][2], 2:][hit].isnan().all())
    assert bool((got[T0:c["cu"][2], 2:][~hit] == clean[T0:c["cu"][2], 2:][~hit]).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_attention_many_requests_and_long_chains(dtype):
    """More requests than the pieces are looked at for; rows that fill several tiles of keys and of queries."""
    B = 2100
    c = attention_case(dtype, [b % 70 for b in range(B)], [1 + b % 2 for b in range(B)], 2, 1, 64, seed=11)
    out = attention_run(c)
    full = attention_run(dict(c, slots=c["slots"], new=c["new"]))
    assert torch.equal(out, full)
    got = out.float().cpu().double().view(c["T"], 2, 64)
    for b in range(0, B, 97):
        rows, ctx = slice(c["cu"][b], c["cu"][b + 1]), c["context"][b]
        at = [c["table"][c["slots"][b]][j // PAGE] * PAGE + j % PAGE for j in range(ctx)]
        k, v = (torch.cat([p.transpose(1, 2).reshape(-1, 1, 64)[at], r[rows].reshape(-1, 1, 64)]) for p, r in ((c["kp"], c["k"]), (c["vp"], c["v"])))
        part = plain.tree_sees([0, c["new"][b]], [ctx], c["positions"][rows], c["parents"][rows], [ctx], 0, c["new"][b])[0]
        o, A, S = plain.tree_attention(c["q"][rows].reshape(-1, 2, 64), k, v, part, c["scale"])
        E = 2 * 68 * U * S[..., None] + 2 * (168 + len(k)) * U
        assert bool(((got[rows] - o).abs() <= E * A + (HALF * (o.abs() + A) if dtype == torch.bfloat16 else U * o.abs()) + 1e-30).all())
    c = attention_case(dtype, [70, 3], [300, 190], 4, 2, 64, drafts=False, seed=12)
    attention_check(c, attention_run(c))
    attention_check(c, attention_run(c, window=100), 100)


def test_offsets_beyond_32_bits():
    """A pool of 4.6 GB of keys and as many of values, the last pages in use: places, rows, attention and reordering at its far end."""
    n, KV, hd = 140000, 2, 128
    pages = [torch.empty(n, KV, PAGE, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    assert pages[0].numel() > 1 << 31
    pool = plain.Pool(2, 3, n)
    pool.refs = [1] * (n - 4) + [0] * 4                               # all but the last pages are somebody else's
    dev = DevicePool(pool)
    assert pool.resize([0, 1], [100, 100]) == 0
    dev.resize([0, 1], [100, 100])
    dev.equals(pool)
    g = torch.Generator(device=DEV).manual_seed(3)
    k, v = (torch.randn(200, KV * hd, device=DEV, generator=g).bfloat16() for _ in range(2))
    maps = ops.row_maps(dev.table, ints([0, 1]), ints([0, 0]), ints([100, 100]), 200)
    assert int(maps.row_map.min()) >= (n - 4) * PAGE
    ops.kv_store(k, v, maps.row_map, *pages)
    where = maps.row_map.long()
    assert torch.equal(pages[0][where // PAGE, :, where % PAGE].view(200, -1), k) and torch.equal(pages[1][where // PAGE, :, where % PAGE].view(200, -1), v)
    q = torch.randn(2, 4 * hd, device=DEV, generator=g).bfloat16()
    outs = [torch.empty_like(q) for _ in range(2)]
    wide = torch.empty(2, 4 * hd + 1, dtype=torch.bfloat16, device=DEV)[:, 1:]                  # off 16-byte boundaries: the other kernel
    wide.copy_(q)
    for o, x in zip(outs, (q, wide)):
        ops.tree_attention(x, k[:2], v[:2], *pages, dev.table, ints([0, 1]), ints([100, 100]), ints([0, 1, 2]), ints([100, 100]), o, 4, KV, hd, 0.088,
                           max_context=100, max_new=1, mask=ints([[0], [0]]))
    for r in range(2):
        K, V = (x[100 * r:100 * r + 100].view(100, KV, hd).cpu() for x in (k, v))
        o, A, S = plain.tree_attention(q[r:r + 1].view(1, 4, hd).cpu(), K, V, torch.ones(1, 100, dtype=torch.bool), 0.088)
        allow = (2 * (hd + 4) * U * S[..., None] + 2 * 268 * U) * A + HALF * (o.abs() + A)
        for out in outs:
            assert bool(((out[r].view(1, 4, hd).cpu().double() - o).abs() <= allow).all())
    ops.beam_reorder_pages(dev.table, dev.refs, dev.lengths, ints([[0, 1]]), ints([[0, 0]]), *pages, dev.status)
    pool.reorder([0, 1], [0, 0])
    dev.equals(pool)
    a, b = pool.table[0][1], pool.table[1][1]
    assert a != b and torch.equal(pages[0][a, :, :36], pages[0][b, :, :36]) and dev.status.tolist() == [0]


def test_calls_made_again_and_tensors_elsewhere(monkeypatch):
    """Calls noted and made again from the library's table; a call while another device is current is refused."""
    import numpy as np
    pool = plain.Pool(2, 2, 8)
    dev = DevicePool(pool)
    q = torch.randn(3, 64, device=DEV)
    pages = torch.zeros(8, 1, PAGE, 64, device=DEV)
    out, state, logits = torch.zeros(3, 64, device=DEV), torch.randn(1, 2, 5, device=DEV), torch.randn(2, 30, device=DEV)
    slots, length, three, beams, up, scores = ints([0]), ints([3]), ints([3]), ints([[0, 1]]), ints([[0, 0]]), torch.zeros(1, 2, device=DEV)
    zero, cu, pos, place = ints([0]), ints([0, 3]), ints([0, 1, 2]), ints([64, 65, 66])
    calls = [lambda: ops.page_resize(dev.table, dev.refs, dev.lengths, slots, length, dev.status), lambda: ops.row_maps(dev.table, slots, zero, three, 3),
             lambda: ops.kv_store(q, q, place, pages, pages), lambda: ops.beam_select(logits, scores, 2), lambda: ops.beam_reorder_states(state, beams, up),
             lambda: ops.tree_attention(q, q, q, pages, pages, dev.table, slots, zero, cu, pos, out, 1, 1, 64, 0.1, max_context=0, max_new=3),
             lambda: ops.beam_reorder_pages(dev.table, dev.refs, dev.lengths, beams, ints([[0, 1]]), pages, None, dev.status)]
    with ops.noting() as notes:
        for call in calls:
            call()
    assert notes.complete and len(notes.functions) == len(calls)
    first = out.clone()
    out.zero_()
    dev.lengths.zero_()
    dev.refs.zero_()
    ops.replay(np.array(notes.functions, dtype=np.int32), np.array(notes.words, dtype=np.uint64), 1)
    torch.cuda.synchronize()
    assert torch.equal(out, first) and dev.lengths.tolist() == [3, 0] and dev.refs.tolist() == [1] + [0] * 7 and dev.status.tolist() == [0]
    monkeypatch.setattr(ops, "_get_device", lambda: 1)
    for call in calls:
        with pytest.raises(ops.KernelError, match="current device"):
            call()


def test_tree_attention_repeats_itself_and_replays():
    c = attention_case(torch.bfloat16, [900, 64, 2000], [33, 5, 64], 8, 2, 128, seed=8)
    first = attention_run(c)
    assert torch.equal(first, attention_run(c))
    args = dict(q=c["q"].to(DEV), k=c["k"].to(DEV), v=c["v"].to(DEV), kp=c["kp"].to(DEV), vp=c["vp"].to(DEV), t=ints(c["table"]), s=ints(c["slots"]),
                c=ints(c["context"]), cu=ints(c["cu"]), p=ints(c["positions"]))
    outs = [torch.full_like(first, 3.0) for _ in range(2)]

    def call(out):
        ops.tree_attention(args["q"], args["k"], args["v"], args["kp"], args["vp"], args["t"], args["s"], args["c"], args["cu"], args["p"], out, 8, 2, 128,
                           c["scale"], max_context=4096, max_new=64, mask=c["mask"])

    call(outs[0])
    reference = outs[0].clone()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g, o in zip(graphs, outs):                            # two captured calls, replayed at once on two streams
        with torch.cuda.graph(g):
            call(o)
    for o in outs:
        o.fill_(3.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, reference) for o in outs)
    # other lengths in the same graph
    args["c"].copy_(ints([10, 0, 129]))
    graphs[0].replay()
    torch.cuda.synchronize()
    c["context"] = [10, 0, 129]
    base = [c["context"][b] for b in range(3) for _ in range(c["new"][b])]
    old = [[900, 64, 2000][b] for b in range(3) for _ in range(c["new"][b])]
    c["positions"] = [p - o + n for p, o, n in zip(c["positions"], old, base)] + [0] * 3
    attention_check(c, outs[0])
    ops.check_errors()


# ---- beam search ----------------------------------------------------------------------------------------
def select_check(logits, scores, n, **kw):
    got = ops.beam_select(logits, scores, n, **kw)
    host = {k: (v.cpu() if torch.is_tensor(v) else v) for k, v in kw.items()}
    tokens, parents, values = plain.beam_select(logits.cpu(), scores.cpu(), n, **host)
    assert got[1].tolist() == parents and got[0].tolist() == tokens
    s = got[2].cpu().double()
    assert bool((s == values)[~torch.isfinite(values)].all())
    err = (s - values).abs()[torch.isfinite(values)]
    assert bool((err <= U * values.abs()[torch.isfinite(values)] + 2.0 ** -21).all())


@pytest.mark.parametrize("R,K,V,n", [(1, 1, 1, 1), (1, 4, 300, 4), (3, 5, 1000, 10), (2, 2, 511, 64), (1, 3, 70001, 6), (40, 4, 9001, 8), (2, 64, 513, 64),
                                     (1, 8, 130048, 16), (20, 8, 65537, 16)])
def test_beam_select(R, K, V, n):
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = torch.randn(R * K, V, device=DEV, generator=g) * 3
    scores = -10 * torch.rand(R, K, device=DEV, generator=g)
    select_check(logits, scores, n)
    if V > 8:
        wide = torch.randn(R * K, V + 5, device=DEV, generator=g)
        select_check(wide[:, 3:3 + V], scores, n)
    ended = torch.rand(R, K, device=DEV, generator=g) < 0.4
    ended[:, 0] = False
    select_check(logits, scores, n, ended=ended, pad=V // 2)
    if n >= K:
        select_check(logits, scores, K, placed=True)
        select_check(logits, scores, K, placed=True, ended=ended)


@pytest.mark.parametrize("V", [40, 700, 5000])
def test_beam_select_equal_values_and_infinities(V):
    inf = float("inf")
    same = torch.zeros(8, V, device=DEV)
    scores = torch.tensor([[-1.0, -1.0, -inf, -1.0], [-2.0, -inf, -inf, -inf]], device=DEV)
    select_check(same, scores, 4)
    select_check(same, scores, 8, ended=torch.tensor([[False, True, True, False]] * 2, device=DEV), pad=3)
    banned = torch.randn(8, V, device=DEV)
    banned[:, 3:] = -inf
    select_check(banned, scores, 8)
    banned[1] = -inf
    select_check(banned, scores, 20)
    steps = torch.zeros(8, V, device=DEV)
    steps[:, V // 2:] = 1.0
    select_check(steps, scores, 33)
    big = torch.randn(8, V, device=DEV)
    big[0, 5], big[3, 7], big[4, 0] = inf, float("nan"), -0.0
    select_check(big, scores, 6)
    select_check(big, torch.full((2, 4), -inf, device=DEV), 6)
    select_check(big, torch.tensor([[inf, float("nan"), -1.0, -2.0], [0.0, 0.0, 0.0, 0.0]], device=DEV), 6)
    select_check(torch.full((8, V), 60000.0, device=DEV) + torch.arange(V, device=DEV), scores, 5)


def test_beam_select_clustered_values():
    """All of the largest in one lane's reach."""
    logits = torch.randn(4, 8192, device=DEV)
    logits[0, 2048:2048 + 64] += 20
    logits[1, ::128] += 20
    logits[2, 100:4000] = 9.0
    select_check(logits, torch.zeros(1, 4, device=DEV), 64)
    select_check(logits, torch.zeros(4, 1, device=DEV), 64)


@pytest.mark.parametrize("R,K,V,n", [(16, 4, 30000, 16), (3, 2, 20001, 64), (24, 8, 9000, 16), (1, 1, 130048, 64), (2, 16, 65537, 32)])
def test_beam_select_of_few_alive_beams(R, K, V, n):
    """A first step (one beam is alive), beams of which only a few tokens are allowed, and values that rise from token to token."""
    g = torch.Generator(device=DEV).manual_seed(V + n)
    inf = float("inf")
    logits = torch.randn(R * K, V, device=DEV, generator=g) * 3
    first = torch.full((R, K), -inf, device=DEV)
    first[torch.arange(R), torch.arange(R) % K] = -0.5
    select_check(logits, first, n)
    zeros = torch.zeros(R, K, device=DEV)
    allowed = logits.clone()
    allowed[:, 5000:] = -inf
    select_check(allowed, first, n)
    lowest = logits.clone()
    lowest[:, 3:] = torch.finfo(torch.float32).min
    select_check(lowest, first, n)
    lowest[:, :3] = torch.finfo(torch.float32).min
    select_check(lowest, torch.arange(R * K, device=DEV).view(R, K) * -0.25, n)
    rising = (torch.arange(V, device=DEV) * 2.0 ** -10).expand(R * K, V).contiguous()
    select_check(rising, zeros, n)
    select_check(rising.flip(1).contiguous(), first, n)


# ---- beams that go on from another one ------------------------------------------------------------------
MAPS = {"copies": lambda K, rng: [0] * K, "cycle": lambda K, rng: [(k + 1) % K for k in range(K)], "swap": lambda K, rng: list(range(K))[::-1],
        "any": lambda K, rng: [rng.randrange(K) for _ in range(K)], "none": lambda K, rng: [rng.choice([k, -1, K, 99]) for k in range(K)]}


@pytest.mark.parametrize("kind", sorted(MAPS))
@pytest.mark.parametrize("K", [1, 2, 4, 5, 17, 64])
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (1000,)), (torch.bfloat16, (3, 7)), (torch.uint8, (5,)), (torch.float32, (5000, 3)), (torch.bfloat16, (64, 128))])
def test_beam_reorder_states(kind, K, dtype, shape):
    rng, R, L = random.Random(K), 3, 2
    state = torch.randint(0, 200, (L, R * K + 2, *shape), device=DEV).to(dtype)
    slots = rng.sample(range(R * K + 2), R * K)
    parents = [MAPS[kind](K, rng) for _ in range(R)]
    if K > 2:
        slots[1], slots[2 * K] = -1, R * K + 50
    want = state.clone()
    for r in range(R):
        for k in range(K):
            p = parents[r][k]
            s, f = slots[r * K + k], slots[r * K + p] if 0 <= p < K else -1
            if 0 <= s < R * K + 2 and 0 <= f < R * K + 2:
                want[:, s] = state[:, f]
    ops.beam_reorder_states(state, ints(slots).view(R, K), ints(parents))
    assert torch.equal(state, want)


@pytest.mark.parametrize("kind", sorted(MAPS))
@pytest.mark.parametrize("K,dtype,KV,hd,layers", [(2, torch.bfloat16, 2, 128, 3), (4, torch.float32, 1, 5, 1), (5, torch.bfloat16, 3, 7, 2), (20, torch.bfloat16, 1, 9, 0),
                                                  (64, torch.bfloat16, 1, 16, 1)])
def test_beam_reorder_pages(kind, K, dtype, KV, hd, layers):
    rng, R = random.Random(K * 7), 3
    max_pages, n_slots = 6, R * K + 2
    pool = plain.Pool(n_slots, max_pages, n_slots * max_pages)
    slots = [rng.sample(range(n_slots), R * K)[r * K:(r + 1) * K] for r in range(R)]
    taken = rng.sample(range(n_slots), R * K)
    slots = [taken[r * K:(r + 1) * K] for r in range(R)]
    for r in range(R):
        n = rng.choice([1, 63, 64, 100, 128, 300])
        lens = [n] * K if r < 2 else [rng.randint(1, max_pages * PAGE) for _ in range(K)]      # (lengths of their own)
        assert pool.resize(slots[r], lens) == 0
    lead = (layers,) if layers else ()
    pages = [torch.randint(0, 250, (*lead, n_slots * max_pages, KV, PAGE, hd), device=DEV).to(dtype) for _ in range(2)]
    dev, want = DevicePool(pool), [p.clone() for p in pages]
    for again in range(2):                                              # (twice: rows that already share pages, with lengths of their own the last too)
        parents, codes = [MAPS[kind](K, rng) for _ in range(R)], []
        for r in range(R):
            code, copies = pool.reorder(slots[r], parents[r])
            codes.append(code)
            assert code == 0 or (again and r == 2 and code == 5)
            for w in want:
                old = w.clone()
                for a, b, used in copies.values():
                    w[..., b, :, :used, :] = old[..., a, :, :used, :]
        ops.beam_reorder_pages(dev.table, dev.refs, dev.lengths, ints(slots), ints(parents), pages[0], pages[1], dev.status)
        dev.equals(pool)
        assert dev.status.tolist() == [max(codes)]
        dev.status.zero_()
        assert all(torch.equal(p, w) for p, w in zip(pages, want))
    # everything given back: no page is lost
    everyone = [s for row in slots for s in row]
    dev.resize(everyone, [0] * len(everyone))
    assert dev.refs.tolist() == [0] * len(pool.refs) and dev.status.tolist() == [0]


def test_beam_reorder_pages_that_cannot_be():
    """A request for which it cannot be done stays as it is; the others go on."""
    pool = plain.Pool(8, 4, 32)
    assert pool.resize([0, 1, 2, 3, 6, 7], [100, 100, 100, 100, 70, 70]) == 0
    shared = pool.copy()
    page = shared.table[3][1]
    shared.refs[page] = 2
    for slots, parents, code in [([[0, 1], [2, 4]], [[0, 0], [0, 0]], 4), ([[0, 1], [2, 2]], [[1, 1], [0, 0]], 3), ([[0, 1], [2, 9]], [[0, 0], [0, 1]], 3),
                                 ([[0, 1], [-1, 3]], [[0, 0], [0, 0]], 3), ([[0, 1], [2, 3]], [[0, 0], [0, 0]], 5)]:
        mine = (shared if code == 5 else pool).copy()
        dev = DevicePool(mine)
        pages = torch.randn(32, 1, PAGE, 8, device=DEV)
        want = pages.clone()
        assert mine.reorder(slots[1], parents[1])[0] == code
        good, copies = mine.reorder(slots[0], parents[0])
        assert good == 0
        for a, b, used in copies.values():
            want[b, :, :used] = pages[a, :, :used]
        ops.beam_reorder_pages(dev.table, dev.refs, dev.lengths, ints(slots), ints(parents), pages, None, dev.status)
        dev.equals(mine)
        assert dev.status.tolist() == [code] and torch.equal(pages, want)


def test_calls_of_nothing():
    """No requests, no rows, states of no values: nothing is launched that would touch anything."""
    zeros = lambda *shape, dtype=torch.int32: torch.zeros(*shape, dtype=dtype, device=DEV)
    table, refs, lengths, status, none = zeros(2, 3), zeros(6), zeros(2), zeros(1), zeros(0)
    pages = zeros(3, 6, 2, PAGE, 64, dtype=torch.bfloat16)
    rows = zeros(3, 0, 128, dtype=torch.bfloat16)
    ops.page_resize(table, refs, lengths, none, none, status)
    ops.kv_store(rows, rows, none, pages, pages)
    for n, slots in ((0, [0]), (2, [])):                               # a request of no rows, rows of no request
        q, kv, out = zeros(n, 256, dtype=torch.bfloat16), zeros(n, 128, dtype=torch.bfloat16), torch.full((n, 256), 3.0, dtype=torch.bfloat16, device=DEV)
        ops.tree_attention(q, kv, kv, pages[0], pages[0], table, ints(slots), ints(slots), zeros(len(slots) + 1), zeros(n), out, 4, 2, 64, 0.1,
                           max_context=10, max_new=2)
        assert bool((out == 3.0).all())
    assert ops.beam_select(zeros(0, 50, dtype=torch.float32), zeros(0, 4, dtype=torch.float32), 4)[0].shape == (0, 4)
    ops.beam_reorder_states(zeros(2, 3, 8), zeros(0, 4), zeros(0, 4))
    ops.beam_reorder_states(zeros(2, 3, 0), ints([[0, 1]]), ints([[1, 1]]))
    ops.beam_reorder_pages(table, refs, lengths, zeros(0, 4), zeros(0, 4), pages, pages, status)
    assert status.tolist() == [0] and not bool(pages.any()) and not bool(table.any())
    ops.check_errors()


# ---- together --------------------------------------------------------------------------------------------
def test_drafts_verified_and_accepted():
    """Drafts of three sequences through the whole path: masks, attention without storing, room for the accepted rows, storing; then the next row sees
    the same keys as if its path had been appended one by one."""
    rng, g = random.Random(4), torch.Generator(device=DEV).manual_seed(4)
    H, KV, hd, L = 4, 2, 64, 2
    pool = plain.Pool(4, 4, 14)
    slots, context, new = [2, 0, 3], [60, 130, 0], [9, 20, 6]
    assert pool.resize(slots, context) == 0
    dev = DevicePool(pool)
    pages = [torch.randn(L, 14, KV, PAGE, hd, device=DEV, generator=g).bfloat16() for _ in range(2)]
    T = sum(new)
    parents = [p for n in new for p in plain.draft(rng, n)]
    q = torch.randn(L, T, H * hd, device=DEV, generator=g).bfloat16()
    k, v = (torch.randn(L, T, KV * hd, device=DEV, generator=g).bfloat16() for _ in range(2))
    maps = ops.row_maps(dev.table, ints(slots), ints(context), ints(new), T, ints(parents), None, max(new))
    assert bool((maps.row_map == -1).all())
    out = torch.empty(L, T, H * hd, dtype=torch.bfloat16, device=DEV)
    for l in range(L):
        ops.tree_attention(q[l], k[l], v[l], pages[0][l], pages[1][l], dev.table, ints(slots), ints(context), maps.cu_seqlens, maps.positions, out[l], H, KV, hd,
                           0.125, max_context=192, max_new=max(new), mask=maps.mask)
    # the deepest row of every request and the rows above it are accepted
    keep, accepted, at = [False] * T, [], 0
    for n in new:
        pos = maps.positions[at:at + n].tolist()
        i, chain = max(range(n), key=lambda j: pos[j]), []
        while i >= 0:
            chain.insert(0, i)
            i = parents[at + i]
        for j in chain:
            keep[at + j] = True
        accepted.append([at + j for j in chain])
        at += n
    want = [c + len(a) for c, a in zip(context, accepted)]
    dev.resize(slots, want)
    again = ops.row_maps(dev.table, ints(slots), ints(context), ints(new), T, ints(parents), torch.tensor(keep, device=DEV), max(new))
    ops.kv_store(k, v, again.row_map, *pages)
    assert pool.resize(slots, want) == 0
    dev.equals(pool)
    # the last accepted row again, now alone over the pages (its own key among them): the same attention as inside the tree
    rows = [a[-1] for a in accepted]
    for l in range(L):
        alone = torch.empty(3, H * hd, dtype=torch.bfloat16, device=DEV)
        ops.attention(q[l][rows].contiguous(), pages[0][l], pages[1][l], dev.table, ints([w - 1 for w in want]), ints([0, 1, 2]), ints(slots), alone, H, KV, hd, 0.125,
                      decode_max_keys=256)
        # both are the same sum, each off by at most the weights' and the output's rounding
        vmax = max(float(pages[1][l].float().abs().max()), float(v.float().abs().max()))
        assert float((alone.float() - out[l][rows].float()).abs().max()) <= 4 * HALF * vmax
    ops.check_errors()


def test_a_beam_search_over_shared_pages():
    """Beams of two requests over a toy model whose next logits are a function of what its attention reads from the pages: ten steps of select, reorder,
    room, store against a search that keeps every beam's history in lists."""
    g = torch.Generator(device=DEV).manual_seed(9)
    R, K, V, hd, prompt = 2, 4, 50, 16, 61
    emb = torch.randn(V, hd, device=DEV, generator=g)
    head = torch.randn(hd, V, device=DEV, generator=g) * 2
    n_slots, n_pages, width = R * K, 40, 4
    pool = plain.Pool(n_slots, width, n_pages)
    dev = DevicePool(pool)
    k_pages, v_pages = (torch.zeros(n_pages, 1, PAGE, hd, device=DEV) for _ in range(2))
    state = torch.zeros(1, n_slots, 3, device=DEV)
    slots = [[r * K + (k * 3) % K for k in range(K)] for r in range(R)]
    flat = [s for row in slots for s in row]
    prompts = torch.randint(0, V, (R, prompt), generator=torch.Generator().manual_seed(1)).tolist()
    # the prompt in each request's first slot; the others get one position and the parent 0
    dev.resize([row[0] for row in slots], [prompt] * R)
    maps = ops.row_maps(dev.table, ints([row[0] for row in slots]), ints([0] * R), ints([prompt] * R), R * prompt)
    x = emb[torch.tensor(sum(prompts, []), device=DEV)]
    ops.kv_store(x, x * 0.5, maps.row_map, k_pages, v_pages)
    dev.resize([s for row in slots for s in row[1:]], [1] * (R * (K - 1)))
    zero = ints([[0] * K] * R)
    ops.beam_reorder_pages(dev.table, dev.refs, dev.lengths, ints(slots), zero, k_pages, v_pages, dev.status)
    scores = torch.tensor([[0.0] + [-float("inf")] * (K - 1)] * R, device=DEV)
    histories = [[list(p) for _ in range(K)] for p in prompts]
    list_scores = [[0.0] + [-float("inf")] * (K - 1) for _ in range(R)]

    def attend(rows, length):
        q = emb[torch.tensor(rows, device=DEV)].contiguous()
        out = torch.empty_like(q)
        ops.tree_attention(q, torch.zeros_like(q), torch.zeros_like(q), k_pages, v_pages, dev.table, ints(flat), ints([length] * (R * K)), ints(list(range(R * K + 1))),
                           ints([length] * (R * K)), out, 1, 1, hd, 0.25, max_context=width * PAGE, max_new=1, mask=ints([[0]] * (R * K)))
        return out

    for step in range(10):
        length = prompt + step
        logits = attend([h[-1] for row in histories for h in row], length) @ head
        tokens, parents, scores = ops.beam_select(logits, scores, K, placed=step % 2 == 1)
        # the same search over lists, in 64 bits from each beam's own history
        want = []
        for r in range(R):
            lg = []
            for h in histories[r]:
                e = emb[torch.tensor(h, device=DEV)].double()
                p = torch.softmax(e @ e[-1] * 0.25, 0)
                lg.append((p @ (e * 0.5)) @ head.double())
            want.append(plain.beam_select(torch.stack(lg).cpu(), torch.tensor([list_scores[r]], dtype=torch.float64), K, placed=step % 2 == 1))
        assert parents.tolist() == [w[1][0] for w in want] and tokens.tolist() == [w[0][0] for w in want]
        # 50 logits of 16 products, scores of ten steps in 32 bits: each step adds less than 1e-5
        assert torch.allclose(scores.cpu().double(), torch.cat([w[2] for w in want]), rtol=0, atol=1e-5 * (step + 1))
        list_scores = [w[2][0].tolist() for w in want]
        histories = [[histories[r][p] + [t] for p, t in zip(want[r][1][0], want[r][0][0])] for r in range(R)]
        ops.beam_reorder_pages(dev.table, dev.refs, dev.lengths, ints(slots), parents, k_pages, v_pages, dev.status)
        ops.beam_reorder_states(state, ints(slots), parents)
        dev.resize(flat, [length + 1] * (R * K))
        maps = ops.row_maps(dev.table, ints(flat), ints([length] * (R * K)), ints([1] * (R * K)), R * K)
        x = emb[tokens.flatten().long()]
        ops.kv_store(x, x * 0.5, maps.row_map, k_pages, v_pages)
        state[0, torch.tensor(flat, device=DEV).long(), step % 3] = tokens.flatten().float()
        for r in range(R):
            for k in range(K):
                assert state[0, slots[r][k]].tolist() == [float(histories[r][k][prompt + i] if i <= step else 0) for i in
                                                          [max([s for s in range(step + 1) if s % 3 == m], default=m) for m in range(3)]]
    assert dev.status.tolist() == [0]
    assert max(dev.refs.tolist()) > 1                               # the prompt's page is shared
    dev.resize(flat, [0] * (R * K))
    assert dev.refs.tolist() == [0] * n_pages
