"""What the operators for several candidates of a request are measured on: drafted tokens that may be thrown away and beams that share
pages, over the paged cache.  A page holds 64 positions; keys and values are [pages, kv heads, 64, head size] per layer; block_table
[slots, pages a slot] names the page of every 64 positions of a slot; refs [pages] counts the table entries that name a page (0: free).

  rows      a step's bookkeeping: room for the positions that requests want (the lowest free pages, request by request), sums,
            sequences, positions and places of the step's rows; with layers, the rows' keys and values go to their places (drafts:
            only the rows of the accepted path); then the room is given back, as when a step is withdrawn
  tree      attention of drafted tokens: every row sees its request's context and the drafts among its ancestors
  select    beam search: log softmax of every beam's logits, plus the beam's score; the best candidates of each request
  reorder   beam search: beams whose parent is another beam take over its pages, what its last page holds and its states

The plain form and exact() are written from these definitions.
"""
import math
import random

import torch

own = False

PAGE = 64


def _rows(name, requests, pool, context, new, drafts=0, layers=0, kv=2, hd=128, x="bfloat16"):
    """context, new: the shortest and the longest; pool: pages; drafts: length of the accepted path of a draft (0: rows are plain)."""
    case = dict(kind="rows", requests=requests, pool=pool, context_lo=context[0], context_hi=context[1], new_lo=new[0], new_hi=new[1],
                drafts=drafts, layers=layers, kv=kv, hd=hd, x=x)
    return dict(case, name=name) if name else case


def _tree(name, requests, context, new, heads, kv, hd, x="bfloat16", window=0, softcap=0.0, sink=False):
    case = dict(kind="tree", requests=requests, context_lo=context[0], context_hi=context[1], new_lo=new[0], new_hi=new[1], heads=heads,
                kv=kv, hd=hd, x=x, window=window, softcap=softcap, sink=sink)
    return dict(case, name=name) if name else case


def _select(name, requests, beams, vocab, n, first=False, ended=0, placed=False):
    """first: only beam 0 is alive; ended: beams of each request that have ended; placed: children stay where their parents are."""
    case = dict(kind="select", requests=requests, beams=beams, vocab=vocab, n=n, first=first, ended=ended, placed=placed)
    return dict(case, name=name) if name else case


def _reorder(name, requests, beams, moved, context, layers, kv, hd, state_layers=0, state=0):
    """moved: beams of each request that are replaced by copies of others; state: 32-bit values of a beam's state in each state layer."""
    case = dict(kind="reorder", requests=requests, beams=beams, moved=moved, context_lo=context[0], context_hi=context[1], layers=layers,
                kv=kv, hd=hd, state_layers=state_layers, state=state)
    return dict(case, name=name) if name else case


def listed():
    return [
        # eight sequences decode one token each: the smallest bookkeeping
        _rows("rows-8", 8, 2048, (1, 2000), (1, 1)),
        # a scheduler's step over many sequences, prompts among them, in a large pool
        _rows("rows-700", 700, 150000, (0, 9000), (1, 150)),
        # drafts of 16 sequences: the accepted rows of all 24 layers go into the cache
        _rows("accept-16", 16, 800, (100, 4000), (20, 48), drafts=5, layers=24),
        # prompts of 8,192 rows in all, keys and values of a layer from 32-bit projections
        _rows("prompt-4", 4, 4096, (0, 3000), (1500, 2600), layers=2, x="float32"),
        # one sequence, eight drafted tokens: the smallest attention
        _tree("tree-1", 1, (600, 600), (8, 8), 8, 2, 128),
        # a batch of ragged contexts and drafts
        _tree("tree-16", 16, (150, 6000), (17, 64), 10, 2, 128),
        # two documents, wide drafts
        _tree("tree-2-long", 2, (45000, 60001), (48, 63), 8, 2, 128),
        # 32 bits, capped scores and a sink, a window, an odd head size
        _tree("tree-3-f32", 3, (70, 1900), (5, 21), 6, 3, 80, "float32", 700, 30.0, True),
        # one request, four beams, the first step
        _select("select-1", 1, 4, 65536, 4, first=True),
        # a batch of requests; twice the beams as candidates, some beams have ended
        _select("select-32", 32, 8, 130048, 16, ended=2),
        # one request, attention layers only
        _reorder("reorder-1", 1, 4, 2, (310, 310), 4, 2, 128),
        # eight requests, states of recurrent layers and pages of attention layers
        _reorder("reorder-8", 8, 4, 2, (40, 1500), 8, 2, 128, 6, 48 * 64 * 256),
    ]


_MOST_KEYS = 2 * 60001 * 2 * 128 * 2              # values of keys and values that the largest listed attention reads
_MOST_PRODUCTS = 2 * 60001 * 63 * 8 * 128         # and its products of a query with a key, value by value


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "rows", "tree", "tree", "tree", "select", "select", "reorder"])
    if kind == "rows":
        requests, drafts, layers = _log_int(rng, 1, 700), 0, rng.choice([0, 0, 1, 3, 8, 24])
        context_hi = _log_int(rng, 64, 9000)
        if rng.random() < 0.5:
            drafts, new = rng.randint(1, 8), (8, rng.randint(8, 64))
        else:
            new = (rng.randint(0, 1), _log_int(rng, 1, 300))
        kv, hd = rng.choice([1, 2, 3, 8]), rng.choice([16, 64, 80, 128])
        while layers * requests * new[1] * kv * hd > 1 << 24 or (layers and requests * context_hi * layers * kv * hd > 1 << 28):
            requests = max(1, requests // 2)
            layers, context_hi = (layers + 1) // 2, max(64, context_hi // 2)
            if requests == 1 and layers == 1:
                break
        need = requests * ((context_hi + new[1] + PAGE - 1) // PAGE + 1)
        return _rows(None, requests, need + _log_int(rng, 16, 60000) if not layers else need + rng.randint(0, 256), (0, context_hi), new,
                     drafts, layers, kv, hd, rng.choice(["bfloat16", "float32"]))
    if kind == "tree":
        x = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        kv, group = rng.choice([1, 2, 2, 3, 8]), rng.choice([1, 3, 4, 5, 6, 8])
        hd = rng.choice([128, 128, 64]) if x == "bfloat16" and rng.random() < 0.8 else rng.choice([16, 40, 80, 128, 256])
        requests, context_hi, most = _log_int(rng, 1, 64), _log_int(rng, 16, 60000), _log_int(rng, 1, 128)
        share = 1 if x == "bfloat16" and hd in (64, 128) else 16
        while share * 2 * requests * context_hi * kv * hd > _MOST_KEYS or share * requests * context_hi * most * kv * group * hd > _MOST_PRODUCTS:
            requests, context_hi = max(1, requests // 2), (2 * context_hi + 2) // 3
        return _tree(None, requests, (rng.choice([0, context_hi // 10]), context_hi), (max(1, most // 3), most), kv * group, kv, hd, x,
                     rng.choice([0, 0, 0, 100, 1000]), rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.3)
    if kind == "select":
        beams, requests = rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), _log_int(rng, 1, 64)
        vocab = rng.choice([_log_int(rng, 200, 130048), 65536, 65537, 130048])
        while requests * beams * vocab > 32 * 8 * 130048:
            requests = max(1, requests // 2)
        placed = rng.random() < 0.4
        return _select(None, requests, beams, vocab, beams if placed else beams * rng.choice([1, 2]), rng.random() < 0.2,
                       rng.randint(0, beams - 1) if rng.random() < 0.5 else 0, placed)
    beams = rng.choice([2, 3, 4, 5, 8, 12])
    requests, layers, kv, hd, hi = _log_int(rng, 1, 16), rng.choice([1, 3, 8]), rng.choice([1, 2, 4]), rng.choice([64, 128, 24]), _log_int(rng, 8, 1500)
    state_layers, state = rng.choice([(0, 0), (2, _log_int(rng, 100, 800000)), (6, 24 * 128 * 16)])
    while requests > 1 and requests * beams * max(4 * layers * kv * hd * (hi + PAGE), 4 * state_layers * state) > 1 << 29:
        requests //= 2
    return _reorder(None, requests, beams, rng.randint(1, beams // 2), (max(1, hi // 8), hi), layers, kv, hd, state_layers, state)


# ---- inputs ------------------------------------------------------------------------------------------
_TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _ragged(n, lo, hi, salt):
    """n lengths lo..hi, the same for every seed (what a pass has to do is then the case's); the longest among them."""
    rng = random.Random(n * 1000003 + lo * 10007 + hi * 101 + salt)
    return [hi] + [rng.randint(lo, hi) for _ in range(n - 1)]


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _random(g, shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


def _pool(g, seed, n_slots, slots, lengths, pool, width):
    """A pool in use: every slot's pages, at random places.  (block_table, refs, lengths of all slots)."""
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(n_slots, width, dtype=torch.int32)
    held = torch.zeros(n_slots, dtype=torch.int32)
    order, at = order.cpu(), 0
    for s, n in zip(slots, lengths):
        k = _pages(n)
        table[s, :k] = order[at:at + k]
        at += k
        held[s] = n
    refs = torch.zeros(pool, dtype=torch.int32)
    refs[order[:at].long()] = 1
    return table.cuda(), refs.cuda(), held.cuda()


def _draft(rng, n, path):
    """Parents (-1: the context) of n drafted rows; the accepted path: `path` of them, each the child of the one before."""
    chain = sorted(rng.sample(range(n), min(path, n)))
    parents = [rng.randint(max(-1, i - 9), i - 1) for i in range(n)]
    for before, i in zip([-1] + chain, chain):
        parents[i] = before
    return parents, chain


def _masks(parents, words):
    """Bits of what each row of a draft sees, itself among it: words of 32 bits."""
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    out = [[(m >> 32 * w) & 0xFFFFFFFF for w in range(words)] for m in seen]
    return [[v - (1 << 32) if v >> 31 else v for v in row] for row in out]


def prepare(case, seed):
    g, rng = _generator(seed), random.Random(int(seed))
    s = dict(case=case)
    if case["kind"] == "rows":
        b = case["requests"]
        start, new = _ragged(b, case["context_lo"], case["context_hi"], 1), _ragged(b, case["new_lo"], case["new_hi"], 2)[::-1]
        width = _pages(case["context_hi"] + case["new_hi"]) + 2
        slots = rng.sample(range(b + 3), b)
        s["table"], s["refs"], s["lengths"] = _pool(g, seed, b + 3, slots, start, case["pool"], width)
        s["slots"], s["start"], s["new"], s["rows"], s["status"] = _ints(slots), _ints(start), _ints(new), sum(new), _ints([0, 0])
        s["parents"] = s["keep"] = None
        kept = new
        if case["drafts"]:
            parents, keep, kept = [], [], []
            for n in new:
                p, chain = _draft(rng, n, case["drafts"])
                parents += p
                keep += [i in chain for i in range(n)]
                kept.append(len(chain))
            s["parents"], s["keep"] = _ints(parents), torch.tensor(keep, device="cuda")
        s["want"], s["most"] = _ints([a + k for a, k in zip(start, kept)]), max(new)
        if case["layers"]:
            shape = (case["layers"], s["rows"], case["kv"] * case["hd"])
            s["k"], s["v"] = _random(g, shape, _TYPES[case["x"]]), _random(g, shape, _TYPES[case["x"]])
            shape = (case["layers"], case["pool"], case["kv"], PAGE, case["hd"])
            s["k_pages"], s["v_pages"] = torch.zeros(shape, dtype=torch.bfloat16, device="cuda"), torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    elif case["kind"] == "tree":
        b, dtype = case["requests"], _TYPES[case["x"]]
        start, new = _ragged(b, case["context_lo"], case["context_hi"], 1), _ragged(b, case["new_lo"], case["new_hi"], 2)[::-1]
        slots = rng.sample(range(b + 3), b)
        pool = sum(_pages(n) for n in start) + 5
        s["table"], _, _ = _pool(g, seed, b + 3, slots, start, pool, _pages(case["context_hi"] + case["new_hi"]) + 1)
        parents = [_draft(rng, n, 1 + n // 4)[0] for n in new]
        words = (max(new) + 31) // 32
        s["mask"] = _ints([row for p in parents for row in _masks(p, words)])
        depth = []
        for p, at in zip(parents, start):
            d = []
            for q in p:
                d.append(d[q] + 1 if q >= 0 else at)
            depth += d
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        s["cu"], s["positions"], s["slots"], s["start"] = _ints(cu), _ints(depth), _ints(slots), _ints(start)
        s["host"] = (start, new, cu)
        rows, kv, hd = cu[-1], case["kv"], case["hd"]
        s["q"] = _random(g, (rows, case["heads"] * hd), dtype)
        s["k"], s["v"] = _random(g, (rows, kv * hd), dtype), _random(g, (rows, kv * hd), dtype)
        s["k_pages"], s["v_pages"] = _random(g, (pool, kv, PAGE, hd), dtype), _random(g, (pool, kv, PAGE, hd), dtype)
        s["sinks"] = _random(g, (case["heads"],)) if case["sink"] else None
    elif case["kind"] == "select":
        r, k = case["requests"], case["beams"]
        # logits of a language model: a few tokens far above the rest, unequally many of them a row
        x = _random(g, (r * k, case["vocab"]))
        s["logits"] = x * 2.0 + x.clamp(min=2.5).sub_(2.5) * (4.0 * torch.rand(r * k, 1, generator=g, device="cuda"))
        s["scores"] = -5.0 * torch.rand(r, k, generator=g, device="cuda") - 3.0
        s["ended"] = None
        if case["first"]:
            s["scores"][:, 1:] = -math.inf
        elif case["ended"]:
            s["ended"] = torch.rand(r, k, generator=g, device="cuda").argsort(1) < case["ended"]
    else:
        r, k, moved = case["requests"], case["beams"], case["moved"]
        length = _ragged(r, case["context_lo"], case["context_hi"], 3)
        slots = rng.sample(range(r * k + 2), r * k)
        # every beam with pages of its own: more of them than a search that shared its prompt's would hold
        each = [length[i // k] for i in range(r * k)]
        pool = sum(_pages(n) for n in each) + 3
        s["table"], s["refs"], s["lengths"] = _pool(g, seed, r * k + 2, slots, each, pool, _pages(case["context_hi"]) + 2)
        parents = []
        for _ in range(r):
            order = rng.sample(range(k), k)
            gone, stay = order[:moved], order[moved:]
            row = list(range(k))
            for c, p in zip(gone, stay):
                row[c] = p
            parents.append(row)
        s["slots"], s["parents"], s["status"] = _ints(slots).view(r, k), _ints(parents), _ints([0, 0])
        shape = (case["layers"], pool, case["kv"], PAGE, case["hd"])
        s["k_pages"], s["v_pages"] = _random(g, shape, torch.bfloat16), _random(g, shape, torch.bfloat16)
        s["state"] = _random(g, (case["state_layers"], r * k + 2, case["state"])) if case["state_layers"] else None
    return s


# ---- one pass ----------------------------------------------------------------------------------------
def _plain_resize(s, want):
    table, refs, lengths, slots = s["table"], s["refs"], s["lengths"], s["slots"].long()
    have, need = (lengths[slots].long() + PAGE - 1) // PAGE, (want.long() + PAGE - 1) // PAGE
    column = torch.arange(table.shape[1], device="cuda")
    rows = table[slots]
    drop = (column >= need[:, None]) & (column < have[:, None])
    refs.index_add_(0, rows[drop].long(), torch.full((), -1, dtype=torch.int32, device="cuda").expand(int(drop.sum())))
    take = (column >= have[:, None]) & (column < need[:, None])
    rows[drop] = 0
    pages = torch.nonzero(refs == 0).flatten()[:int(take.sum())]
    rows[take] = pages.to(torch.int32)
    refs[pages] = 1
    table[slots] = rows
    lengths[slots] = want
    s["status"].zero_()


def _plain_rows(s):
    case, slots, start, new, n = s["case"], s["slots"].long(), s["start"].long(), s["new"].long(), s["rows"]
    _plain_resize(s, s["want"])
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    row_seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), new)
    index = torch.arange(n, device="cuda") - cu[row_seq]
    outs = []
    if s["parents"] is None:
        depth = index
    else:
        # step by step up the tree, all rows at once
        base, depth, at = cu[row_seq], torch.zeros_like(index), s["parents"].long()
        words = (s["most"] + 31) // 32
        mask = torch.zeros(n, words, dtype=torch.int64, device="cuda")
        here = torch.arange(n, device="cuda")
        mask[here, index // 32] = 1 << index % 32
        for _ in range(s["most"]):
            up = at >= 0
            if not bool(up.any()):
                break
            depth = depth + up
            word = at.clamp(min=0) // 32
            mask[here, word] |= torch.where(up, 1 << at.clamp(min=0) % 32, 0)
            at = torch.where(up, s["parents"].long()[base + at.clamp(min=0)], at)
        outs.append(torch.where(mask >> 31 > 0, mask - (1 << 32), mask).to(torch.int32))
    position = start[row_seq] + depth
    width = s["table"].shape[1]
    place = s["table"][slots[row_seq], (position // PAGE).clamp(max=width - 1)].long() * PAGE + position % PAGE
    if s["keep"] is not None:
        place = torch.where(s["keep"], place, -1)
    elif s["parents"] is not None:
        place = torch.full_like(place, -1)
    if case["layers"]:
        to = place[place >= 0]
        for rows, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
            rows = rows.view(case["layers"], n, case["kv"], case["hd"])[:, place >= 0]
            pages[:, to // PAGE, :, to % PAGE] = rows.transpose(0, 1).to(torch.bfloat16)
        outs += [s["k_pages"], s["v_pages"]]
    _plain_resize(s, s["start"])
    return [t.to(torch.int32) for t in (cu, row_seq, position, place)] + outs + [s["table"], s["refs"], s["lengths"], s["status"]]


def _bits(mask, n):
    """[rows, words] -> truth values [rows, n]."""
    at = torch.arange(n, device=mask.device)
    return (mask[:, at // 32] >> (at % 32).to(torch.int32) & 1) != 0


def _plain_tree(s):
    case, (start, new, cu) = s["case"], s["host"]
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    out = torch.empty(cu[-1], heads, hd, dtype=s["q"].dtype, device="cuda")
    for b, (n_old, n) in enumerate(zip(start, new)):
        here = slice(cu[b], cu[b] + n)
        pages = s["table"][s["slots"][b], :_pages(n_old)].long()
        k, v = (torch.cat([p[pages].transpose(0, 1).reshape(kv, -1, hd)[:, :n_old], r[here].view(n, kv, hd).transpose(0, 1)], 1).float()
                for p, r in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])))
        q = s["q"][here].float().view(n, kv, heads // kv, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd)
        score = (q @ k.transpose(1, 2) * hd ** -0.5).view(kv, heads // kv, n, n_old + n)
        if case["softcap"]:
            score = case["softcap"] * torch.tanh(score / case["softcap"])
        at = s["positions"][here]
        seen = torch.cat([torch.ones(n, n_old, dtype=torch.bool, device="cuda"), _bits(s["mask"][here], n)], 1)
        if case["window"]:
            key_at = torch.cat([torch.arange(n_old, device="cuda", dtype=torch.int32), at])
            seen &= key_at[None, :] > at[:, None] - case["window"]
        score = score.masked_fill(~seen, -math.inf)
        most = score.amax(-1, keepdim=True)
        if case["sink"]:
            sink = s["sinks"].view(kv, heads // kv, 1, 1)
            most = torch.maximum(most, sink)
        p = torch.exp(score - most)
        total = p.sum(-1, keepdim=True)
        if case["sink"]:
            total = total + torch.exp(sink - most)
        y = (p / total).view(kv, -1, n_old + n) @ v
        out[here] = y.view(kv, heads // kv, n, hd).permute(2, 0, 1, 3).reshape(n, heads, hd).to(out.dtype)
    return out.view(cu[-1], heads * hd)


def _plain_select(s):
    case = s["case"]
    r, k, v, n = case["requests"], case["beams"], case["vocab"], case["n"]
    x = s["logits"].double()
    most = x.amax(1, keepdim=True)
    x = x - (most + torch.log(torch.exp(x - most).sum(1, keepdim=True)))
    x = x.view(r, k, v) + s["scores"].double()[:, :, None]
    if s["ended"] is not None:                              # an ended beam stands for itself, with token 0
        x = x.masked_fill(s["ended"][:, :, None], -math.inf)
        x[:, :, 0] = torch.where(s["ended"], s["scores"].double(), x[:, :, 0])
    best = x.view(r, k * v).topk(2 * n if 2 * n <= k * v else n)
    at = best.indices.sort(1)                               # equal values: the lowest index first
    value = best.values.gather(1, at.indices).sort(dim=1, descending=True, stable=True)
    score, at = value.values[:, :n], at.values.gather(1, value.indices)[:, :n]
    parent, token = at // v, at % v
    if case["placed"]:
        # the first child of a beam takes its place, the others the places that are left, in order
        place = torch.full_like(parent, -1)
        free = torch.ones(r, k, dtype=torch.bool, device=x.device)
        rows = torch.arange(r, device=x.device)
        for i in range(n):
            ok = free[rows, parent[:, i]]
            place[:, i] = torch.where(ok, parent[:, i], -1)
            free[rows, parent[:, i]] = False
        for i in range(n):
            left = free.int().argmax(1)
            late = place[:, i] < 0
            place[:, i] = torch.where(late, left, place[:, i])
            free[rows[late], left[late]] = False
        order = place.argsort(1)
        parent, token, score = (t.gather(1, order) for t in (parent, token, score))
    return token.to(torch.int32), parent.to(torch.int32), score.float()


def _plain_reorder(s):
    case, table, refs, lengths = s["case"], s["table"], s["refs"], s["lengths"]
    slots = s["slots"].long()
    source = slots.gather(1, s["parents"].long()).flatten()
    slots = slots.flatten()
    moved = source != slots
    slots, source = slots[moved], source[moved]
    column = torch.arange(table.shape[1], device="cuda")
    have, length = (lengths[slots].long() + PAGE - 1) // PAGE, lengths[source].long()
    full, used = length // PAGE, length % PAGE
    old, new = table[slots], table[source]
    last, from_page = old.gather(1, have[:, None] - 1), new.gather(1, full.clamp(max=table.shape[1] - 1)[:, None])
    # whole pages are shared; the page that is being filled stays the beam's own and takes over what the parent's holds
    own_last = (column == have[:, None] - 1) & (used > 0)[:, None]
    gone = old[(column < have[:, None]) & ~own_last].long()
    shared = new[column < full[:, None]].long()
    refs.index_add_(0, gone, torch.full((len(gone),), -1, dtype=torch.int32, device="cuda"))
    refs.index_add_(0, shared, torch.ones(len(shared), dtype=torch.int32, device="cuda"))
    row = torch.where(column < full[:, None], new, 0)
    row = torch.where((column == full[:, None]) & (used > 0)[:, None], last, row)
    table[slots] = row.to(torch.int32)
    lengths[slots] = length.to(torch.int32)
    to, fr = last.flatten()[used > 0].long(), from_page.flatten()[used > 0].long()
    inside = (torch.arange(PAGE, device="cuda") < used[used > 0][:, None])[None, :, None, :, None]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[:, to] = torch.where(inside, pages[:, fr], pages[:, to])
    outs = [table, refs, lengths, s["k_pages"], s["v_pages"]]
    if s["state"] is not None:
        s["state"][:, slots] = s["state"][:, source]
        outs.append(s["state"])
    return outs


def _own(s):
    from tinyllama_c_b200 import ops
    case = s["case"]
    if case["kind"] == "rows":
        ops.page_resize(s["table"], s["refs"], s["lengths"], s["slots"], s["want"], s["status"])
        maps = ops.row_maps(s["table"], s["slots"], s["start"], s["new"], s["rows"], parents=s["parents"], keep=s["keep"], max_new=s["most"])
        outs = [] if s["parents"] is None else [maps.mask]
        if case["layers"]:
            ops.kv_store(s["k"], s["v"], maps.row_map, s["k_pages"], s["v_pages"])
            outs += [s["k_pages"], s["v_pages"]]
        ops.page_resize(s["table"], s["refs"], s["lengths"], s["slots"], s["start"], s["status"])
        return [maps.cu_seqlens, maps.row_seq, maps.positions, maps.row_map] + outs + [s["table"], s["refs"], s["lengths"], s["status"]]
    if case["kind"] == "tree":
        heads, kv, hd = case["heads"], case["kv"], case["hd"]
        out = torch.empty_like(s["q"])
        ops.tree_attention(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["slots"], s["start"], s["cu"], s["positions"],
                           out, heads, kv, hd, hd ** -0.5, max_context=case["context_hi"], max_new=case["new_hi"], mask=s["mask"],
                           window=case["window"], softcap=case["softcap"], sink_values=s["sinks"])
        return out
    if case["kind"] == "select":
        return ops.beam_select(s["logits"], s["scores"], case["n"], ended=s["ended"], placed=case["placed"])
    ops.beam_reorder_pages(s["table"], s["refs"], s["lengths"], s["slots"], s["parents"], s["k_pages"], s["v_pages"], s["status"])
    outs = [s["table"], s["refs"], s["lengths"], s["k_pages"], s["v_pages"]]
    if s["state"] is not None:
        ops.beam_reorder_states(s["state"], s["slots"], s["parents"])
        outs.append(s["state"])
    return outs


def run(state):
    if own:
        return _own(state)
    return {"rows": _plain_rows, "tree": _plain_tree, "select": _plain_select, "reorder": _plain_reorder}[state["case"]["kind"]](state)


def work(case):
    size = dict(bfloat16=2, float32=4)
    if case["kind"] == "rows":
        start = _ragged(case["requests"], case["context_lo"], case["context_hi"], 1)
        new = _ragged(case["requests"], case["new_lo"], case["new_hi"], 2)[::-1]
        kept = [min(case["drafts"], n) if case["drafts"] else n for n in new]
        pages = sum(_pages(a + n) - _pages(a) for a, n in zip(start, kept))
        held = sum(_pages(a) for a in start)
        # refs up to the last page taken (free ones lie everywhere), taken entries written twice, lengths and counts, what a row is told
        looked = min(case["pool"], pages * case["pool"] // max(1, case["pool"] - held))
        total = 4 * looked + 16 * pages + 28 * len(new) + 12 * sum(new)
        if case["drafts"]:
            total += sum(new) * (5 + 4 * ((case["new_hi"] + 31) // 32))
        return {"bytes": total + 2 * case["layers"] * sum(kept) * case["kv"] * case["hd"] * (size[case["x"]] + 2), "flops": 0}
    if case["kind"] == "tree":
        start = _ragged(case["requests"], case["context_lo"], case["context_hi"], 1)
        new = _ragged(case["requests"], case["new_lo"], case["new_hi"], 2)[::-1]
        heads, kv, hd = case["heads"], case["kv"], case["hd"]
        seen = [min(a, case["window"] + n) if case["window"] else a for a, n in zip(start, new)]
        keys = [min(a, case["window"]) if case["window"] else a for a in start]
        values = 2 * kv * hd * (sum(seen) + sum(new)) + 2 * heads * hd * sum(new)
        return {"bytes": size[case["x"]] * values, "flops": 4 * heads * hd * sum(n * (c + (n + 1) // 4) for n, c in zip(new, keys))}
    if case["kind"] == "select":
        rows = case["requests"] * (case["beams"] - case["ended"] if not case["first"] else 1)
        return {"bytes": 4 * rows * case["vocab"] + 16 * case["requests"] * case["n"], "flops": 4 * rows * case["vocab"]}
    used = [n % PAGE for n in _ragged(case["requests"], case["context_lo"], case["context_hi"], 3)]
    values = 2 * case["layers"] * case["kv"] * case["hd"] * 2 * sum(used) + 4 * case["requests"] * case["state_layers"] * case["state"]
    tables = sum(_pages(n) for n in _ragged(case["requests"], case["context_lo"], case["context_hi"], 3))
    return {"bytes": case["moved"] * (2 * values + 28 * tables), "flops": 0}


# ---- in 64 bits --------------------------------------------------------------------------------------
def _exact_tree(s):
    case, (start, new, cu) = s["case"], s["host"]
    kv, hd = case["kv"], case["hd"]
    group = case["heads"] // kv
    out = torch.zeros(cu[-1], case["heads"], hd, dtype=torch.float64, device="cuda")
    table, slots = s["table"].cpu(), s["slots"].cpu()
    for b in range(len(start)):
        rows = torch.arange(cu[b], cu[b + 1], device="cuda")
        place = torch.arange(start[b])
        page = table[int(slots[b])].long()[place // PAGE].cuda()
        place = (place % PAGE).cuda()
        at = s["positions"].double()[rows]
        where = torch.cat([torch.arange(start[b], device="cuda").double(), at])
        j = torch.arange(new[b], device="cuda")
        visible = torch.cat([at.new_ones(len(rows), start[b]), ((s["mask"][rows][:, j // 32].long() >> (j % 32)) % 2).double()], 1) > 0
        if case["window"]:
            visible = visible & (at[:, None] - where[None, :] < case["window"])
        for h in range(kv):
            k = torch.cat([s["k_pages"][page, h, place].double(), s["k"][rows, h * hd:(h + 1) * hd].double()])
            v = torch.cat([s["v_pages"][page, h, place].double(), s["v"][rows, h * hd:(h + 1) * hd].double()])
            for i in range(h * group, (h + 1) * group):
                z = torch.einsum("id,jd->ij", s["q"][rows, i * hd:(i + 1) * hd].double(), k) / math.sqrt(hd)
                if case["softcap"]:
                    z = torch.tanh(z / case["softcap"]) * case["softcap"]
                z = torch.where(visible, z, torch.full_like(z, -math.inf))
                if case["sink"]:
                    z = torch.cat([z, s["sinks"][i].double().expand(len(rows), 1)], 1)
                w = torch.softmax(z, 1)[:, :len(where)]
                out[rows, i] = torch.einsum("ij,jd->id", w, v)
    return out.flatten(1)


def _exact_select(s):
    case = s["case"]
    r, k, v, n = case["requests"], case["beams"], case["vocab"], case["n"]
    tokens, parents, scores = [], [], []
    for i in range(r):
        rows = torch.log_softmax(s["logits"][i * k:(i + 1) * k].double(), 1) + s["scores"][i].double()[:, None]
        if s["ended"] is not None:
            for b in torch.nonzero(s["ended"][i]).flatten().tolist():
                rows[b] = -math.inf
                rows[b, 0] = s["scores"][i, b].double()
        flat = rows.flatten()
        order = torch.sort(flat, descending=True, stable=True).indices[:n].tolist()
        if case["placed"]:
            spot, seen, later = {}, set(), []
            for c in order:
                if c // v in seen:
                    later.append(c)
                else:
                    seen.add(c // v)
                    spot[c // v] = c
            for p in range(k):
                if p not in spot:
                    spot[p] = later.pop(0)
            order = [spot[p] for p in range(k)]
        tokens.append([c % v for c in order])
        parents.append([c // v for c in order])
        scores.append(flat[order])
    return _ints(tokens), _ints(parents), torch.stack(scores)


def _exact_reorder(s):
    case = s["case"]
    slots, parents, lengths, table = s["slots"].tolist(), s["parents"].tolist(), s["lengths"].tolist(), s["table"].tolist()
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    state = None if s["state"] is None else s["state"].double()
    for beams, ups in zip(slots, parents):
        for slot, up in zip(beams, ups):
            if beams[up] == slot:
                continue
            n = lengths[beams[up]]
            if n % PAGE:
                fr, to = table[beams[up]][n // PAGE], table[slot][(lengths[slot] - 1) // PAGE]
                for new, old in ((k_pages, s["k_pages"]), (v_pages, s["v_pages"])):
                    new[:, to, :, :n % PAGE] = old[:, fr, :, :n % PAGE].double()
            if state is not None:
                state[:, slot] = s["state"][:, beams[up]].double()
    outs = [None, None, None, k_pages, v_pages]
    return outs if state is None else outs + [state]


def _exact_rows(s):
    case, start, new = s["case"], s["start"].tolist(), s["new"].tolist()
    outs = [None] * 4 + ([] if s["parents"] is None else [None])
    if case["layers"]:
        # a row's page: the one it has, or the lowest free ones in the requests' order
        table, slots, want = s["table"].tolist(), s["slots"].tolist(), s["want"].tolist()
        free = iter(torch.nonzero(s["refs"] == 0).flatten().tolist())
        for slot, a, w in zip(slots, start, want):
            for c in range(_pages(a), _pages(w)):
                table[slot][c] = next(free)
        keep = [True] * s["rows"] if s["keep"] is None else s["keep"].tolist()
        row, rows, pages, offsets = 0, [], [], []
        for slot, a, n in zip(slots, start, new):
            at = a
            for i in range(n):
                if keep[row]:
                    rows.append(row)
                    pages.append(table[slot][at // PAGE])
                    offsets.append(at % PAGE)
                    at += 1
                row += 1
        pages, offsets = torch.tensor(pages, dtype=torch.long, device="cuda"), torch.tensor(offsets, dtype=torch.long, device="cuda")
        for x, y in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
            y = y.double()
            for layer in range(case["layers"]):
                y[layer][pages, :, offsets] = x[layer][rows].double().view(len(rows), case["kv"], case["hd"])
            outs.append(y)
    return outs + [None] * 4


def exact(case, seed):
    if case["kind"] == "rows" and not case["layers"]:
        return None
    s = prepare(case, seed)
    return {"rows": _exact_rows, "tree": _exact_tree, "select": _exact_select, "reorder": _exact_reorder}[case["kind"]](s)
