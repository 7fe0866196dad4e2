"""Plain forms of the operators for several candidates of a request: Python lists for the pool, 64-bit arithmetic for the rest."""
import math

import torch

PAGE = 64


def pages_of(n):
    return -(-n // PAGE)


class Pool:
    """The pool as lists: table rows, counts, lengths."""

    def __init__(self, n_slots, max_pages, n_pages):
        self.table = [[0] * max_pages for _ in range(n_slots)]
        self.refs = [0] * n_pages
        self.lengths = [0] * n_slots

    def copy(self):
        p = Pool(0, 0, 0)
        p.table, p.refs, p.lengths = [list(r) for r in self.table], list(self.refs), list(self.lengths)
        return p

    def resize(self, slots, want):
        """The code; with one, nothing has changed."""
        code, named = 0, set()
        for s, w in zip(slots, want):
            if s < 0:
                continue
            if s >= len(self.table) or s in named:
                code = max(code, 3)
                continue
            named.add(s)
            if w < 0 or pages_of(w) > len(self.table[s]):
                code = max(code, 2)
        if code:
            return code
        new = self.copy()
        live = [(s, w) for s, w in zip(slots, want) if s >= 0]
        for s, w in live:
            for c in range(pages_of(w), pages_of(self.lengths[s])):
                new.refs[new.table[s][c]] -= 1
        for s, w in live:
            n = self.lengths[s]
            if w > n and n % PAGE and new.refs[new.table[s][pages_of(n) - 1]] != 1:
                return 5
        for s, w in live:
            for c in range(pages_of(self.lengths[s]), pages_of(w)):
                if 0 not in new.refs:
                    return 1
                p = new.refs.index(0)
                new.refs[p], new.table[s][c] = 1, p
        for s, w in live:
            for c in range(pages_of(w), pages_of(self.lengths[s])):
                new.table[s][c] = 0
            new.lengths[s] = w
        self.__dict__.update(new.__dict__)
        return 0

    def reorder(self, slots, parents):
        """One request's beams; (code, {beam: (page from, page to, positions)})."""
        K, old = len(slots), self.copy()
        parents = [p if 0 <= p < K else k for k, p in enumerate(parents)]
        live = [s for s in slots if s >= 0]
        if len(set(live)) != len(live) or any(s >= len(self.table) for s in live):
            return 3, {}
        moved = [k for k in range(K) if parents[k] != k and slots[k] >= 0]
        if any(slots[parents[k]] < 0 for k in moved):
            return 3, {}
        own = {k: old.table[s][pages_of(old.lengths[s]) - 1] if s >= 0 and old.lengths[s] else None for k, s in enumerate(slots)}
        needs = [own[k] for k in moved if old.lengths[slots[parents[k]]] % PAGE]
        code = max([4 if page is None else 5 if old.refs[page] != 1 else 0 for page in needs] + [0])
        if code:
            return code, {}
        # a last page that is whole and that a child of the beam takes over cannot be filled by the beam too: it fills a page that the beams give
        # back, the last one of a beam that fills none and whose child does not take it, in order
        fills = [k for k in moved if old.lengths[slots[parents[k]]] % PAGE]
        taken = {parents[k] for k in moved if old.lengths[slots[parents[k]]] % PAGE == 0}
        lost = [k for k in fills if k in taken]
        spare = [own[k] for k in moved if k not in fills and k not in taken and own[k] is not None and old.refs[own[k]] == 1]
        if len(spare) < len(lost):
            return 5, {}
        copies = {}
        for k in moved:
            s, p = slots[k], slots[parents[k]]
            n, full, used = old.lengths[s], old.lengths[p] // PAGE, old.lengths[p] % PAGE
            for c in range(pages_of(n)):
                if not (used and c == pages_of(n) - 1):
                    self.refs[old.table[s][c]] -= 1
                self.table[s][c] = 0
            for c in range(full):
                self.table[s][c] = old.table[p][c]
                self.refs[old.table[p][c]] += 1
            if used:
                self.table[s][full] = own[k]
                copies[k] = (own[parents[k]], own[k], used)
            self.lengths[s] = old.lengths[p]
        for k, page in zip(lost, spare):
            source, mine, used = copies[k]
            self.refs[mine] -= 1
            self.refs[page] += 1
            self.table[slots[k]][old.lengths[slots[parents[k]]] // PAGE] = page
            copies[k] = (source, page, used)
        return 0, copies


def row_maps(table, slots, start, new, T, parents=None, keep=None, words=0):
    """cu, row_seq, positions, row_map, mask (signed 32-bit words)."""
    cu, width = [0], len(table[0])
    for n in new:
        cu.append(min(T, cu[-1] + max(0, n)))
    seq, pos, place, mask = [-1] * T, [0] * T, [-1] * T, [[0] * words for _ in range(T)]
    for b in range(len(new)):
        seen = []
        for i in range(cu[b + 1] - cu[b]):
            t, depth, ok = cu[b] + i, i, True
            if parents is not None:
                p = parents[t]
                up = (0, 0) if p == -1 else seen[p] if 0 <= p < i else None
                seen.append(None if up is None else (up[0] | 1 << i, up[1] + (p >= 0)))
                ok = seen[i] is not None
                depth = seen[i][1] if ok else 0
                bits = seen[i][0] if ok else 0
                mask[t] = [v - (1 << 32) if v >> 31 else v for v in ((bits >> 32 * w) & 0xFFFFFFFF for w in range(words))]
            seq[t], pos[t] = b, start[b] + depth
            stored = keep[t] if keep is not None else parents is None
            if ok and stored and 0 <= slots[b] < len(table) and pos[t] // PAGE < width:
                place[t] = table[slots[b]][pos[t] // PAGE] * PAGE + pos[t] % PAGE
    return cu, seq, pos, place, mask


def draft(rng, n):
    """Parents of n drafted rows, each a smaller index or -1."""
    return [rng.randint(max(-1, i - 6), i - 1) for i in range(n)]


def tree_sees(cu, start, positions, parents, context, window, T):
    """Per request: truth values [rows, context + rows]."""
    out = []
    for b in range(len(cu) - 1):
        n = cu[b + 1] - cu[b]
        at = torch.tensor(positions[cu[b]:cu[b + 1]])
        see = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            j = i
            while j >= 0:
                see[i, j] = True
                j = parents[cu[b] + j] if parents is not None else j - 1
        full = torch.cat([torch.ones(n, context[b], dtype=torch.bool), see], 1)
        if window:
            where = torch.cat([torch.arange(context[b]), at])
            full &= where[None, :] > at[:, None] - window
        out.append(full)
    return out


def tree_attention(q, k, v, sees, scale, softcap=0.0, sink=None):
    """One request in 64 bits: q [n, H, hd], k and v [keys, KV, hd], sees [n, keys] -> (o [n, H, hd], sum p |v|, sum |q| |k| scale at most).
    Keys that a row does not see contribute nothing, whatever they hold."""
    n, H, hd = q.shape
    KV = k.shape[1]
    o, a, s = torch.zeros(n, H, hd, dtype=torch.float64), torch.zeros(n, H, hd, dtype=torch.float64), torch.zeros(n, H, dtype=torch.float64)
    for h in range(H):
        for i in range(n):
            kk, vv = k[sees[i], h // (H // KV)].double(), v[sees[i], h // (H // KV)].double()
            z = kk @ q[i, h].double() * scale
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            if sink is not None:
                z = torch.cat([z, torch.tensor([float(sink[h])], dtype=torch.float64)])
            if not len(kk):
                continue
            p = torch.softmax(z, 0)[:len(kk)]
            o[i, h] = p @ vv
            a[i, h] = p @ vv.abs()
            s[i, h] = (kk.abs() @ q[i, h].double().abs()).max() * abs(scale)
    return o, a, s


def beam_select(logits, scores, n, ended=None, pad=0, placed=False):
    """One call in 64 bits, request by request: lists of tokens and parents, scores [R, n]."""
    R, K = scores.shape
    V = logits.shape[1]
    tokens, parents, values = [], [], []
    for r in range(R):
        c = torch.full((K, V), -math.inf, dtype=torch.float64)
        for k in range(K):
            s = float(scores[r, k])
            if not math.isfinite(s):
                continue
            if ended is not None and bool(ended[r, k]):
                c[k, pad] = s
                continue
            x = logits[r * K + k].double()
            top = x.max()
            lse = torch.log(torch.exp(x - top).sum())
            if torch.isfinite(lse):
                c[k] = s + ((x - top) - lse)
        flat = c.flatten()
        order = torch.sort(flat, descending=True, stable=True).indices[:n].tolist()
        if placed:
            at, later = {}, []
            for i in order:
                (later.append(i) if i // V in at else at.setdefault(i // V, i))
            for k in range(K):
                if k not in at:
                    at[k] = later.pop(0)
            order = [at[k] for k in range(K)]
        tokens.append([i % V for i in order])
        parents.append([i // V for i in order])
        values.append(flat[order])
    return tokens, parents, torch.stack(values)
