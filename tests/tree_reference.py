"""Plain 64-bit forms of the operators over paged caches and drafted trees, one request and one row
at a time, for the tests."""

import math

import numpy as np


def block_tables(lens, adds, bs, ring, state, owned, table, rows_cap):
    """The plan of a step, request by request. Returns a dict of what the call writes."""
    ring, table, owned = list(ring), [list(t) for t in table], list(owned)
    cap, width = len(ring), len(table[0])
    head, free = int(state[0]), int(state[1])
    tail, upto, refused, given = head + free, 0, 0, 0
    row_start, row_seq, slots = [0], [], []
    for s, (n, add) in enumerate(zip(map(int, lens), map(int, adds))):
        if add < 0:
            for b in table[s][:owned[s]]:
                ring[tail % cap] = b
                tail += 1
            owned[s] = 0
            row_start.append(row_start[-1])
            continue
        want = -(-(n + add) // bs)
        ok = want <= width
        if ok:
            need = max(0, want - owned[s])
            upto += need
            ok = need == 0 or upto <= free
            if ok:
                for _ in range(need):
                    table[s][owned[s]] = ring[(head + given) % cap]
                    owned[s] += 1
                    given += 1
        refused += not ok
        for i in range(add):
            row_seq.append(s)
            slots.append(table[s][(n + i) // bs] * bs + (n + i) % bs if ok else -1)
        row_start.append(row_start[-1] + add)
    rows = len(slots)
    pad = [-1] * max(0, rows_cap - rows)
    return {"table": table, "ring": ring, "owned_out": owned, "row_start": row_start,
            "row_seq": (row_seq + pad)[:rows_cap], "slots": (slots + pad)[:rows_cap],
            "state_out": [(head + given) % cap, free - given + tail - head - free, rows, refused]}


def position(pool, table, p):
    """(block, offset) of position p of a request with this table, None if it is not in the pool."""
    bs = pool.shape[-2]
    if p // bs >= len(table):
        return None
    b = int(table[p // bs])
    return (b, p % bs) if 0 <= b < pool.shape[-5] else None


def sees(words, j):
    return j // 32 < len(words) and bool(int(words[j // 32]) >> (j % 32) & 1)


def attend(q, pool, table, row_start, lens, mask, heads):
    """f64 outputs of every row, and what a bound on their error needs: sum p|v|, the largest
    sum |q k| / sqrt(hd), sum |k| / sqrt(hd) (largest) and sum |v| / sum e over what a row sees."""
    _, _, kvh, _, hd = pool.shape
    group = heads // kvh
    rows = q.shape[0]
    o = np.zeros((rows, heads, hd))
    size = np.zeros((rows, heads, hd))
    qk = np.zeros((rows, heads, 1))
    k1 = np.zeros((rows, heads, 1))
    flat = np.zeros((rows, heads, hd))
    seen_keys = 0
    for s, n in enumerate(lens):
        for r in range(row_start[s], row_start[s + 1]):
            t = row_start[s + 1] - row_start[s]
            pos = list(range(n))
            if mask is not None:
                pos += [n + j for j in range(t) if sees(mask[r], j)]
            at = [a for a in (position(pool, table[s], p) for p in pos) if a is not None]
            if not at:
                continue
            seen_keys = max(seen_keys, len(at))
            b, i = map(list, zip(*at))
            for h in range(heads):
                k = pool[b, 0, h // group, i].astype(np.float64)
                v = pool[b, 1, h // group, i].astype(np.float64)
                x = k @ q[r, h * hd:(h + 1) * hd].astype(np.float64) / math.sqrt(hd)
                e = np.exp(x - x.max())
                p = e / e.sum()
                o[r, h] = p @ v
                size[r, h] = p @ np.abs(v)
                qk[r, h] = (np.abs(k) @ np.abs(q[r, h * hd:(h + 1) * hd])).max() / math.sqrt(hd)
                k1[r, h] = np.abs(k).sum(1).max() / math.sqrt(hd)
                flat[r, h] = np.abs(v).sum(0) / e.sum()
    shape = (rows, heads * hd)
    return o.reshape(shape), {"size": size.reshape(shape), "flat": flat.reshape(shape), "qk": np.repeat(
        qk, hd, 2).reshape(shape), "k1": np.repeat(k1, hd, 2).reshape(shape), "keys": seen_keys, "hd": hd}


def attend_bound(o, b, f16):
    """How far an output may be from the 64-bit one. A score is a sum of hd products in f32 (2^-23 a
    step allows for truncating adders), its exponential good to 2^-21, and a relative error of p
    moves o by at most twice that of sum p|v|; the sum over keys takes 16 products at a time, one
    addition a step. f16: the probability and the output are rounded once each (2^-11). f32: q and p
    enter as two f16 parts, whose rest is below 2^-22 of the value or 2^-25 where it is subnormal."""
    score = (b["hd"] + 4) * 2.0 ** -23 * b["qk"]
    sums = (b["keys"] / 16 + 20) * 2.0 ** -23
    if f16:
        return 2.0 ** -11 * (np.abs(o) + b["size"]) * 1.01 + b["size"] * (2 * score + 2.0 ** -20 + sums) + \
            2.0 ** -25 * (1 + b["flat"])
    score = score + 2.0 ** -22 * b["qk"] + 2.0 ** -25 * b["k1"]
    return 2.0 ** -23 * np.abs(o) + b["size"] * (2 * score + 2.0 ** -20 + sums) + 2.0 ** -25 * b["flat"]


def shape_logits(x, vocab, said, pen, bias, allow):
    """One row: x f32 [vocab]; said: the tokens before it; pen (repetition, presence, frequency) or
    None; bias (ids, values) or None; allow bool [vocab] or None. Every step rounded to f32."""
    f = np.float32
    x = np.array(x[:vocab], dtype=f)
    with np.errstate(over="ignore", invalid="ignore"):
        if pen is not None:
            rep, pres, freq = map(f, pen)
            ids, count = np.unique([t for t in said if 0 <= t < vocab], return_counts=True)
            for t, c in zip(ids.astype(int), count):
                v = f(x[t] / rep) if x[t] > 0 else f(x[t] * rep)
                x[t] = f(v - f(f(freq * f(c)) + pres))
        if bias is not None:
            last = {int(i): f(v) for i, v in zip(*bias) if 0 <= i < vocab}
            for t, v in last.items():
                x[t] = f(x[t] + v)
    if allow is not None:
        x[~allow] = -np.inf
    best, top = -1, -np.inf
    live = x[~np.isnan(x)]
    if live.size and live.max() > -np.inf:
        top = live.max()
        best = int(np.flatnonzero(x == top)[0])
    if best < 0:
        lp = np.nan if np.isnan(x).any() else -np.inf
    else:
        with np.errstate(invalid="ignore"):
            lp = -np.log(np.exp(x.astype(np.float64) - np.float64(top)).sum())
    return x, best, lp


def tree_accept(picks, tokens, mask, row_start, lens):
    """(path, next) of each request, by the walk."""
    out = []
    for s in range(len(lens)):
        lo, hi = row_start[s], row_start[s + 1]
        word = [sum(int(w) << 32 * k for k, w in enumerate(row)) for row in mask[lo:hi]]
        path, after = [], -1
        node = 0 if hi > lo else None
        while node is not None:
            path.append(node)
            after = int(picks[lo + node])
            node = next((j for j in range(node + 1, hi - lo) if tokens[lo + j] == after and
                         word[j] ^ (1 << j) == word[node]), None)
        out.append((path, after))
    return out


def random_trees(rng, counts, words, spread=3):
    """Mask words of random drafted trees, parents first, and each row's parent."""
    mask = np.zeros((int(sum(counts)), words), np.uint32)
    parent, at = [], 0
    for c in counts:
        for i in range(c):
            p = max(0, i - 1 - int(rng.integers(0, spread))) if i else -1
            parent.append(p)
            if i:
                mask[at + i] = mask[at + p]
            mask[at + i, i // 32] |= np.uint32(1) << np.uint32(i % 32)
        at += c
    return mask, parent


def paged(rng, lens, bs, spare=3, width=0):
    """Tables of distinct random blocks holding `lens` positions a request, and the blocks."""
    want = [-(-n // bs) for n in lens]
    blocks = sum(want) + spare
    ids = list(rng.permutation(blocks))
    table = np.zeros((len(lens), max(max(want), width, 1)), np.int32)
    for s, w in enumerate(want):
        table[s, :w] = [ids.pop() for _ in range(w)]
    return table, blocks
