"""The operators of a decode step that verifies drafted tokens over a paged KV cache, as measured.

Five operators, in the order a step calls them: `tables` (block tables and the slot map of the
step's rows), `pack` (K and V rows into the paged cache), `attend` (attention of a tree of drafted
tokens over the cache), `shape` (penalties, biases and grammar masks on the logits, and the pick) and
`accept` (the drafted path that the picks confirm, its K and V moved together). `run` computes them
in elementary torch operations, or with `own` set through wavo_b200.

The listed sizes are those of a Whisper-turbo decoder (20 heads of 64, 4 layers, 448 positions, 1500
encoder frames, 51866 tokens, batches of 32) and generic longer ones with shared heads.
"""

import math
import zlib

import numpy as np
import torch

own = False

# A paged cache: [blocks][K, V][kv_heads][bs][hd] in f16. A slot is block * bs + offset.
# A tree: row i of a request sees the drafted rows whose bits its mask words hold (itself included).


def listed():
    turbo = {"heads": 20, "kv_heads": 20, "hd": 64, "bs": 16}
    return [
        # A verify step's plan: 32 segments with 16 drafted tokens each.
        {"name": "tables step", "op": "tables", "n": 32, "bs": 16, "max_len": 432, "max_add": 16,
         "release": 0.0, "short": False},
        # A large server: 2048 requests, prompts among the drafts, finished requests giving blocks
        # back, and a ring that runs short.
        {"name": "tables server", "op": "tables", "n": 2048, "bs": 16, "max_len": 8192,
         "max_add": 96, "release": 0.05, "short": True},
        # The drafted rows' K and V out of the f16 q|k|v rows of one layer, some rows padding.
        {"name": "pack step", "op": "pack", "rows": 512, "dtype": "f16", "kv_heads": 20, "hd": 64,
         "bs": 16, "before": 1280},
        # The encoder's K and V of 32 segments of 1500 frames, from the f32 projection.
        {"name": "pack cross", "op": "pack", "rows": 48000, "dtype": "f32", "kv_heads": 20,
         "hd": 64, "bs": 16, "before": 0},
        # Plain decoding: one token a segment over its own positions (f32 rows, the small-row form).
        {"name": "attend token", "op": "attend", "dtype": "f32", "n": 32, "rows": 1, "len": 448,
         "tree": False, **turbo},
        # Verification over the self cache: up to 64 drafted tokens a segment.
        {"name": "attend self", "op": "attend", "dtype": "f32", "n": 32, "rows": 64, "len": 384,
         "tree": True, **turbo},
        # Verification over the encoder frames: 16 drafted tokens share each segment's K and V.
        {"name": "attend cross", "op": "attend", "dtype": "f16", "n": 32, "rows": 16, "len": -1500,
         "tree": False, **turbo},
        # Two long requests with shared heads.
        {"name": "attend long", "op": "attend", "dtype": "f16", "n": 2, "rows": 24, "len": 131072,
         "tree": True, "heads": 32, "kv_heads": 8, "hd": 128, "bs": 32},
        # Plain decoding of 32 segments: penalties and biases, no grammar.
        {"name": "shape token", "op": "shape", "dtype": "f32", "n": 32, "rows": 1, "vocab": 51866,
         "hist": 224, "bias": 32, "grammars": 0},
        # A verify step: 16 drafted tokens a segment, a grammar state a row, long histories.
        {"name": "shape tree", "op": "shape", "dtype": "f32", "n": 32, "rows": 16, "vocab": 51866,
         "hist": 448, "bias": 200, "grammars": 64},
        # The commit after a verify step, and one of a larger batch with larger trees.
        {"name": "accept step", "op": "accept", "n": 32, "rows": 16, "len": 384, "layers": 4,
         "kv_heads": 20, "hd": 64, "bs": 16},
        {"name": "accept batch", "op": "accept", "n": 128, "rows": 64, "len": 384, "layers": 4,
         "kv_heads": 20, "hd": 64, "bs": 16},
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((20, 20, 64), (16, 16, 64), (32, 8, 128), (8, 1, 64), (12, 4, 80), (6, 2, 96), (5, 5, 40))


def draw(rng):
    op = rng.choice(("tables", "pack", "attend", "attend", "shape", "accept"))
    bs = rng.choice((8, 16, 32, 64))
    heads, kv_heads, hd = rng.choice(HEADS)
    dtype = rng.choice(("f16", "f32"))
    if op == "tables":
        return {"op": op, "n": log_int(rng, 1, 2048), "bs": bs, "max_len": log_int(rng, 16, 8192),
                "max_add": log_int(rng, 1, 96), "release": rng.choice((0.0, 0.1)),
                "short": rng.random() < 0.3}
    if op == "pack":
        most = min(48000, 48000 * 2560 // (2 * kv_heads * hd))
        return {"op": op, "rows": log_int(rng, 1, most), "dtype": dtype, "kv_heads": kv_heads,
                "hd": hd, "bs": bs, "before": rng.choice((0, heads * hd))}
    if op == "attend":
        n, rows = log_int(rng, 1, 64), log_int(rng, 1, 64)
        most = min(131072, 2 * 131072 * 1024 // (n * kv_heads * hd),
                   2 * 131072 * 24 * 32 // (n * rows * heads))
        return {"op": op, "dtype": dtype, "n": n, "rows": rows, "len": log_int(rng, 1, max(2, most)),
                "tree": rng.random() < 0.6, "heads": heads, "kv_heads": kv_heads, "hd": hd, "bs": bs}
    if op == "shape":
        vocab = log_int(rng, 500, 51866)
        n = log_int(rng, 1, 32)
        return {"op": op, "dtype": dtype, "n": n, "rows": log_int(rng, 1, 16), "vocab": vocab,
                "hist": log_int(rng, 1, 448), "bias": rng.choice((0, log_int(rng, 1, 200))),
                "grammars": rng.choice((0, log_int(rng, 1, 64)))}
    return {"op": op, "n": log_int(rng, 1, 128), "rows": log_int(rng, 1, 64),
            "len": log_int(rng, 1, 384), "layers": rng.randint(1, 4), "kv_heads": kv_heads,
            "hd": hd, "bs": bs}


TYPES = {"f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


def i32(a):
    return torch.as_tensor(np.ascontiguousarray(a, np.int32)).to(DEV)


def lengths(c):
    """The positions that each request holds and the rows that it brings: from the case, whatever
    the seed of the values, so that the outputs of a case have one shape. Trees and verify steps
    are ragged; single tokens, and the queries of a batch over the encoder frames, are not."""
    z = np.random.default_rng(zlib.crc32(repr(sorted(
        (k, v) for k, v in c.items() if k != "name")).encode()))
    n, most = c["n"], c.get("len", 1)
    lens = np.full(n, -most) if most < 0 else z.integers(most // 2 if most > 1024 else 1,
                                                         most + 1, n)
    if not c.get("tree", True):
        return lens, np.full(n, c["rows"])
    counts = z.integers(1, c["rows"] + 1, n)
    counts[int(z.integers(0, n))] = c["rows"]
    return lens, counts


def trees(r, counts, spread=3):
    """Random drafted trees, parents first: (words [rows][w], parent of each row in its tree)."""
    words = -(-int(max(counts)) // 32)
    mask = np.zeros((int(sum(counts)), words), np.uint32)
    parent = np.full(len(mask), -1, np.int64)
    at = 0
    for c in counts:
        for i in range(int(c)):
            if i:
                parent[at + i] = max(0, i - 1 - int(r.integers(0, spread)))
                mask[at + i] = mask[at + parent[at + i]]
            mask[at + i, i // 32] |= np.uint32(1) << np.uint32(i % 32)
        at += int(c)
    return mask, parent


def paged(r, lens, bs, spare=3):
    """A table of distinct random blocks that holds `lens` positions a request."""
    want = [-(-int(v) // bs) for v in lens]
    blocks, width = sum(want) + spare, max(max(want, default=0), 1)
    ids = r.permutation(blocks)
    table = np.zeros((len(want), width), np.int32)
    at = 0
    for s, w in enumerate(want):
        table[s, :w] = ids[at:at + w]
        at += w
    return table, blocks


def starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def prepare(case, seed):
    r = np.random.default_rng(seed)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case, "op": case["op"]}
    globals()["prepare_" + case["op"]](case, r, g, s)
    if own:
        s["pass"] = context().pass_()
        if case["op"] == "shape":
            from wavo_b200.gpu import LogitRules
            s["rules"] = LogitRules(
                case["vocab"], history=(s["history"], s["hist_len"]), penalties=s["penalties"],
                bias=s["bias"], grammar=s["grammar"],
                tree=(s["row_seq"], s["row_start"], s["tokens"], s["mask"]))
    return s


def context():
    """The program's one context on the GPU."""
    if "gpu" not in globals():
        from wavo_b200.gpu import Gpu
        globals()["gpu"] = Gpu(0)
    return globals()["gpu"]


def prepare_tables(c, r, g, s):
    n, bs = c["n"], c["bs"]
    lens = r.integers(0, c["max_len"] + 1, n)
    adds = r.integers(0, c["max_add"] + 1, n)
    adds[r.random(n) < c["release"]] = -1
    # A request owns what its tokens take, some a block more (drafts that were not accepted).
    owned = -(-lens // bs) + (r.random(n) < 0.3)
    width = -(-(c["max_len"] + c["max_add"]) // bs) + 1
    need = np.maximum(0, -(-(lens + np.maximum(adds, 0)) // bs) - owned)
    blocks = n * width
    free = int(need[adds >= 0].sum()) // 2 if c["short"] else blocks - int(owned.sum())
    ids = r.permutation(blocks).astype(np.int32)[:int(owned.sum()) + free]
    table = np.full((n, width), -1, np.int32)
    at = starts(owned)
    for q in range(n):
        table[q, :owned[q]] = ids[at[q]:at[q + 1]]
    ring = np.full(blocks, -1, np.int32)
    head = int(r.integers(0, blocks))
    ring[(head + np.arange(free)) % blocks] = ids[at[-1]:]
    rows = n * c["max_add"]
    s.update(bs=bs, lens=i32(lens), adds=i32(adds), owned=i32(owned), table=i32(table),
             ring=i32(ring), state=i32([head, free]), state_out=i32([0] * 4),
             owned_out=i32([0] * n), row_start=i32([0] * (n + 1)), row_seq=i32([0] * rows),
             slots=i32([0] * rows))


def prepare_pack(c, r, g, s):
    rows, bs, kvd = c["rows"], c["bs"], c["kv_heads"] * c["hd"]
    blocks = -(-rows // bs) + 4
    slots = r.permutation(blocks * bs)[:rows]
    slots[r.random(rows) < 0.02] = -1
    x = torch.randn(rows, c["before"] + 2 * kvd, generator=g, device=DEV).to(TYPES[c["dtype"]])
    # One block more than the cache has: what the plain form does with the rows that have no slot.
    pool = torch.zeros(blocks + 1, 2, c["kv_heads"], bs, c["hd"], dtype=torch.float16, device=DEV)
    s.update(x=x, slots=i32(slots), pool=pool, before=c["before"])


def prepare_attend(c, r, g, s):
    hd, bs = c["hd"], c["bs"]
    lens, counts = lengths(c)
    table, blocks = paged(r, lens + (counts if c["tree"] else 0), bs)
    pool = torch.randn(blocks, 2, c["kv_heads"], bs, hd, generator=g, device=DEV,
                       dtype=torch.float16)
    rows = int(counts.sum())
    q = torch.randn(rows, c["heads"] * hd, generator=g, device=DEV) * 1.5
    q = q.to(TYPES[c["dtype"]])
    mask, _ = trees(r, counts) if c["tree"] else (None, None)
    # What the host knows ahead of the lengths on the device: the longest a request can be.
    most = abs(c["len"]) + (c["rows"] if c["tree"] else 0)
    s.update(q=q, o=torch.empty_like(q), pool=pool, table=i32(table), lens=i32(lens),
             row_start=i32(starts(counts)), mask=None if mask is None else i32(mask.view(np.int32)),
             max_rows=c["rows"], max_len=min(most, table.shape[1] * bs), heads=c["heads"])


def prepare_shape(c, r, g, s):
    n, vocab = c["n"], c["vocab"]
    _, counts = lengths(c)
    rows = int(counts.sum())
    # Text repeats itself: tokens by a rank distribution.
    pick = lambda shape: np.minimum((vocab ** r.random(shape)).astype(np.int64), vocab) - 1  # noqa: E731
    hist = c["hist"]
    history = pick((n, hist))
    hist_len = r.integers(0, hist + 1, n)
    mask, _ = trees(r, counts)
    pen = np.stack([1 + 0.3 * r.random(n), 0.5 * r.random(n), 0.5 * r.random(n)], 1)
    bias = grammar = None
    if c["bias"]:
        most = min(c["bias"], vocab)
        ids = np.stack([r.choice(vocab, most, replace=False) for _ in range(n)])
        val = r.normal(0, 3, (n, most)).astype(np.float32)
        val[r.random((n, most)) < 0.1] = -np.inf
        bias = (i32(ids), torch.as_tensor(val).to(DEV), i32(r.integers(0, most + 1, n)))
    if c["grammars"]:
        words = -(-vocab // 32)
        bits = torch.randint(-2 ** 31, 2 ** 31, (c["grammars"], words), generator=g, device=DEV)
        # Some states allow a lot, some next to nothing.
        few = torch.rand(c["grammars"], words, generator=g, device=DEV) < 0.02
        bits[::2] = torch.where(few[::2], bits[::2], 0)
        grammar = (bits.to(torch.int32), i32(r.integers(-1, c["grammars"], rows)))
    logits = (3 * torch.randn(rows, vocab, generator=g, device=DEV)).to(TYPES[c["dtype"]])
    s.update(logits=logits, out=torch.empty_like(logits), vocab=vocab, history=i32(history),
             hist_len=i32(hist_len), penalties=torch.as_tensor(pen.astype(np.float32)).to(DEV),
             bias=bias, grammar=grammar, row_seq=i32(np.repeat(np.arange(n), counts)),
             row_start=i32(starts(counts)), tokens=i32(pick(rows)), mask=i32(mask.view(np.int32)),
             picks=i32([0] * rows), logprobs=torch.empty(rows, device=DEV))


def prepare_accept(c, r, g, s):
    n, bs = c["n"], c["bs"]
    lens, counts = lengths(c)
    table, blocks = paged(r, lens + counts, bs)
    mask, parent = trees(r, counts)
    rows = int(counts.sum())
    tokens = r.integers(0, 50000, rows)
    picks = r.integers(0, 50000, rows)
    first = np.repeat(starts(counts)[:-1], counts)
    child = np.flatnonzero((parent >= 0) & (r.random(rows) < 0.6))
    picks[first[child] + parent[child]] = tokens[child]
    pool = torch.randn(c["layers"], blocks, 2, c["kv_heads"], bs, c["hd"], generator=g, device=DEV,
                       dtype=torch.float16)
    s.update(picks=i32(picks), tokens=i32(tokens), mask=i32(mask.view(np.int32)),
             row_start=i32(starts(counts)), lens=i32(lens), table=i32(table), pool=pool,
             path=i32(np.zeros((n, c["rows"]))), count=i32([0] * n), next=i32([0] * n),
             new_lens=i32([0] * n))


def run(s):
    if own:
        return globals()["own_" + s["op"]](s, s["pass"])
    return globals()["plain_" + s["op"]](s)


# ---- through the framework -----------------------------------------------------------------------

def own_tables(s, p):
    p.block_tables(s["lens"], s["adds"], s["bs"], s["ring"], s["state"], s["owned"], s["table"],
                   s["row_start"], s["row_seq"], s["slots"], s["state_out"], s["owned_out"])
    return {k: s[k] for k in ("table", "ring", "row_start", "row_seq", "slots", "state_out",
                              "owned_out")}


def own_pack(s, p):
    pool = s["pool"][:-1]
    p.pack_slots(s["x"], (s["before"], s["x"].shape[1]), s["slots"], pool)
    return pool


def own_attend(s, p):
    p.attend_tree(s["q"], s["pool"], s["table"], s["lens"], s["o"], s["max_len"],
                  row_start=s["row_start"], mask=s["mask"], max_rows=s["max_rows"])
    return s["o"]


def own_shape(s, p):
    p.shape_logits(s["logits"], s["rules"], s["picks"], s["logprobs"], out=s["out"])
    return {"out": s["out"], "picks": s["picks"], "logprobs": s["logprobs"]}


def own_accept(s, p):
    p.tree_accept(s["picks"], s["tokens"], s["mask"], s["row_start"], s["lens"], s["table"],
                  s["pool"], s["path"], s["count"], s["next"], s["new_lens"])
    return {k: s[k] for k in ("path", "count", "next", "new_lens", "pool")}


# ---- the plain forms -----------------------------------------------------------------------------

def bits_of(words, width):
    """[.., w] words to [.., width] truth values, bit j % 32 of word j / 32 at j."""
    at = torch.arange(32, device=words.device, dtype=torch.int32)
    return ((words.unsqueeze(-1) >> at) & 1).flatten(-2)[..., :width].bool()


def plain_tables(s):
    bs, table, ring = s["bs"], s["table"], s["ring"]
    (n, width), cap = table.shape, ring.numel()
    lens, adds, owned = s["lens"].long(), s["adds"].long(), s["owned"].long()
    head, free = s["state"].long()
    add, back = adds.clamp(min=0), adds < 0
    want = (lens + add + bs - 1) // bs
    can = ~back & (want <= width)
    need = torch.where(can, (want - owned).clamp(min=0), 0)
    upto = need.cumsum(0)
    ok = can & ((need == 0) | (upto <= free))
    got = torch.where(ok, need, 0)
    col = torch.arange(width, device=table.device)
    # Blocks given back go to the ring's tail in request order.
    gone = torch.where(back, owned, 0)
    to = (head + free + (gone.cumsum(0) - gone)[:, None] + col) % cap
    more = torch.cat([ring, ring.new_zeros(1)])
    more.scatter_(0, torch.where(col < gone[:, None], to, cap).flatten(), table.flatten())
    # New blocks come from its head.
    new = (col >= owned[:, None]) & (col < (owned + got)[:, None])
    src = (head + (upto - need)[:, None] + col - owned[:, None]) % cap
    table.copy_(torch.where(new, ring[src], table))
    ring.copy_(more[:cap])
    ends = add.cumsum(0)
    row_start = torch.cat([ends.new_zeros(1), ends])
    r = torch.arange(s["slots"].numel(), device=table.device)
    live = r < ends[-1]
    seq = torch.searchsorted(ends, r, right=True).clamp(max=n - 1)
    pos = lens[seq] + r - row_start[seq]
    slot = table[seq, (pos // bs).clamp(max=width - 1)].long() * bs + pos % bs
    taken = got.sum()
    state = torch.stack([(head + taken) % cap, free - taken + gone.sum(), ends[-1],
                         (~ok & ~back).sum()])
    return {"table": table, "ring": ring, "row_start": row_start.int(),
            "row_seq": torch.where(live, seq, -1).int(),
            "slots": torch.where(live & ok[seq], slot, -1).int(),
            "state_out": state.int(), "owned_out": torch.where(back, 0, owned + got).int()}


def plain_pack(s):
    pool, x, slots = s["pool"], s["x"], s["slots"].long()
    _, _, kvh, bs, hd = pool.shape
    to = torch.where(slots >= 0, slots, (pool.shape[0] - 1) * bs)
    kv = x[:, s["before"]:].float().reshape(-1, 2, kvh, hd).half()
    pool[to // bs, :, :, to % bs] = kv
    return pool[:-1]


def plain_attend(s):
    q, pool, start = s["q"], s["pool"], s["row_start"].long()
    _, _, kvh, bs, hd = pool.shape
    n, heads, span = s["table"].shape[0], s["heads"], s["table"].shape[1] * pool.shape[3]
    lens, most = s["lens"].long(), s["max_rows"]
    kv = pool[s["table"].long()].float()  # [n][blocks][2][kvh][bs][hd]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, n, kvh, span, hd)
    i = torch.arange(most, device=q.device)
    j = torch.arange(span, device=q.device)
    row = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)
    seen = (j < lens[:, None])[:, None].expand(n, most, span)
    if s["mask"] is not None:
        bits = bits_of(s["mask"], 32 * s["mask"].shape[1])[row]  # [n][most][drafted]
        d = j - lens[:, None]
        there = (d >= 0) & (d < (start[1:] - start[:-1])[:, None])
        at = d.clamp(0, bits.shape[2] - 1)[:, None].expand(n, most, span)
        seen = seen | (there[:, None] & bits.gather(2, at))
    qs = q.float().reshape(-1, heads, hd)[row]  # [n][most][heads][hd]
    qs = qs.reshape(n, most, kvh, heads // kvh, hd).permute(0, 2, 3, 1, 4).reshape(
        n, kvh, heads // kvh * most, hd)
    x = (qs @ kv[0].transpose(2, 3)).reshape(n, kvh, heads // kvh, most, span) / math.sqrt(hd)
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = (x - torch.where(top == -math.inf, 0.0, top)).exp()
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    o = p.reshape(n, kvh, heads // kvh * most, span) @ kv[1]
    o = o.reshape(n, kvh, heads // kvh, most, hd).permute(0, 3, 1, 2, 4).reshape(n * most, heads * hd)
    r = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(start[1:].contiguous(), r, right=True)
    return o[seq * most + r - start[seq]].to(q.dtype)


def plain_shape(s):
    x, vocab, seq = s["logits"].float(), s["vocab"], s["row_seq"].long()
    hist, n = s["history"].long(), s["history"].shape[0]
    live = torch.arange(hist.shape[1], device=x.device) < s["hist_len"][:, None]
    c = torch.zeros(n, vocab + 1, device=x.device)
    c.scatter_add_(1, torch.where(live, hist, vocab), torch.ones_like(hist, dtype=torch.float32))
    c = c[seq]
    w = 32 * s["mask"].shape[1]
    on = bits_of(s["mask"], w)  # [rows][w]: the row's path
    at = (s["row_start"].long()[seq][:, None] + torch.arange(w, device=x.device)).clamp(
        max=x.shape[0] - 1)
    c.scatter_add_(1, torch.where(on, s["tokens"].long()[at], vocab), on.float())
    c = c[:, :vocab]
    rep, pres, freq = s["penalties"][seq].unsqueeze(-1).unbind(1)
    x = torch.where(c > 0, torch.where(x > 0, x / rep, x * rep) - (freq * c + pres), x)
    if s["bias"] is not None:
        ids, val, count = s["bias"]
        there = torch.arange(ids.shape[1], device=x.device) < count[:, None]
        b = torch.zeros(n, vocab + 1, device=x.device)
        b.scatter_(1, torch.where(there, ids.long(), vocab), val)
        x = x + b[seq, :vocab]
    if s["grammar"] is not None:
        words, of = s["grammar"]
        on = bits_of(words, vocab)[of.long().clamp(min=0)] | (of < 0)[:, None]
        x = x.masked_fill(~on, -math.inf)
    top = x.amax(-1)
    first = torch.where(x == top[:, None], torch.arange(vocab, device=x.device), vocab).amin(-1)
    dead = top == -math.inf
    total = (x - torch.where(dead, 0.0, top)[:, None]).exp().sum(-1)
    return {"out": x.to(s["out"].dtype), "picks": torch.where(dead, -1, first).int(),
            "logprobs": torch.where(dead, -math.inf, -total.log())}


def plain_accept(s):
    start, lens, mask, pool = s["row_start"].long(), s["lens"].long(), s["mask"], s["pool"]
    (n, most), bs = s["path"].shape, pool.shape[4]
    i = torch.arange(most, device=mask.device)
    there = i < (start[1:] - start[:-1])[:, None]
    row = (start[:-1, None] + i).clamp(max=mask.shape[0] - 1)
    tok, pick = s["tokens"].long()[row], s["picks"].long()[row]
    on = bits_of(mask, most)
    on = torch.nn.functional.pad(on, (0, most - on.shape[1]))[row] & there[:, :, None]  # [n][j][i]
    before = on & ~torch.eye(most, dtype=torch.bool, device=mask.device)
    # j's parent is the node whose own path is j's less j; of equal siblings the first counts.
    child = (before[:, :, None] == on[:, None]).all(-1) & there[:, None] & there[:, :, None]
    fits = (child & (tok[:, :, None] == pick[:, None])).any(-1)
    same = (before[:, :, None] == before[:, None]).all(-1) & (tok[:, :, None] == tok[:, None])
    later = (same & (i < i[:, None]) & there[:, None]).any(-1)
    good = (fits & ~later & on.diagonal(dim1=1, dim2=2)) | (i == 0)
    taken = ~(on & ~good[:, None]).any(-1) & there
    taken &= good & (on[:, :, 0] | (i == 0))
    path = torch.where(taken, i, most).sort(-1)[0]
    count = taken.sum(-1)
    live = path < most
    # Positions: the accepted nodes' to consecutive ones; every other entry copies onto itself.
    src = lens[:, None] + torch.where(live, path, 0)
    dst = lens[:, None] + torch.where(live, i, 0)
    blk = lambda pos: s["table"].long().gather(1, pos // bs)  # noqa: E731
    pool[:, blk(dst), :, :, dst % bs] = pool[:, blk(src), :, :, src % bs]
    last = path.gather(1, (count - 1).clamp(min=0)[:, None])
    return {"path": torch.where(live, path, -1).int(), "count": count.int(),
            "next": pick.gather(1, last.clamp(max=most - 1))[:, 0].int(),
            "new_lens": (lens + count).int(), "pool": pool}


# ---- what a pass cannot do without ---------------------------------------------------------------

SIZE = {"f16": 2, "f32": 4}


def work(c):
    op = c["op"]
    if op == "tables":
        rows = c["n"] * c["max_add"] / 2  # the mean of the drawn counts
        # Lengths, counts and owned blocks in and out; row_seq and slots; a table entry a block.
        return {"bytes": 20 * c["n"] + 8 * c["n"] * c["max_add"] + 8 * rows / c["bs"], "flops": 0}
    if op == "pack":
        kvd = c["kv_heads"] * c["hd"]
        return {"bytes": c["rows"] * (2 * kvd * (SIZE[c["dtype"]] + 2) + 4), "flops": 0}
    lens, counts = lengths(c)
    rows = int(counts.sum())
    if op == "attend":
        keys = lens + (counts if c["tree"] else 0)
        wide = c["heads"] * c["hd"]
        return {"bytes": int(keys.sum()) * 4 * c["kv_heads"] * c["hd"] +
                rows * 2 * wide * SIZE[c["dtype"]],
                "flops": 4 * int((keys * counts).sum()) * wide}
    if op == "shape":
        each = 2 * c["vocab"] * SIZE[c["dtype"]] + (c["vocab"] / 8 if c["grammars"] else 0)
        return {"bytes": rows * (each + 16) + c["n"] * (2 * c["hist"] + 4 * c["bias"]),
                "flops": 2 * rows * c["vocab"]}
    # The nodes off their place: about two of a tree's path, each read and written a layer.
    return {"bytes": rows * 12 + c["n"] * 2 * 2 * c["layers"] * 4 * c["kv_heads"] * c["hd"],
            "flops": 0}


# ---- in 64 bits, from the definitions ------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return exact_attend(s)
    if case["op"] == "shape":
        return exact_shape(s)
    if case["op"] == "pack":
        return exact_pack(s)
    if case["op"] == "accept":
        return exact_accept(s)
    return None  # whole numbers


def exact_pack(s):
    pool = s["pool"][:-1].double()
    _, _, kvh, bs, hd = pool.shape
    rows = s["x"][:, s["before"]:].double()
    there = torch.nonzero(s["slots"] >= 0)[:, 0]
    at = s["slots"].long()[there]
    for part in range(2):
        for h in range(kvh):
            lo = part * kvh * hd + h * hd
            pool[at // bs, part, h, at % bs] = rows[there, lo:lo + hd]
    return pool


def exact_attend(s):
    pool, start, lens = s["pool"], s["row_start"].tolist(), s["lens"].tolist()
    _, _, kvh, bs, hd = pool.shape
    group = s["heads"] // kvh
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    words = None if s["mask"] is None else s["mask"].cpu().numpy().view(np.uint32)
    for b, n in enumerate(lens):
        lo, hi = start[b], start[b + 1]
        drafted = hi - lo if words is not None else 0
        keys = n + drafted
        blocks = s["table"][b, :-(-keys // bs)].long()
        hidden = torch.zeros(hi - lo, keys, dtype=torch.bool, device=DEV)
        if drafted:
            bit = np.unpackbits(words[lo:hi].view(np.uint8), axis=1, bitorder="little")[:, :drafted]
            hidden[:, n:] = torch.as_tensor(bit == 0).to(DEV)
        for h in range(s["heads"]):
            k, v = (pool[blocks, part, h // group].reshape(-1, hd)[:keys].double()
                    for part in range(2))
            q = s["q"][lo:hi, h * hd:(h + 1) * hd].double()
            x = (q @ k.T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
            o[lo:hi, h * hd:(h + 1) * hd] = torch.softmax(x, -1) @ v
    return o


def exact_shape(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    logprobs = torch.empty(rows, dtype=torch.float64, device=DEV)
    start, seqs, lens = s["row_start"].tolist(), s["row_seq"].tolist(), s["hist_len"].tolist()
    words = s["mask"].cpu().numpy().view(np.uint32)
    on = np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")
    for r, b in enumerate(seqs):
        path = start[b] + np.flatnonzero(on[r])
        said = torch.cat([s["history"][b, :lens[b]], s["tokens"][torch.as_tensor(path).to(DEV)]])
        ids, count = torch.unique(said.long(), return_counts=True)
        rep, pres, freq = s["penalties"][b].double()
        v = x[r, ids]
        v = torch.where(v > 0, v / rep, v * rep)
        x[r, ids] = v - freq * count.double() - pres
        if s["bias"] is not None:
            k = int(s["bias"][2][b])
            x[r, s["bias"][0][b, :k].long()] += s["bias"][1][b, :k].double()
        if s["grammar"] is not None and int(s["grammar"][1][r]) >= 0:
            w = s["grammar"][0][int(s["grammar"][1][r])].cpu().numpy().view(np.uint8)
            off = np.unpackbits(w, bitorder="little")[:vocab] == 0
            x[r, torch.as_tensor(off).to(DEV)] = -math.inf
        top = x[r].max()
        logprobs[r] = top if top == -math.inf else top - torch.logsumexp(x[r], 0)
    return {"out": x, "picks": None, "logprobs": logprobs}


def exact_accept(s):
    start, lens, table = s["row_start"].tolist(), s["lens"].tolist(), s["table"].tolist()
    tokens, picks, bs = s["tokens"].tolist(), s["picks"].tolist(), s["pool"].shape[4]
    words = s["mask"].cpu().numpy().view(np.uint32)
    paths = [sum(int(w) << 32 * k for k, w in enumerate(row)) for row in words]
    src, dst = [], []
    for b, n in enumerate(lens):
        lo, hi = start[b], start[b + 1]
        node, depth = 0, 0
        while True:
            src.append((table[b][(n + node) // bs], (n + node) % bs))
            dst.append((table[b][(n + depth) // bs], (n + depth) % bs))
            said = picks[lo + node]
            node = next((j for j in range(node + 1, hi - lo) if tokens[lo + j] == said and
                         paths[lo + j] == paths[lo + node] | 1 << j), None)
            if node is None:
                break
            depth += 1
    pool = s["pool"].double()
    (sb, so), (db, do) = (torch.tensor(v, device=DEV).T for v in (src, dst))
    pool[:, db, :, :, do] = pool[:, sb, :, :, so]
    return {"path": None, "count": None, "next": None, "new_lens": None, "pool": pool}
