"""Paged caches and drafted trees on the GPU, against the plain 64-bit forms: block tables and slot
maps, K and V rows into the cache, attention of drafted tokens, logit rules and the pick, and the
commit of the drafted path; and what they refuse."""

import numpy as np
import pytest
import torch

import tree_reference as R

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def gpu():
    from wavo_b200.gpu import Gpu
    g = Gpu(0)
    yield g
    g.close()


def i32(a):
    return torch.as_tensor(np.ascontiguousarray(a).astype(np.int64).astype(np.int32)).cuda()


def words(mask):
    return torch.as_tensor(mask.view(np.int32)).cuda()


# ---- block tables --------------------------------------------------------------------------

def plan(gpu, lens, adds, bs, ring, state, owned, table, rows_cap):
    n = len(lens)
    t = {"ring": i32(ring), "table": i32(table), "row_start": i32([-7] * (n + 1)),
         "row_seq": i32([-7] * rows_cap), "slots": i32([-7] * rows_cap), "state_out": i32([-7] * 4),
         "owned_out": i32([-7] * n)}
    gpu.pass_().block_tables(i32(lens), i32(adds), bs, t["ring"], i32(state), i32(owned),
                             t["table"], t["row_start"], t["row_seq"], t["slots"],
                             t["state_out"], t["owned_out"])
    gpu.sync()
    return {k: v.cpu().numpy().tolist() for k, v in t.items()}


def tables_case(rng, n, bs, width, most, release=0.0, free=None, spare_cap=0):
    lens = rng.integers(0, width * bs + 1, n)
    adds = rng.integers(0, most + 1, n)
    adds[rng.random(n) < release] = -1
    owned = np.minimum(-(-lens // bs) + (rng.random(n) < 0.3), width)
    free = n * width - int(owned.sum()) if free is None else free
    cap = int(owned.sum()) + free + spare_cap
    cap = max(cap, 1)
    ids = rng.permutation(cap)[:int(owned.sum()) + free]
    table = np.full((n, width), -5)
    at = 0
    for s in range(n):
        table[s, :owned[s]] = ids[at:at + owned[s]]
        at += owned[s]
    head = int(rng.integers(0, cap))
    ring = np.full(cap, -9)
    ring[(head + np.arange(free)) % cap] = ids[at:]
    return lens, adds, bs, ring, [head, free], owned, table


@pytest.mark.parametrize("n,bs,width,most,release,free", [
    (1, 16, 4, 5, 0.0, None), (1, 8, 1, 0, 0.0, 0), (3, 256, 2, 300, 0.0, None),
    (32, 16, 30, 16, 0.0, None), (33, 16, 30, 40, 0.3, None), (300, 32, 9, 20, 0.2, 40),
    (300, 8, 6, 64, 0.1, 0), (1500, 16, 5, 70, 0.1, 900), (40000, 16, 3, 2, 0.2, 2500)])
def test_block_tables(gpu, n, bs, width, most, release, free):
    rng = np.random.default_rng(n + bs)
    case = tables_case(rng, n, bs, width, most, release, free, spare_cap=3)
    rows = int(np.maximum(case[1], 0).sum())
    for rows_cap in {rows + 700, max(rows // 2, 1), 0}:
        want = R.block_tables(*case, rows_cap)
        assert plan(gpu, *case, rows_cap) == {k: np.asarray(v).tolist() for k, v in want.items()}


def test_block_tables_one_long_prompt_and_everyone_done(gpu):
    rng = np.random.default_rng(5)
    case = list(tables_case(rng, 2, 16, 4096, 0))
    case[0], case[1] = np.array([7, 100]), np.array([60001, 3])
    case[5] = np.array([1, 7])
    case[6][:] = -5
    case[6][0, :1], case[6][1, :7] = 8000, np.arange(7001, 7008)
    case[3], case[4] = np.arange(8192), [8000, 5000]
    want = R.block_tables(*case, 70000)
    assert plan(gpu, *case, 70000) == {k: np.asarray(v).tolist() for k, v in want.items()}
    case[1] = np.array([-1, -1])
    want = R.block_tables(*case, 5)
    assert plan(gpu, *case, 5) == {k: np.asarray(v).tolist() for k, v in want.items()}


# ---- rows into the cache -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rows,kvh,hd,bs,src,extra", [
    (1, 1, 8, 8, 0, 0), (5, 3, 40, 16, 8, 8), (70, 20, 64, 16, 1280, 0), (33, 2, 128, 256, 1, 3),
    (300, 4, 80, 32, 4, 1), (2500, 5, 24, 64, 0, 5), (70001, 1, 16, 8, 0, 0)])
def test_pack_slots(gpu, dtype, rows, kvh, hd, bs, src, extra):
    rng = np.random.default_rng(rows)
    stride = src + 2 * kvh * hd + extra
    blocks = -(-rows // bs) + 2
    x = torch.randn(rows, stride, generator=torch.Generator().manual_seed(rows)) * 3
    x[0, src] = 1e6  # inf in f16, as any rounding to f16
    x = x.to(TYPES[dtype]).cuda()
    slots = rng.permutation(blocks * bs)[:rows]
    slots[rng.random(rows) < 0.1] = -1
    slots[rng.random(rows) < 0.05] = blocks * bs
    pool = torch.full((blocks, 2, kvh, bs, hd), 7.0, dtype=torch.float16, device="cuda")
    want = pool.clone()
    live = torch.as_tensor((slots >= 0) & (slots < blocks * bs)).cuda()
    at = torch.as_tensor(slots).cuda()[live]
    kv = x[:, src:src + 2 * kvh * hd].to(torch.float16).reshape(rows, 2, kvh, hd)[live]
    want[at // bs, :, :, at % bs] = kv
    gpu.pass_().pack_slots(x, (src, stride), i32(slots), pool)
    gpu.sync()
    assert torch.equal(pool.view(torch.int16), want.view(torch.int16))


# ---- attention -----------------------------------------------------------------------------

def attend_case(gpu, seed, dtype, counts, lens, heads, kvh, hd, bs, mask, width=0, strides=(0, 0),
                spoil=True, single=False, scale=1.5):
    """Runs a case and returns (output, 64-bit output, the bound's terms). `spoil`: NaN and infinities
    in every position that no row sees."""
    rng = np.random.default_rng(seed)
    t = sum(counts)
    table, blocks = R.paged(rng, [n + (c if mask is not None else 0) for n, c in zip(lens, counts)],
                            bs, width=width)
    pool = rng.standard_normal((blocks, 2, kvh, bs, hd)).astype(np.float16)
    used = np.zeros((blocks, bs), bool)
    for s, (n, c) in enumerate(zip(lens, counts)):
        for p in range(n + (c if mask is not None else 0)):
            used[table[s, p // bs], p % bs] = True
    if spoil:
        for b, i in np.argwhere(~used):
            pool[b, :, :, i] = rng.choice([np.nan, np.inf, -np.inf])
    q = (scale * rng.standard_normal((t, heads * hd))).astype(np.float16 if dtype == "f16" else np.float32)
    row_start = [0, *np.cumsum(counts).tolist()]
    wide = torch.zeros(t, heads * hd + strides[0], dtype=TYPES[dtype], device="cuda")
    qd = wide[:, strides[0]:]
    qd.copy_(torch.as_tensor(q))
    od = torch.full((t, heads * hd + strides[1]), 9.0, dtype=TYPES[dtype], device="cuda")
    gpu.pass_().attend_tree(
        qd, torch.as_tensor(pool).cuda(), i32(table), i32(lens), od[:, strides[1]:],
        max(n + c for n, c in zip(lens, counts)), row_start=None if single else i32(row_start),
        mask=None if mask is None else words(mask), max_rows=max(counts))
    gpu.sync()
    if strides[1]:
        assert (od[:, :strides[1]] == 9).all()
    want, terms = R.attend(q, pool, table, row_start, lens, mask, heads)
    return od[:, strides[1]:].double().cpu().numpy(), want, terms


def hold(got, want, terms, dtype):
    bound = R.attend_bound(want, terms, dtype == "f16")
    far = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (far <= bound).all(), (far.max(), (far / np.maximum(bound, 1e-30)).max())


HEADS = [(20, 20, 64), (8, 2, 128), (6, 1, 64), (3, 3, 40), (4, 2, 96), (2, 1, 8)]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", HEADS)
@pytest.mark.parametrize("bs", [8, 16, 64, 256])
def test_attend_tree(gpu, dtype, heads, kvh, hd, bs):
    rng = np.random.default_rng(heads * hd + bs)
    counts, lens = [5, 1, 17, 3, 8, 2], [70, 0, 200, 1, 15, 64]
    mask, _ = R.random_trees(rng, counts, 1)
    hold(*attend_case(gpu, 1, dtype, counts, lens, heads, kvh, hd, bs, mask), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 448, 1500])
def test_attend_tree_single_tokens(gpu, dtype, n):
    counts, lens = [1] * 4, [n, max(n - 1, 0), 1, 0]
    hold(*attend_case(gpu, n, dtype, counts, lens, 4, 4, 64, 16, None, single=True), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("t,group", [(2, 1), (15, 1), (16, 1), (17, 1), (33, 1), (64, 1), (65, 1),
                                     (100, 1), (256, 1), (3, 7), (16, 8), (40, 4)])
def test_attend_tree_sizes_of_trees(gpu, dtype, t, group):
    rng = np.random.default_rng(t)
    counts, lens = [t, 1, max(t // 2, 1)], [100, 33, 0]
    mask, _ = R.random_trees(rng, counts, -(-t // 32))
    hold(*attend_case(gpu, t, dtype, counts, lens, 2 * group, 2, 64, 16, mask), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attend_tree_any_mask_and_rows_that_see_nothing(gpu, dtype):
    rng = np.random.default_rng(3)
    counts, lens = [40, 7, 0, 64, 12], [0, 0, 5, 90, 0]
    mask = rng.integers(0, 2 ** 32, (sum(counts), 2), dtype=np.uint32)
    mask[rng.random(len(mask)) < 0.3] = 0
    mask[-12:] = 0
    got, want, terms = attend_case(gpu, 2, dtype, counts, lens, 4, 2, 64, 16, mask)
    hold(got, want, terms, dtype)
    assert (got[-12:] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kind", ["nan", "inf", "large"])
def test_attend_tree_branches_do_not_touch_one_another(gpu, dtype, kind):
    # One drafted row's K and V hold NaN, infinities or f16's largest values: rows that do not see
    # it keep their outputs to the bit, rows that see NaN get NaN.
    rng = np.random.default_rng(4)
    t, n, hd, bs = 20, 50, 64, 16
    mask, parent = R.random_trees(rng, [t], 1)
    table, blocks = R.paged(rng, [n + t], bs)
    pool = torch.as_tensor(rng.standard_normal((blocks, 2, 2, bs, hd)).astype(np.float16)).cuda()
    q = torch.as_tensor(rng.standard_normal((t, 2 * hd))).to(TYPES[dtype]).cuda()
    node = 4

    def go():
        o = torch.empty_like(q)
        gpu.pass_().attend_tree(q, pool, i32(table), i32([n]), o, n + t, row_start=i32([0, t]),
                                mask=words(mask), max_rows=t)
        gpu.sync()
        return o
    before = go()
    v = {"nan": float("nan"), "inf": float("inf"), "large": 65504.0}[kind]
    pool[table[0, (n + node) // bs], :, :, (n + node) % bs] = v
    after = go()
    blind = torch.as_tensor([not R.sees(m, node) for m in mask]).cuda()
    assert blind.sum() > 4 and (~blind).sum() > 2
    assert torch.equal(before[blind], after[blind])
    if kind == "nan":
        assert torch.isnan(after[~blind]).all()


# The kernel for many rows (more than 128 of a K and V head, or more than 32 over a long cache).

@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hd", [64, 128, 40])
def test_attend_tree_many_rows_any_mask(gpu, dtype, hd):
    rng = np.random.default_rng(30)
    counts, lens = [40, 7, 0, 64, 12, 1], [0, 0, 5, 90, 0, 700]
    mask = rng.integers(0, 2 ** 32, (sum(counts), 2), dtype=np.uint32)
    mask[rng.random(len(mask)) < 0.3] = 0
    mask[-13:-1] = 0
    got, want, terms = attend_case(gpu, 2, dtype, counts, lens, 16, 2, hd, 16, mask)
    hold(got, want, terms, dtype)
    assert (got[-13:-1] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd,n,t,bs", [
    (8, 1, 128, 5000, 12, 32), (6, 1, 64, 9001, 9, 8), (40, 4, 80, 1300, 20, 256), (5, 1, 64, 20000, 8, 64)])
def test_attend_tree_many_rows_long(gpu, dtype, heads, kvh, hd, n, t, bs):
    rng = np.random.default_rng(n)
    counts, lens = [t, 3, t // 2], [n, n // 3, 130]
    mask, _ = R.random_trees(rng, counts, 1)
    hold(*attend_case(gpu, n, dtype, counts, lens, heads, kvh, hd, bs, mask, spoil=n < 2000), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("strides", [(8, 8), (1, 3)])
def test_attend_tree_many_rows_strides(gpu, dtype, strides):
    rng = np.random.default_rng(31)
    counts, lens = [20, 4], [77, 300]
    mask, _ = R.random_trees(rng, counts, 1)
    hold(*attend_case(gpu, 6, dtype, counts, lens, 16, 2, 64, 16, mask, strides=strides), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kind", ["nan", "inf", "large"])
def test_attend_tree_many_rows_branches_do_not_touch_one_another(gpu, dtype, kind):
    rng = np.random.default_rng(32)
    t, n, hd, bs, heads = 20, 150, 64, 16, 16
    mask, _ = R.random_trees(rng, [t], 1)
    table, blocks = R.paged(rng, [n + t], bs)
    pool = torch.as_tensor(rng.standard_normal((blocks, 2, 2, bs, hd)).astype(np.float16)).cuda()
    q = torch.as_tensor(rng.standard_normal((t, heads * hd))).to(TYPES[dtype]).cuda()
    node = 4

    def go():
        o = torch.empty_like(q)
        gpu.pass_().attend_tree(q, pool, i32(table), i32([n]), o, n + t, row_start=i32([0, t]),
                                mask=words(mask), max_rows=t)
        gpu.sync()
        return o
    before = go()
    v = {"nan": float("nan"), "inf": float("inf"), "large": 65504.0}[kind]
    pool[table[0, (n + node) // bs], :, :, (n + node) % bs] = v
    after = go()
    blind = torch.as_tensor([not R.sees(m, node) for m in mask]).cuda()
    assert blind.sum() > 4 and (~blind).sum() > 2
    assert torch.equal(before[blind], after[blind])
    if kind == "nan":
        assert torch.isnan(after[~blind]).all()


def test_attend_tree_positions_past_max_len_are_not_seen(gpu):
    rng = np.random.default_rng(33)
    for heads, t in ((4, 3), (16, 20)):
        n, hd, bs, most = 300, 64, 16, 200
        table, blocks = R.paged(rng, [n], bs)
        pool = rng.standard_normal((blocks, 2, 2, bs, hd)).astype(np.float16)
        q = rng.standard_normal((t, heads * hd)).astype(np.float32)
        qd = torch.as_tensor(q).cuda()
        o = torch.empty_like(qd)
        gpu.pass_().attend_tree(qd, torch.as_tensor(pool).cuda(), i32(table), i32([n]), o, most,
                                row_start=i32([0, t]), max_rows=t)
        gpu.sync()
        want, terms = R.attend(q, pool, table, [0, t], [most], None, heads)
        hold(o.double().cpu().numpy(), want, terms, "f32")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd,n", [(8, 2, 128, 5000), (4, 4, 64, 9001), (1, 1, 64, 30000)])
def test_attend_tree_long(gpu, dtype, heads, kvh, hd, n):
    rng = np.random.default_rng(n)
    counts, lens = [6, 3], [n, n // 3]
    mask, _ = R.random_trees(rng, counts, 1)
    hold(*attend_case(gpu, n, dtype, counts, lens, heads, kvh, hd, 32, mask, spoil=False), dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("strides", [(0, 8), (8, 0), (1, 3), (128, 64)])
def test_attend_tree_strides(gpu, dtype, strides):
    rng = np.random.default_rng(9)
    counts, lens = [9, 4], [77, 20]
    mask, _ = R.random_trees(rng, counts, 1)
    hold(*attend_case(gpu, 6, dtype, counts, lens, 4, 2, 64, 16, mask, strides=strides), dtype)


def test_attend_tree_tables_wider_than_needed_and_entries_outside_the_pool(gpu):
    rng = np.random.default_rng(11)
    t, n, hd, bs = 3, 60, 64, 16
    table, blocks = R.paged(rng, [n + t], bs, width=9)
    table[0, 1] = blocks + 5   # positions 16..31: not in the pool, seen by nobody
    table[0, 5:] = -1
    pool = rng.standard_normal((blocks, 2, 2, bs, hd)).astype(np.float16)
    q = rng.standard_normal((t, 4 * hd)).astype(np.float32)
    mask, _ = R.random_trees(rng, [t], 1)
    qd = torch.as_tensor(q).cuda()
    o = torch.empty_like(qd)
    gpu.pass_().attend_tree(qd, torch.as_tensor(pool).cuda(), i32(table), i32([n]), o, n + t,
                            row_start=i32([0, t]), mask=words(mask), max_rows=t)
    gpu.sync()
    want, terms = R.attend(q, pool, table, [0, t], [n], mask, 4)
    hold(o.double().cpu().numpy(), want, terms, "f32")


def test_attend_tree_scores_far_apart(gpu):
    # Rows whose scores spread over hundreds: the running maximum carries the sums.
    rng = np.random.default_rng(12)
    mask, _ = R.random_trees(rng, [12, 3], 1)
    got, want, terms = attend_case(gpu, 8, "f32", [12, 3], [300, 40], 4, 4, 64, 16, mask, scale=60)
    hold(got, want, terms, "f32")


def test_attend_tree_a_pool_past_32_bits(gpu):
    # The last blocks of a pool of more than 2^32 bytes and 2^31 elements.
    kvh, hd, bs, n, t = 8, 128, 32, 100, 4
    blocks = (1 << 31) // (2 * kvh * bs * hd) + 40
    pool = torch.empty(blocks, 2, kvh, bs, hd, dtype=torch.float16, device="cuda")
    rng = np.random.default_rng(13)
    table, small = R.paged(rng, [n + t], bs, spare=0)
    part = rng.standard_normal((small, 2, kvh, bs, hd)).astype(np.float16)
    pool[-small:] = torch.as_tensor(part).cuda()
    mask, _ = R.random_trees(rng, [t], 1)
    q = rng.standard_normal((t, 16 * hd)).astype(np.float16)
    qd = torch.as_tensor(q).cuda()
    o = torch.empty_like(qd)
    p = gpu.pass_()
    p.attend_tree(qd, pool, i32(table + blocks - small), i32([n]), o, n + t, row_start=i32([0, t]),
                  mask=words(mask), max_rows=t)
    x = torch.randn(1, 2 * kvh * hd, device="cuda")
    p.pack_slots(x, (0, x.shape[1]), i32([blocks * bs - 1]), pool)
    gpu.sync()
    want, terms = R.attend(q, part, table, [0, t], [n], mask, 16)
    hold(o.double().cpu().numpy(), want, terms, "f16")
    assert torch.equal(pool[-1, :, :, -1].flatten(), x.half().flatten())


# ---- logit rules -----------------------------------------------------------------------------

def shape_case(gpu, seed, dtype, vocab, counts, hist, bias, grammars, tree=True, pen=True,
               pad=0, inplace=False, x=None, picks=True):
    from wavo_b200.gpu import LogitRules
    rng = np.random.default_rng(seed)
    n, rows = len(counts), sum(counts)
    ld = vocab + pad
    if x is None:
        x = 4 * rng.standard_normal((rows, ld))
    x = x.astype(np.float16 if dtype == "f16" else np.float32)
    row_start = [0, *np.cumsum(counts).tolist()]
    seq = np.repeat(np.arange(n), counts)
    mask, _ = R.random_trees(rng, counts, -(-max(counts) // 32))
    tokens = rng.integers(-2, vocab + 2, rows)
    history = rng.integers(-2, min(vocab, 40) + 2, (n, max(hist, 1)))
    hist_len = rng.integers(0, hist + 1, n)
    penalties = np.stack([1 + rng.random(n), rng.random(n), rng.random(n)], 1).astype(np.float32)
    ids = rng.integers(-2, min(vocab, 60) + 2, (n, max(bias, 1)))  # with repetitions
    vals = rng.normal(0, 3, ids.shape).astype(np.float32)
    vals[rng.random(ids.shape) < 0.1] = -np.inf
    count = rng.integers(0, bias + 1, n)
    words_n = -(-vocab // 32) + 1
    allow = rng.integers(0, 2 ** 32, (max(grammars, 1), words_n), dtype=np.uint32)
    allow[0] = 0  # a set that allows nothing
    of = rng.integers(-1, max(grammars, 1), rows)
    rules = LogitRules(
        vocab, n=n, history=(i32(history), i32(hist_len)) if hist else None,
        penalties=torch.as_tensor(penalties).cuda() if pen else None,
        bias=(i32(ids), torch.as_tensor(vals).cuda(), i32(count)) if bias else None,
        grammar=(words(allow), i32(of)) if grammars else None,
        tree=(i32(seq), i32(row_start), i32(tokens), words(mask)) if tree else None)
    xd = torch.as_tensor(x).cuda()
    out = xd if inplace else torch.full_like(xd, 9.0)
    pk = i32([-7] * rows)
    lp = torch.full((rows,), 7.0, device="cuda")
    gpu.pass_().shape_logits(xd, rules, pk if picks else None, lp if picks else None, out=out)
    gpu.sync()
    got = out.cpu().numpy()
    for r in range(rows):
        s = seq[r]
        said = list(history[s][:hist_len[s]]) if hist else []
        if tree:
            said += [tokens[row_start[s] + j] for j in range(counts[s]) if R.sees(mask[r], j)]
        ok = None
        if grammars and of[r] >= 0:
            ok = np.unpackbits(allow[of[r]].view(np.uint8), bitorder="little")[:vocab] == 1
        want, best, lprob = R.shape_logits(
            x[r].astype(np.float32), vocab, said, penalties[s] if pen else None,
            (ids[s][:count[s]], vals[s][:count[s]]) if bias else None, ok)
        assert np.array_equal(got[r, :vocab], want.astype(x.dtype), equal_nan=True), r
        if pad:
            assert np.array_equal(got[r, vocab:], x[r, vocab:] if inplace else got[r, vocab:] * 0 + 9)
        if picks:
            assert int(pk[r]) == best
            # The exponentials are good to 2^-21, their sum to a few more roundings.
            near = 2e-6 + 1e-6 * abs(lprob) if np.isfinite(lprob) else 0
            assert np.array_equal(float(lp[r]), lprob, equal_nan=True) or \
                abs(float(lp[r]) - lprob) <= near, (r, float(lp[r]), lprob)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [1, 31, 33, 500, 8191, 8192, 8193, 51866, 70001, 151936])
def test_shape_logits(gpu, dtype, vocab):
    shape_case(gpu, vocab, dtype, vocab, [3, 1, 5], 50, 30, 4)


@pytest.mark.parametrize("hist,bias,grammars,tree,pen", [
    (0, 0, 0, False, False), (20, 0, 0, False, True), (0, 9, 0, False, False),
    (0, 0, 3, False, False), (0, 0, 0, True, True), (300, 200, 0, True, True),
    (20, 0, 3, True, False)])
def test_shape_logits_each_rule(gpu, hist, bias, grammars, tree, pen):
    shape_case(gpu, 5, "f32", 3001, [1, 1, 1] if not tree else [40, 1, 2], hist, bias, grammars,
               tree, pen)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("pad", [0, 1, 8, 22])
@pytest.mark.parametrize("inplace", [False, True])
def test_shape_logits_strides_and_in_place(gpu, dtype, pad, inplace):
    shape_case(gpu, 6, dtype, 20002, [4, 2], 30, 10, 3, pad=pad, inplace=inplace)


def test_shape_logits_infinities_and_nan(gpu):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((6, 9000))
    x[0, 100] = np.nan                 # never picked
    x[1] = -np.inf                     # nothing left
    x[2, 5] = np.inf
    x[3, :] = -np.inf
    x[3, 8999] = -3.0                  # one token left
    x[4, :] = 1.0                      # ties: the lowest index
    x[5] = np.nan
    shape_case(gpu, 7, "f32", 9000, [1] * 6, 0, 0, 0, tree=False, pen=False, x=x)
    shape_case(gpu, 7, "f32", 9000, [2, 4], 40, 20, 3, x=x)


def test_shape_logits_picks_alone_long_history_and_padding(gpu):
    from wavo_b200.gpu import LogitRules
    rng = np.random.default_rng(8)
    vocab, hist = 5000, 40000
    x = torch.as_tensor(rng.standard_normal((4, vocab)).astype(np.float32)).cuda()
    history = rng.integers(0, 50, (2, hist))
    pen = torch.tensor([[1.2, 0.3, 0.01], [1.0, 0.0, 0.5]]).cuda()
    rules = LogitRules(vocab, history=(i32(history), i32([hist, 39999])), penalties=pen,
                       tree=(i32([0, 1, -1, 5]), i32([0, 1, 2]), i32([3, 4, 0, 0]),
                             i32(np.ones((4, 1)))))
    picks, lp = i32([5] * 4), torch.zeros(4, device="cuda")
    keep = x.clone()
    gpu.pass_().shape_logits(x, rules, picks, lp)
    gpu.sync()
    assert torch.equal(x, keep)
    for r, (n, t) in enumerate([(hist, 3), (39999, 4)]):
        _, best, _ = R.shape_logits(keep[r].cpu().numpy(), vocab, list(history[r][:n]) + [t],
                                    pen[r].tolist(), None, None)
        assert int(picks[r]) == best
    assert picks[2:].tolist() == [-1, -1] and lp[2:].tolist() == [-np.inf] * 2


# ---- the commit --------------------------------------------------------------------------------

def accept_case(gpu, seed, counts, lens, layers, kvh, hd, bs, chance=0.7, mask=None, repeat=False):
    rng = np.random.default_rng(seed)
    n, most = len(counts), max(counts)
    mw = -(-most // 32)
    made, parent = R.random_trees(rng, counts, mw)
    mask = made if mask is None else mask
    rows = sum(counts)
    tokens = rng.integers(0, 6 if repeat else 50000, rows)
    picks = rng.integers(0, 6 if repeat else 50000, rows)
    row_start = [0, *np.cumsum(counts).tolist()]
    for s in range(n):
        for r in range(row_start[s], row_start[s + 1]):
            if parent[r] >= 0 and rng.random() < chance:
                picks[row_start[s] + parent[r]] = tokens[r]
    table, blocks = R.paged(rng, [a + b for a, b in zip(lens, counts)], bs)
    pool = torch.randn(layers, blocks, 2, kvh, bs, hd, device="cuda").half()
    want = pool.clone()
    path, count = i32(np.full((n, most), -7)), i32([-7] * n)
    nxt, new = i32([-7] * n), i32([-7] * n)
    gpu.pass_().tree_accept(i32(picks), i32(tokens), words(mask), i32(row_start), i32(lens),
                            i32(table), pool, path, count, nxt, new)
    gpu.sync()
    longest = 0
    for s, (nodes, after) in enumerate(R.tree_accept(picks, tokens, mask, row_start, lens)):
        assert path[s].tolist() == nodes + [-1] * (most - len(nodes))
        assert (int(count[s]), int(nxt[s]), int(new[s])) == (len(nodes), after, lens[s] + len(nodes))
        longest = max(longest, len(nodes))
        moved = [want[:, table[s, (lens[s] + j) // bs], :, :, (lens[s] + j) % bs].clone()
                 for j in nodes]
        for k, kv in enumerate(moved):
            want[:, table[s, (lens[s] + k) // bs], :, :, (lens[s] + k) % bs] = kv
    assert torch.equal(pool.view(torch.int16), want.view(torch.int16))
    return longest


@pytest.mark.parametrize("counts,lens,layers,kvh,hd,bs", [
    ([1], [0], 1, 1, 8, 8), ([16, 1, 0, 9], [40, 0, 3, 15], 2, 20, 64, 16),
    ([64] * 5, [100, 1, 2, 3, 4], 4, 3, 40, 8), ([256, 100], [7, 300], 1, 2, 128, 256),
    ([33] * 40, [11] * 40, 3, 5, 24, 32)])
def test_tree_accept(gpu, counts, lens, layers, kvh, hd, bs):
    accept_case(gpu, sum(counts), counts, lens, layers, kvh, hd, bs)
    accept_case(gpu, sum(counts), counts, lens, layers, kvh, hd, bs, repeat=True)


def test_tree_accept_a_whole_chain_and_no_child(gpu):
    chain = np.zeros((256, 8), np.uint32)
    for i in range(256):
        chain[i] = chain[i - 1] if i else 0
        chain[i, i // 32] |= np.uint32(1 << (i % 32))
    assert accept_case(gpu, 1, [256], [50], 2, 2, 64, 16, chance=0.0, mask=chain) == 1
    # Every pick is the next token: the whole chain, nothing to move.
    tokens = np.arange(256)
    picks = tokens + 1
    path, count, nxt, new = i32(np.zeros((1, 256))), i32([0]), i32([0]), i32([0])
    gpu.pass_().tree_accept(i32(picks), i32(tokens), words(chain), i32([0, 256]), i32([9]), None,
                            None, path, count, nxt, new)
    gpu.sync()
    assert path[0].tolist() == list(range(256))
    assert (int(count), int(nxt), int(new)) == (256, 256, 265)


def test_tree_accept_rows_that_are_not_on_their_own_path(gpu):
    mask = np.zeros((6, 1), np.uint32)
    mask[:, 0] = [1, 1, 3, 2, 0, 33]   # rows 1, 2 and 4 lack their own bit
    accept_case(gpu, 3, [6], [4], 1, 1, 8, 8, mask=mask, repeat=True)


# ---- streams, graphs, refusals ----------------------------------------------------------------

def test_on_another_stream_and_in_a_graph(gpu):
    rng = np.random.default_rng(20)
    n, t, bs, hd, heads = 3, 6, 16, 64, 4
    lens = [20, 5, 33]
    width = 4
    ring, state = i32(np.arange(12)[::-1].copy()), i32([0, 12])
    owned, table = i32([0] * n), i32(np.full((n, width), -1))
    total = [a + t for a in lens]
    row_start, row_seq, slots = i32([0] * (n + 1)), i32([0] * 90), i32([0] * 90)
    state_out, owned_out = i32([0] * 4), i32([0] * n)
    pool = torch.zeros(12, 2, heads, bs, hd, dtype=torch.float16, device="cuda")
    x = torch.randn(90, 2 * heads * hd, device="cuda")
    q = torch.randn(n * t, heads * hd, device="cuda")
    o = torch.empty_like(q)
    mask, _ = R.random_trees(rng, [t] * n, 1)
    m, starts, ln, add, zero = words(mask), i32([0, t, 2 * t, 3 * t]), i32(lens), i32(total), i32([0] * n)

    def record(p):
        p.block_tables(zero, add, bs, ring, state, owned, table, row_start, row_seq, slots,
                       state_out, owned_out)
        p.pack_slots(x, (0, x.shape[1]), slots, pool)
        p.attend_tree(q, pool, table, ln, o, 64, row_start=starts, mask=m, max_rows=t)
    record(gpu.pass_())
    gpu.sync()
    first = o.clone()
    want, terms = R.attend(q.cpu().numpy(), pool.cpu().numpy(), table.cpu().numpy(),
                           [0, t, 2 * t, 3 * t], lens, mask, heads)
    hold(first.double().cpu().numpy(), want, terms, "f32")
    side = torch.cuda.Stream()
    o.zero_()
    side.wait_stream(torch.cuda.current_stream())
    gpu.use_stream(side)
    record(gpu.pass_())
    gpu.sync()
    gpu.use_stream(torch.cuda.current_stream())
    assert torch.equal(o, first)
    g = gpu.capture(record)
    o.zero_()
    g.launch()
    g.launch()
    gpu.sync()
    assert torch.equal(o, first)


@pytest.mark.parametrize("heads,t", [(4, 3), (32, 24)])   # one kernel of the attention each
def test_scratch_before_a_capture(heads, t):
    from wavo_b200 import WavoError
    from wavo_b200.gpu import Gpu
    rng = np.random.default_rng(21)
    n, hd, kvh, bs, most = 2, 64, 4, 16, 6000
    lens, rows = [5000, 700], 2 * t
    mask, _ = R.random_trees(rng, [t] * n, 1)
    table, blocks = R.paged(rng, [a + t for a in lens], bs)
    pool = torch.randn(blocks, 2, kvh, bs, hd, device="cuda").half()
    q = torch.randn(rows, heads * hd, device="cuda").half()
    want, o = torch.empty_like(q), torch.empty_like(q)
    tb, ln, starts, m = i32(table), i32(lens), i32([0, t, rows]), words(mask)
    g = Gpu(0)
    go = lambda p, to: p.attend_tree(q, pool, tb, ln, to, most, row_start=starts, mask=m,  # noqa: E731
                                     max_rows=t)
    with pytest.raises(WavoError, match="wavo_reserve"):
        g.capture(lambda p: go(p, o))
    need = g.attend_tree_scratch(n, rows, t, most, heads, kvh, hd)
    assert need > 0
    g.reserve(need)
    graph = g.capture(lambda p: go(p, o))
    go(g.pass_(), want)
    graph.launch()
    g.sync()
    assert torch.equal(o, want)
    ref, terms = R.attend(q.cpu().numpy(), pool.cpu().numpy(), table, [0, t, rows], lens, mask, heads)
    hold(o.double().cpu().numpy(), ref, terms, "f16")
    del graph
    g.close()


def refused(gpu, call, what):
    from wavo_b200 import WavoError, _lib as L
    with pytest.raises(WavoError) as e:
        call()
    assert e.value.status == L.EINVAL and what in str(e.value)


def test_refusals(gpu):
    from wavo_b200 import _lib as L
    from wavo_b200.gpu import LogitRules
    p = gpu.pass_()
    one, two = i32([1]), i32([0, 1])
    pool = torch.zeros(2, 2, 2, 16, 64, dtype=torch.float16, device="cuda")
    q = torch.zeros(1, 128, device="cuda")
    # Block tables.
    four = i32([0] * 4)
    refused(gpu, lambda: p.block_tables(one, one, 12, four, two, one, i32([[0, 0]]), two, one, one,
                                        four.clone(), i32([0])), "block_tables")
    refused(gpu, lambda: p.block_tables(one, one, 16, four, two, one, i32([[0, 0]]), two, one, one,
                                        four.clone(), one), "of their own")
    with pytest.raises(ValueError):
        p.block_tables(one, two, 16, four, two, one, i32([[0]]), two, one, one, four, i32([0]))
    with pytest.raises(TypeError):
        p.block_tables(one.long(), one, 16, four, two, one, i32([[0]]), two, one, one, four, one)
    # Rows into the cache: positions a block, head size, a stride below a row, too few rows.
    for bad in (torch.zeros(2, 2, 2, 12, 64), torch.zeros(2, 2, 2, 16, 60),
                torch.zeros(2, 2, 2, 512, 64), torch.zeros(1, 2, 1, 16, 136)):
        bad = bad.half().cuda()
        refused(gpu, lambda: p.pack_slots(torch.zeros(1, 600, device="cuda"), (0, 600), one, bad),
                "pack_slots: pool")
        refused(gpu, lambda: p.attend_tree(torch.zeros(1, bad.shape[2] * bad.shape[4], device="cuda"),
                                           bad, i32([[0]]), one,
                                           torch.zeros(1, bad.shape[2] * bad.shape[4], device="cuda"),
                                           16), "attend_tree: pool")
    refused(gpu, lambda: p.pack_slots(torch.zeros(9, 256, device="cuda"), (0, 255), two, pool),
            "stride 255")
    with pytest.raises(ValueError):
        p.pack_slots(torch.zeros(1, 256, device="cuda"), (0, 256), two, pool)
    with pytest.raises(TypeError):
        p.pack_slots(q, (0, 128), one, pool.float())
    # Attention: heads that do not share evenly, mask words, rows without starts.
    refused(gpu, lambda: p.attend_tree(torch.zeros(1, 192, device="cuda"), pool, i32([[0]]), one,
                                       torch.zeros(1, 192, device="cuda"), 16), "3 heads over 2")
    o = torch.zeros_like(q)
    m1 = torch.zeros(40, 1, dtype=torch.int32, device="cuda")
    q40 = torch.zeros(40, 128, device="cuda")
    refused(gpu, lambda: p.attend_tree(q40, pool, i32([[0]]), one, torch.zeros_like(q40), 16,
                                       row_start=i32([0, 40]), mask=m1, max_rows=33), "mask words")
    refused(gpu, lambda: p.attend_tree(q40, pool, i32([[0]]), one, torch.zeros_like(q40), 16,
                                       max_rows=2), "without row_start")
    with pytest.raises(ValueError):
        p.attend_tree(q, pool, i32([[0]]), one, o.half(), 16)
    with pytest.raises(TypeError):
        p.attend_tree(q, pool[:, :, :, ::2], i32([[0]]), one, o, 16)
    # Logit rules.
    x = torch.zeros(2, 100, device="cuda")
    refused(gpu, lambda: p.shape_logits(x, LogitRules(100, n=1), i32([0, 0])), "without row_seq")
    refused(gpu, lambda: p.shape_logits(x, LogitRules(100, history=(i32(np.zeros((2, 66000))),
                                                                    i32([0, 0]))), None), "66000 tokens")
    refused(gpu, lambda: p.shape_logits(x, LogitRules(100, n=2, grammar=(i32([[0, 0, 0]]),
                                                                         i32([0, 0]))), None),
            "3 grammar words")
    with pytest.raises(ValueError):
        LogitRules(100, n=2, penalties=torch.ones(3, 3, device="cuda"))
    with pytest.raises(ValueError):
        p.shape_logits(x, LogitRules(101, n=2), None)
    refused(gpu, lambda: L.check(L.lib().wavo_shape_logits(
        gpu.ctx, x.data_ptr(), 7, 0, None, 0, 2, LogitRules(100, n=2).c, None, None), gpu.ctx),
        "dtype 7")
    # The commit.
    new = i32([0])
    refused(gpu, lambda: p.tree_accept(one, one, i32([[1]]), two, one, None, None, i32([[0] * 33]),
                                       i32([0]), i32([0]), new), "33 rows")
    refused(gpu, lambda: p.tree_accept(one, one, i32([[1]]), two, one, None, None, i32([[0]]),
                                       i32([0]), i32([0]), one), "of its own")
    refused(gpu, lambda: p.tree_accept(one, one, i32([[1]]), two, one, i32([[0]]),
                                       torch.zeros(1, 1, 2, 1, 16, 4, device="cuda").half(),
                                       i32([[0]]), i32([0]), i32([0]), new), "tree_accept: pool")
    gpu.sync()
    # Nothing to do is not an error.
    none = i32([])
    p.pack_slots(q, (0, 256), none, pool)
    gpu.sync()
