"""The attention kernel for many rows on the GPU over many tiles and items a CTA, against the 64-bit
form: its rings, item changes, references that rise late, and infinities in one item after another."""

import math

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


def attend64(q, pool, table, row_start, lens, mask, heads):
    """tree_reference.attend in torch's 64 bits, a request at a time: the outputs and the terms of
    its bound, all on the GPU."""
    _, _, kvh, bs, hd = pool.shape
    rows, group = q.shape[0], heads // kvh
    names = ("o", "size", "flat", "qk", "k1")
    out = {k: torch.zeros(rows, heads, hd, dtype=torch.float64, device="cuda") for k in names}
    most = 0
    for s, n in enumerate(lens):
        lo, hi = row_start[s], row_start[s + 1]
        t = hi - lo
        keys = n + (t if mask is not None else 0)
        if t == 0 or keys == 0:
            continue
        see = torch.ones(t, keys, dtype=torch.bool, device="cuda")
        if mask is not None:
            bit = np.unpackbits(np.ascontiguousarray(mask[lo:hi]).view(np.uint8), axis=1,
                                bitorder="little")[:, :t]
            see[:, n:] = torch.as_tensor(bit == 1).cuda()
        most = max(most, int(see.sum(1).max()))
        blocks = torch.as_tensor(table[s, :-(-keys // bs)]).long().cuda()
        kv = pool[blocks].permute(1, 2, 0, 3, 4).reshape(2, kvh, -1, hd)[:, :, :keys].double()
        for h in range(heads):
            k, v = kv[0, h // group], kv[1, h // group]
            qh = q[lo:hi, h * hd:(h + 1) * hd].double()
            x = (qh @ k.T / math.sqrt(hd)).masked_fill(~see, -math.inf)
            top = x.amax(1, keepdim=True)
            e = (x - torch.where(top == -math.inf, 0.0, top)).exp()
            total = e.sum(1, keepdim=True)
            p = e / torch.where(total == 0, 1.0, total)
            off = ~see
            out["o"][lo:hi, h] = p @ v
            out["size"][lo:hi, h] = p @ v.abs()
            out["flat"][lo:hi, h] = see.double() @ v.abs() / torch.where(total == 0, 1.0, total)
            out["qk"][lo:hi, h] = (qh.abs() @ k.abs().T / math.sqrt(hd)).masked_fill(off, 0).amax(
                1, keepdim=True)
            out["k1"][lo:hi, h] = (k.abs().sum(1) / math.sqrt(hd)).expand(t, keys).masked_fill(
                off, 0).amax(1, keepdim=True)
    flat = {k: v.reshape(rows, -1).cpu().numpy() for k, v in out.items()}
    return flat.pop("o"), {**flat, "keys": most, "hd": hd}


def make(seed, dtype, counts, lens, heads, kvh, hd, bs, tree=True):
    """Device inputs of a case: q, pool, table, row starts, mask."""
    rng = np.random.default_rng(seed)
    mask = R.random_trees(rng, counts, max(1, -(-max(counts) // 32)))[0] if tree else None
    table, blocks = R.paged(rng, [n + c * tree for n, c in zip(lens, counts)], bs)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    pool = torch.randn(blocks, 2, kvh, bs, hd, generator=g, device="cuda", dtype=torch.float16)
    q = (1.5 * torch.randn(sum(counts), heads * hd, generator=g, device="cuda")).to(TYPES[dtype])
    return q, pool, table, [0, *np.cumsum(counts).tolist()], mask


def attend(gpu, q, pool, table, starts, lens, mask, counts, times=1):
    """The outputs, which have to be the same every time."""
    first = None
    args = i32(table), i32(lens)
    kw = dict(row_start=i32(starts), max_rows=max(counts),
              mask=None if mask is None else torch.as_tensor(mask.view(np.int32)).cuda())
    most = max(n + (0 if mask is None else c) for n, c in zip(lens, counts))
    for _ in range(times):
        o = torch.full_like(q, 9.0)
        gpu.pass_().attend_tree(q, pool, *args, o, most, **kw)
        gpu.sync()
        first = o if first is None else first
        assert torch.equal(o, first)
    return first


def hold(got, want, terms, dtype):
    got = got.double().cpu().numpy()
    bound = R.attend_bound(want, terms, dtype == "f16")
    far = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (far <= bound).all(), (far.max(), (far / np.maximum(bound, 1e-30)).max())


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", [(32, 8, 128), (16, 4, 64), (12, 4, 80)])
def test_items_that_end_inside_a_run_over_and_over(gpu, dtype, heads, kvh, hd):
    # Long items of drafted rows, cut by the runs at ever other places: their last tiles, whose V the
    # softmax edits, lie anywhere in the ring.
    rng = np.random.default_rng(hd)
    lens = rng.integers(1500, 4001, 20).tolist()
    counts = rng.integers(12, 17, 20).tolist()
    q, pool, table, starts, mask = make(hd, dtype, counts, lens, heads, kvh, hd, 32)
    got = attend(gpu, q, pool, table, starts, lens, mask, counts, times=60)
    want, terms = attend64(q, pool, table, starts, lens, mask, heads)
    hold(got, want, terms, dtype)


SHAPES = [(16, 2, 64), (16, 2, 128), (24, 2, 40)]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
def test_many_short_items_a_run(gpu, dtype, heads, kvh, hd):
    # Several hundred requests of one to four tiles, one or two items a K and V head: a run has more
    # items than the kernel holds at a time. Some have no rows, no positions, or neither.
    rng = np.random.default_rng(hd + 1)
    n = 420
    lens = rng.integers(0, 480, n)
    counts = rng.integers(1, 21, n)
    lens[rng.random(n) < 0.1] = 0
    counts[rng.random(n) < 0.1] = 0
    counts[0], counts[1] = 20, 0
    lens, counts = lens.tolist(), counts.tolist()
    q, pool, table, starts, mask = make(hd, dtype, counts, lens, heads, kvh, hd, 16)
    mask[rng.random(len(mask)) < 0.05] = 0  # rows that see no drafted position
    got = attend(gpu, q, pool, table, starts, lens, mask, counts, times=5)
    want, terms = attend64(q, pool, table, starts, lens, mask, heads)
    hold(got, want, terms, dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
@pytest.mark.parametrize("tree", [True, False])
def test_many_tiles_a_run(gpu, dtype, heads, kvh, hd, tree):
    # Few long items: a run has more than ten tiles of one, and every item spans many runs.
    counts, lens = [20, 9], [70001, 52345]
    q, pool, table, starts, mask = make(hd, dtype, counts, lens, heads, kvh, hd, 64, tree)
    got = attend(gpu, q, pool, table, starts, lens, mask, counts, times=5)
    want, terms = attend64(q, pool, table, starts, lens, mask, heads)
    hold(got, want, terms, dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
def test_scores_that_rise_late(gpu, dtype, heads, kvh, hd):
    # K grows towards a request's end, in steps of its own for every K and V head: the references
    # rise, and the outputs so far are scaled, at tiles anywhere in a run.
    rng = np.random.default_rng(hd + 2)
    lens = rng.integers(1400, 6000, 12).tolist()
    counts = rng.integers(9, 21, 12).tolist()
    q, pool, table, starts, mask = make(hd, dtype, counts, lens, heads, kvh, hd, 16)
    for s, (n, c) in enumerate(zip(lens, counts)):
        for b in range((n + c) // 16):
            grown = 0.2 + 4 * (b * 16 / n) ** (1 + np.arange(kvh) * 3)
            pool[int(table[s, b]), 0] *= torch.as_tensor(grown).cuda().half()[:, None, None]
    got = attend(gpu, q, pool, table, starts, lens, mask, counts, times=3)
    want, terms = attend64(q, pool, table, starts, lens, mask, heads)
    hold(got, want, terms, dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
@pytest.mark.parametrize("long", [False, True])
def test_infinities_in_one_item_after_another(gpu, dtype, heads, kvh, hd, long):
    # Drafted rows of most requests hold infinities and NaN in V, each in elements of its own: rows
    # that see one get it there, and nowhere else.
    rng = np.random.default_rng(hd + 3)
    n = 10 if long else 200
    lens = rng.integers(1400, 4000, n) if long else rng.integers(0, 400, n)
    counts = rng.integers(8, 21, n)
    counts[0] = 20
    lens, counts = lens.tolist(), counts.tolist()
    q, pool, table, starts, mask = make(hd, dtype, counts, lens, heads, kvh, hd, 16)
    clean = pool.clone()
    kinds = np.array([np.nan, np.inf, -np.inf])
    odd = np.zeros((sum(counts), kvh, hd))  # what the drafted rows hold, 0 where it is finite
    for s, (ln, c) in enumerate(zip(lens, counts)):
        for j in rng.choice(c, 2, replace=False) if rng.random() < 0.8 else []:
            for h in range(kvh):
                e = int(rng.integers(0, hd))
                odd[starts[s] + j, h, e] = rng.choice(kinds)
                at = int(table[s, (ln + j) // 16]), (ln + j) % 16
                pool[at[0], 1, h, at[1], e] = odd[starts[s] + j, h, e]
                clean[at[0], 1, h, at[1], e] = 0
    got = attend(gpu, q, pool, table, starts, lens, mask, counts).double().cpu().numpy()
    want, terms = attend64(q, clean, table, starts, lens, mask, heads)
    for s, c in enumerate(counts):
        for r in range(starts[s], starts[s + 1]):
            for j in range(c):
                if R.sees(mask[r], j):
                    add = np.repeat(odd[starts[s] + j], heads // kvh, 0).reshape(-1)
                    with np.errstate(invalid="ignore"):
                        want[r] += add
    whole = np.isfinite(want)
    assert (~whole).any() and np.array_equal(got[~whole], want[~whole], equal_nan=True)
    bound = R.attend_bound(want, terms, dtype == "f16")
    assert (np.abs(got[whole] - want[whole]) <= bound[whole]).all()
