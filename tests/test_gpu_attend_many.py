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
