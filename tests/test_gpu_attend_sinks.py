"""Attention of drafted tokens where a row's probabilities are far apart, on the GPU: one position
holds almost all of a row's sum and adds next to nothing to its output (a sink), so that the output
is the small probabilities'."""

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


def bound(o, b, f16, floor):
    """How far an output may be from the 64-bit one. The products of q and k are whole multiples of
    1/64, so their sums are exact; a score's scaling and its difference to the reference are off by
    2^-22 of the scores at most, its exponential by 2^-21, and a relative error of p moves o by at
    most twice that of sum p|v|; the sum over keys takes 16 products at a time, one addition a step.
    f16: the probability and the output are rounded once each. floor: the step of a probability's
    last part where it is subnormal, against the row's largest probability."""
    each = 2 * 2.0 ** -22 * b["qk"] + 2.0 ** -20 + (b["keys"] / 16 + 20) * 2.0 ** -23
    if f16:
        return 2.0 ** -11 * (np.abs(o) + b["size"]) * 1.01 + b["size"] * each + 2.0 ** -25 + \
            floor * b["flat"]
    return 2.0 ** -23 * np.abs(o) + b["size"] * each + floor * b["flat"]


def sink_case(gpu, dtype, gap, at, n, t, heads, kvh, hd, mean, drafted):
    """Rows whose score at position `at` is `gap`, the others' of deviation 1, V zero there and of
    deviation 200 (with a mean, or without) elsewhere."""
    rng = np.random.default_rng(n + at)
    bs, group = 16, heads // kvh
    keys = n + (t if drafted else 0)
    table, blocks = R.paged(rng, [keys], bs)
    eighths = lambda x: np.round(8 * x) / 8  # noqa: E731
    k = eighths(rng.standard_normal((kvh, keys, hd)))
    v = 200 * (rng.standard_normal((kvh, keys, hd)) + mean)
    q = eighths(np.clip(rng.standard_normal((t, heads, hd)), -4, 4))
    # The first element is the sink's: q has 8 there, k 0, but the sink's.
    q[:, :, 0], k[:, :, 0], v[:, at], k[:, at] = 8, 0, 0, 0
    k[:, at, 0] = eighths(gap * np.sqrt(hd) / 8)
    q = q.reshape(t, heads * hd).astype(np.float16 if dtype == "f16" else np.float32)
    pool = np.zeros((blocks, 2, kvh, bs, hd), np.float16)
    for p in range(keys):
        pool[table[0, p // bs], 0, :, p % bs] = k[:, p]
        pool[table[0, p // bs], 1, :, p % bs] = v[:, p]
    mask = None
    if drafted:  # every row sees all of the drafted ones
        mask = np.full((t, -(-t // 32)), 0xffffffff, np.uint32)
    qd = torch.as_tensor(q).cuda()
    o = torch.empty_like(qd)
    gpu.pass_().attend_tree(
        qd, torch.as_tensor(pool).cuda(), i32(table), i32([n]), o, keys, row_start=i32([0, t]),
        mask=None if mask is None else torch.as_tensor(mask.view(np.int32)).cuda(), max_rows=t)
    gpu.sync()
    want, terms = R.attend(q, pool, table, [0, t], [n], mask, heads)
    return o.double().cpu().numpy(), want, terms


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("gap", [10, 12, 15, 18])
@pytest.mark.parametrize("where", ["first", "middle", "last", "drafted"])
@pytest.mark.parametrize("mean", [0, 1])
def test_a_sink_few_rows(gpu, dtype, gap, where, mean):
    n, t = 300, 5
    at = {"first": 0, "middle": 150, "last": n - 1, "drafted": n + 2}[where]
    got, want, terms = sink_case(gpu, dtype, gap, at, n, t, 4, 2, 64, mean, where == "drafted")
    # The largest probability is 2^15 where it is rounded: f16's step is 2^-24, two parts' 2^-35.
    lim = bound(want, terms, dtype == "f16", 2.0 ** -40 if dtype == "f16" else 2.0 ** -50)
    assert (np.abs(got - want) <= lim).all(), (np.abs(got - want) / lim).max()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("gap", [12, 18])
@pytest.mark.parametrize("hd,n,at", [(64, 1, 0), (128, 77, 40), (40, 1500, 3)])
def test_a_sink_few_rows_sizes(gpu, dtype, gap, hd, n, at):
    got, want, terms = sink_case(gpu, dtype, gap, at, n, 20, 2, 2, hd, 1, False)
    lim = bound(want, terms, dtype == "f16", 2.0 ** -40 if dtype == "f16" else 2.0 ** -50)
    assert (np.abs(got - want) <= lim).all(), (np.abs(got - want) / lim).max()


# The kernel for many rows (more than 128 of a K and V head, or more than 32 over a long cache).

@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("gap", [10, 12, 15, 18])
@pytest.mark.parametrize("where", ["first", "middle", "last", "drafted"])
@pytest.mark.parametrize("mean", [0, 1])
def test_a_sink_many_rows(gpu, dtype, gap, where, mean):
    n, t = 300, 20
    at = {"first": 0, "middle": 150, "last": n - 1, "drafted": n + 2}[where]
    got, want, terms = sink_case(gpu, dtype, gap, at, n, t, 16, 2, 64, mean, where == "drafted")
    # The largest probability is 2^7 to 2^15 where it is rounded.
    lim = bound(want, terms, dtype == "f16", 2.0 ** -32 if dtype == "f16" else 2.0 ** -42)
    assert (np.abs(got - want) <= lim).all(), (np.abs(got - want) / lim).max()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("gap", [12, 18])
@pytest.mark.parametrize("hd,n,at", [(64, 1, 0), (128, 4000, 40), (40, 1500, 1499), (64, 4000, 2000)])
def test_a_sink_many_rows_sizes(gpu, dtype, gap, hd, n, at):
    got, want, terms = sink_case(gpu, dtype, gap, at, n, 17, 8, 1, hd, 1, False)
    lim = bound(want, terms, dtype == "f16", 2.0 ** -32 if dtype == "f16" else 2.0 ** -42)
    assert (np.abs(got - want) <= lim).all(), (np.abs(got - want) / lim).max()
