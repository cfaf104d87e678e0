"""Logit rules at their edges on the GPU, against the plain forms: equal maxima among named tokens,
and log-probabilities of logits of any size."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f16": np.float16, "f32": np.float32}


@pytest.fixture(scope="module")
def gpu():
    from wavo_b200.gpu import Gpu
    g = Gpu(0)
    yield g
    g.close()


def i32(a):
    return torch.as_tensor(np.ascontiguousarray(a).astype(np.int64).astype(np.int32)).cuda()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [5, 40, 2049, 8192, 51866])
@pytest.mark.parametrize("rows", [1, 3, 160])
def test_the_first_of_equal_maxima_among_named_tokens(gpu, dtype, vocab, rows):
    # Rules that change nothing (penalties of 1, 0, 0 and biases of 0) name tokens in rows of equal
    # values: the pick is the lowest index, named or not, below or above the named ones.
    from wavo_b200.gpu import LogitRules
    rng = np.random.default_rng(vocab + rows)
    x = rng.integers(0, 3, (rows, vocab)).astype(TYPES[dtype])  # many maxima
    x[::3] = 0                                                  # all equal
    history = rng.integers(0, vocab, (rows, 30))
    history[:, 0] = np.minimum(4, vocab - 1)
    ids = rng.integers(0, vocab, (rows, 20))
    rules = LogitRules(
        vocab, history=(i32(history), i32(np.arange(rows) % 31)),
        penalties=torch.tensor([[1.0, 0.0, 0.0]] * rows).cuda(),
        bias=(i32(ids), torch.zeros(rows, 20).cuda(), i32(np.arange(rows) * 7 % 21)))
    picks = i32([-7] * rows)
    gpu.pass_().shape_logits(torch.as_tensor(x).cuda(), rules, picks)
    gpu.sync()
    assert picks.tolist() == x.argmax(1).tolist()


def logprobs(gpu, x):
    from wavo_b200.gpu import LogitRules
    picks, lp = i32([-7] * len(x)), torch.full((len(x),), 7.0, device="cuda")
    gpu.pass_().shape_logits(torch.as_tensor(x).cuda(), LogitRules(x.shape[1], n=len(x)), picks, lp)
    gpu.sync()
    assert picks.tolist() == x.argmax(1).tolist()
    return lp.double().cpu().numpy()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [7, 3001, 51866])
@pytest.mark.parametrize("size", [3, 30, 1000, 1e5, 1e30])
def test_log_probabilities_of_logits_of_any_size(gpu, dtype, vocab, size):
    if dtype == "f16":
        size = min(size, 4e3)  # in its range
    rng = np.random.default_rng(vocab)
    x = (size * rng.standard_normal((5, vocab))).astype(TYPES[dtype])
    x[1] += TYPES[dtype](size * 5)
    x[2] = x[2, 0] + (rng.standard_normal(vocab) * min(size, 1.0)).astype(TYPES[dtype])
    got = logprobs(gpu, x)
    d = x.astype(np.float64) - x.max(1, keepdims=True).astype(np.float64)
    e = np.exp(d)
    total = e.sum(1)
    # A difference, its product with log2(e) and the exponential are off by 2^-24, 2^-23 and 2^-21 of
    # their values at most; the sum has 2^-24 a step (a thread's tokens, then the threads'), the
    # logarithm 2^-22 of its value.
    bound = (e * np.abs(d)).sum(1) / total * 2.0 ** -22 + 2.0 ** -21 + \
        (vocab / 512 + 40) * 2.0 ** -24 + 2.0 ** -22 * np.log(total)
    assert (np.abs(got + np.log(total)) <= bound).all(), (got + np.log(total), bound)
    assert (got <= 0).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [7, 3001, 51866])
def test_tokens_masked_by_the_lowest_value(gpu, dtype, vocab):
    # The lowest finite value in place of -inf: all tokens, all but one, all but a few, every second;
    # and the largest value beside it.
    low, high = np.finfo(TYPES[dtype]).min, np.finfo(TYPES[dtype]).max
    rng = np.random.default_rng(vocab)
    x = np.full((6, vocab), low, TYPES[dtype])
    x[1, vocab // 2] = -2
    x[2, rng.integers(0, vocab, 3)] = rng.standard_normal(3)
    x[3, ::2] = rng.standard_normal(len(x[3, ::2]))
    x[4, vocab - 1] = high
    x[5, ::3] = high
    got = logprobs(gpu, x)
    with np.errstate(over="ignore"):
        total = np.exp(x.astype(np.float64) - x.max(1, keepdims=True).astype(np.float64)).sum(1)
    assert np.allclose(got, -np.log(total), rtol=2e-6, atol=2e-6 + vocab / 512 * 2.0 ** -24)
