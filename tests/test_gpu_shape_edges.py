"""Logit rules at their edges on the GPU, against the plain forms: equal maxima among named tokens,
and log-probabilities of logits of any size."""

import numpy as np
import pytest
import torch

import tree_reference as R

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
