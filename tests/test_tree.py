"""CPU checks of the entry points over paged caches and drafted trees, and of the plain forms that
the GPU tests compare with."""

import ctypes

import numpy as np

import tree_reference as R
from wavo_b200 import _lib as L


def test_null_context_is_rejected():
    lib = L.lib()
    rules = L.LogitRulesC()
    assert lib.wavo_block_tables(None, *[None] * 2, 1, 16, None, 1, None, None, None, 1, None, None,
                                 None, 0, None, None) == L.EINVAL
    assert lib.wavo_pack_slots(None, None, 0, 0, 0, None, 1, None, 1, 16, 1, 64) == L.EINVAL
    assert lib.wavo_attend_tree(None, None, 0, 0, None, 1, 16, None, 1, None, None, 1, None, 0, 1, 1,
                                1, None, 0, 1, 1, 64) == L.EINVAL
    assert lib.wavo_shape_logits(None, None, 0, 0, None, 0, 1, ctypes.byref(rules), None,
                                 None) == L.EINVAL
    assert lib.wavo_tree_accept(None, *[None] * 3, 1, 1, None, 1, 1, None, None, 0, None, 0, 0, 0, 0,
                                0, 0, None, None, None, None) == L.EINVAL


def test_rules_struct_is_the_headers():
    # The header's fields in order, with C's alignment of 4- and 8-byte members.
    with open(L.HEADER) as fh:
        text = fh.read()
    body = text[text.index("typedef struct wavo_logit_rules {"):text.index("} wavo_logit_rules;")]
    import re
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    want, at = [], 0
    for line in body[body.index("{") + 1:].split(";"):
        line = line.strip()
        if not line:
            continue
        for name in line.split(","):
            size = 8 if "*" in name or "*" in line.split(",")[0] else 4
            at = -(-at // size) * size
            want.append((name.replace("*", " ").split()[-1], at, size))
            at += size
    got = [(n, getattr(L.LogitRulesC, n).offset, getattr(L.LogitRulesC, n).size)
           for n, _ in L.LogitRulesC._fields_]
    assert got == want


def test_plan_by_hand():
    # 8 positions a block; request 0 grows by one block, 1 is done, 2 lacks two of which one is
    # left, 3 needs none.
    got = R.block_tables([7, 9, 0, 3], [3, -1, 9, 1], 8, [4, 5, -1, -1, -1], [0, 2], [1, 2, 0, 1],
                         [[0, -1], [1, 2], [-1, -1], [3, -1]], 15)
    assert got["table"] == [[0, 4], [1, 2], [-1, -1], [3, -1]]
    assert got["ring"] == [4, 5, 1, 2, -1]
    assert got["owned_out"] == [2, 0, 0, 1]
    assert got["row_start"] == [0, 3, 3, 12, 13]
    assert got["slots"] == [7, 32, 33] + [-1] * 9 + [27] + [-1] * 2
    assert got["state_out"] == [1, 3, 13, 1]


def test_attention_by_hand():
    rng = np.random.default_rng(0)
    pool = rng.standard_normal((2, 2, 1, 8, 8)).astype(np.float16)
    q = rng.standard_normal((2, 8))
    # Ten positions and two drafted rows; the second sees itself alone.
    mask = np.array([[0], [2]], np.uint32)
    o, _ = R.attend(q, pool, np.array([[1, 0]]), [0, 2], [10], mask, 1)
    k = np.concatenate([pool[1, 0, 0], pool[0, 0, 0]]).astype(np.float64)
    v = np.concatenate([pool[1, 1, 0], pool[0, 1, 0]]).astype(np.float64)
    for r, seen in enumerate([list(range(10)), list(range(10)) + [11]]):
        e = np.exp(k[seen] @ q[r] / np.sqrt(8))
        assert np.allclose(o[r], e @ v[seen] / e.sum(), rtol=1e-12)
    o, _ = R.attend(q, pool, np.array([[1, 0]]), [0, 2], [0], mask, 1)
    assert (o[0] == 0).all() and np.allclose(o[1], v[1])


def test_logit_rules_by_hand():
    x, best, lp = R.shape_logits(np.array([2.0, -1.0, 0.5, 3.0]), 4, [0, 1, 0, 9], (2.0, 0.5, 0.25),
                                 ([2, 2], [5.0, 1.0]), np.array([True, True, True, False]))
    assert x.tolist() == [2.0 / 2 - 1.0, -1.0 * 2 - 0.75, 1.5, -np.inf]
    assert best == 2 and abs(lp + np.log(np.exp(x[:3].astype(np.float64) - 1.5).sum())) < 1e-12


def test_walk_by_hand():
    # 0 -> 1, 2; 1 -> 3; both children of 0 carry the pick: the first one counts.
    mask = np.array([[1], [3], [5], [11]], np.uint32)
    assert R.tree_accept([7, 8, 9, 6], [5, 7, 7, 8], mask, [0, 4], [0]) == [([0, 1, 3], 6)]
    assert R.tree_accept([1, 8, 9, 6], [5, 7, 7, 8], mask, [0, 4], [0]) == [([0], 1)]
