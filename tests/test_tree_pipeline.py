"""The order of events in the many-rows attention's pipeline (csrc/tree.cu), on the CPU. Its waits go
by the parity of an mbarrier's phase, and such a wait is sound only if the phase before has completed
when it starts: otherwise it is let through at once."""

import os
import re

import pytest

from wavo_b200 import build


def happened(ring, n, v_after_s):
    """For each of n tiles, whether the load that had V's place in the ring before must have landed
    when the softmax starts to wait for V. Events follow from one another by the program order of
    the loads, the UMMAs and the softmax, and by the waits between them."""
    steps = []  # the loads' order, K of tile g with S, V with P.V
    for g in range(n + 1):
        steps += [("S", g)] * (g < n) + [("PV", g - 1)] * (g > 0)
    after = {}
    for i, (kind, g) in enumerate(steps):
        # A place of the ring is loaded again when the UMMAs that read it are done.
        after["load", i] = {("load", i - 1)} | ({("done", *steps[i - ring])} if i >= ring else set())
        after["landed", i] = {("load", i)}
        after["issue", kind, g] = {("landed", i)} | ({("issue", *steps[i - 1])} if i else set())
        if kind == "S":    # over the P of two tiles before
            after["issue", kind, g] |= {("done", "PV", g - 2)}
        else:
            after["issue", kind, g] |= {("probabilities", g)}
        after["done", kind, g] = {("issue", kind, g)} | ({("done", *steps[i - 1])} if i else set())
    for g in range(n):
        # A tile that every row sees whole has no wait for V.
        after["probabilities", g] = {("done", "S", g), ("probabilities", g - 1)}
        after["wait V", g] = {("probabilities", g - 1)} | ({("done", "S", g)} if v_after_s else set())
    sound = []
    for g in range(n):
        past, todo = set(), [("wait V", g)]
        while todo:
            for e in after.get(todo.pop(), ()):
                if e not in past:
                    past.add(e)
                    todo.append(e)
        i = steps.index(("PV", g))
        assert i == (2 * n - 1 if g == n - 1 else 2 * g + 2)  # as the kernel counts it
        sound.append(i < ring or ("landed", i - ring) in past)
    return sound


@pytest.mark.parametrize("n", [1, 2, 3, 20])
def test_the_wait_for_v_goes_by_the_phase_that_is_next(n):
    with open(os.path.join(build.CSRC, "tree.cu")) as fh:
        text = fh.read()
    rings = [int(x) for x in re.search(r"kRing = HDP == 64 \? (\d+) : WIDE \? (\d+) : (\d+);",
                                       text).groups()]
    soft = text[text.index("// ---- softmax:"):]
    s, v = (soft.index(f"mbar_wait_warp(&sh.{bar}") for bar in ("s_full[g & 1]", "full[p % D]"))
    for ring in rings:
        assert all(happened(ring, n, v_after_s=s < v)), ring


def test_the_model_sees_the_wait_that_is_too_early():
    assert all(happened(5, 20, False)) and all(happened(8, 20, False))
    assert happened(4, 6, False) == [True, True, False, False, False, True]
