"""What TreeDecoder refuses and gives back on the GPU: prompts, segments that are done, the end of the
context, another stream."""

import numpy as np
import pytest
import torch

import test_gpu_tree_decoder as D

pytestmark = pytest.mark.gpu

PROMPTS = [[3, 7, 11], [5], [9, 2, 2, 8, 1, 4]]


@pytest.fixture(scope="module")
def gpu():
    from wavo_b200.gpu import Gpu
    g = Gpu(0)
    yield g
    g.close()


@pytest.fixture(scope="module")
def weights():
    return D.encode(D.weights(np.random.default_rng(5)))


def decoder(gpu, weights, batch=3, max_rows=24, context=D.CONTEXT, blocks=0):
    from wavo_b200 import GGML_F16
    from wavo_b200.blocks import TreeDecoder
    dec = TreeDecoder(gpu, GGML_F16, D.D, D.HEADS, D.D_FF, D.VOCAB, context, D.FRAMES, batch, weights,
                      max_rows, blocks=blocks)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    enc = torch.randn(batch, D.FRAMES, D.D, generator=g, device="cuda")
    torch.cuda.current_stream().synchronize()  # (the encoder's output may come from another stream)
    dec.record_cross(gpu.pass_(), enc)
    return dec


def steps(gpu, dec, last, n):
    """n single-token steps from the last tokens: each segment's tokens."""
    got = [[] for _ in last]
    for _ in range(n):
        for b, more in enumerate(dec.verify(gpu.pass_(), [([t], [-1]) for t in last])):
            got[b] += more
        last = [g[-1] for g in got]
    return got


def test_a_start_that_is_refused_leaves_the_windows(gpu, weights):
    dec = decoder(gpu, weights)
    want = steps(gpu, dec, dec.start(gpu.pass_(), PROMPTS), 6)
    first = dec.start(gpu.pass_(), PROMPTS)
    got = steps(gpu, dec, first, 2)
    for bad in ([[1], [2], [D.VOCAB]], [[1], [2]], [[1], [2], list(range(25))]):
        with pytest.raises(ValueError):
            dec.start(gpu.pass_(), bad)
    for b, more in enumerate(steps(gpu, dec, [g[-1] for g in got], 4)):
        assert got[b] + more == want[b]


@pytest.mark.parametrize("at", [0, 1, 2])
def test_a_prompt_without_tokens_is_refused(gpu, weights, at):
    # It has no last row, whose pick would be the segment's first token.
    dec = decoder(gpu, weights)
    prompts = [list(t) for t in PROMPTS]
    prompts[at] = []
    with pytest.raises(ValueError, match="prompt"):
        dec.start(gpu.pass_(), prompts)


def test_blocks_come_back_when_every_segment_is_done(gpu, weights):
    dec = decoder(gpu, weights)
    blocks = int(dec.state[1])
    steps(gpu, dec, dec.start(gpu.pass_(), PROMPTS), 3)
    assert int(dec.state[1]) < blocks
    assert dec.verify(gpu.pass_(), [None] * 3) == [[]] * 3
    assert int(dec.state[1]) == blocks
    assert dec.owned.tolist() == [0] * 3
    # Again, and beside segments that wait.
    assert dec.verify(gpu.pass_(), [None] * 3) == [[]] * 3
    first = dec.start(gpu.pass_(), PROMPTS)
    assert dec.verify(gpu.pass_(), [None, ([], []), None]) == [[]] * 3
    assert int(dec.state[1]) == blocks - 1
    got = dec.verify(gpu.pass_(), [None, ([first[1]], [-1]), None])
    assert [len(g) for g in got] == [0, 1, 0] and int(dec.state[1]) == blocks - 1
    dec.start(gpu.pass_(), PROMPTS)
    assert int(dec.state[1]) == blocks - 3


@pytest.mark.parametrize("together", [True, False])
def test_a_segment_that_is_done_holds_nothing(gpu, weights, together):
    # What comes for it next begins an empty window, with blocks of its own from then on.
    dec = decoder(gpu, weights)
    blocks = int(dec.state[1])
    want = steps(gpu, dec, [7, 8, 9], 5)
    dec = decoder(gpu, weights)
    first = dec.start(gpu.pass_(), [[4] * 20, [5] * 20, [6] * 20])
    dec.verify(gpu.pass_(), [None] * 3 if together else [None, ([first[1]], [-1]), None])
    dec.verify(gpu.pass_(), [([], [])] * 3)
    assert int(dec.state[1]) == blocks - (0 if together else 2)
    dec.verify(gpu.pass_(), [([], []), None, ([], [])])
    assert int(dec.state[1]) == blocks and dec.lens.tolist() == [0] * 3
    assert steps(gpu, dec, [7, 8, 9], 5) == want


def test_the_end_of_the_context(gpu, weights):
    # A segment gains the tokens that its positions give, one after the last of them included, drafts
    # or not, and is then refused with that reason.
    context = 20
    full = decoder(gpu, weights)
    want = []
    first = full.start(gpu.pass_(), PROMPTS)
    for t, p, more in zip(first, PROMPTS, steps(gpu, full, first, context)):
        want.append([t, *more][:context - len(p) + 1])
    for drafts in (0, 1, 4, 30):
        dec = decoder(gpu, weights, context=context, max_rows=31)
        got = [[t] for t in dec.start(gpu.pass_(), PROMPTS)]
        assert [g[0] for g in got] == first
        for _ in range(context):
            trees = []
            for g, w in zip(got, want):
                # Right drafts to the end of what there is, then wrong ones.
                chain = (w[len(g):] + [1] * 30)[:drafts]
                trees.append(None if len(g) == len(w) else ([g[-1]] + chain, list(range(-1, len(chain)))))
            if trees == [None] * 3:
                break
            for g, more in zip(got, dec.verify(gpu.pass_(), trees)):
                g += more
        assert got == want
        assert dec.verify(gpu.pass_(), [None] * 3) == [[]] * 3
    dec = decoder(gpu, weights, context=context)
    first = dec.start(gpu.pass_(), [[4] * context, [5], [6]])
    with pytest.raises(ValueError, match="context"):
        dec.verify(gpu.pass_(), [([t], [-1]) for t in first])
    assert dec.verify(gpu.pass_(), [None] + [([t], [-1]) for t in first[1:]])[0] == []
    with pytest.raises(ValueError, match="context"):
        dec.start(gpu.pass_(), [[4] * (context + 1), [5], [6]])


@pytest.mark.parametrize("how", ["context", "torch"])
def test_a_step_runs_on_the_contexts_stream(gpu, weights, how):
    # The library's work and torch's of a step are on one stream, whichever is torch's current one,
    # which is kept busy here.
    dec = decoder(gpu, weights)
    want = steps(gpu, dec, dec.start(gpu.pass_(), PROMPTS), 4)
    torch.cuda.synchronize()
    side, here = torch.cuda.Stream(), torch.cuda.current_stream()

    def busy():
        torch.cuda._sleep(20_000_000)  # some 10 ms

    def go():
        busy()
        dec = decoder(gpu, weights)
        busy()
        last, got = dec.start(gpu.pass_(), PROMPTS), [[] for _ in PROMPTS]
        for _ in range(4):
            busy()
            for g, more in zip(got, steps(gpu, dec, last, 1)):
                g += more
            last = [g[-1] for g in got]
        return got
    if how == "context":
        gpu.use_stream(side)
        try:
            got = go()
        finally:
            side.synchronize()
            gpu.use_stream(here)
    else:
        with torch.cuda.stream(side):
            got = go()
    torch.cuda.synchronize()
    assert got == want
