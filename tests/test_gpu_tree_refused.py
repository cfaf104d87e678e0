"""Requests that a step's plan refuses, on the GPU: their rows reach no block of others, in the plan,
in the commit and in a decoder that goes on without them."""

import numpy as np
import pytest
import torch

import test_gpu_tree_decoder as D

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    from wavo_b200.gpu import Gpu
    g = Gpu(0)
    yield g
    g.close()


def i32(a):
    return torch.as_tensor(np.ascontiguousarray(a).astype(np.int64).astype(np.int32)).cuda()


def plan(gpu, lens, adds, bs, ring, state, owned, table, rows):
    n = len(lens)
    t = {"table": i32(table), "ring": i32(ring), "row_start": i32([0] * (n + 1)),
         "row_seq": i32([0] * rows), "slots": i32([0] * rows), "state_out": i32([0] * 4),
         "owned_out": i32([0] * n)}
    gpu.pass_().block_tables(i32(lens), i32(adds), bs, t["ring"], i32(state), i32(owned), t["table"],
                             t["row_start"], t["row_seq"], t["slots"], t["state_out"], t["owned_out"])
    gpu.sync()
    return t


def test_entries_that_a_refused_request_lacks_name_no_block(gpu):
    # Served, refused for want of blocks, wider than the table, done, refused without any block.
    # The entries past what they own name blocks of others.
    table = [[4, 0, 0, 0], [5, 4, 4, 4], [6, 7, 0, -5], [8, 9, 1, 1], [0, 1, 2, 3]]
    t = plan(gpu, [16, 20, 32, 20, 0], [3, 50, 40, -1, 17], 16, [10, -9, -9, -9, -9], [0, 1],
             [1, 1, 2, 2, 0], table, 110)
    assert t["table"].tolist() == [[4, 10, 0, 0], [5, -1, -1, -1], [6, 7, -1, -5], [8, 9, 1, 1],
                                   [-1, -1, 2, 3]]
    assert t["state_out"].tolist() == [1, 2, 110, 3]
    assert t["owned_out"].tolist() == [2, 1, 2, 0, 0]


@pytest.mark.parametrize("n", [2, 700])
def test_the_commit_of_a_refused_request_moves_nothing_of_others(gpu, n):
    # Each request holds 16 positions in a block of its own and drafts [token, wrong, right]. One free
    # block: the first is served, the others' next entries name block 0.
    bs, kvh, hd, layers = 16, 2, 64, 2
    table = np.zeros((n, 2), int)
    table[:, 0] = np.arange(n)
    ring = np.full(n + 1, -9)
    ring[0] = n
    t = plan(gpu, [16] * n, [3] * n, bs, ring, [0, 1], [1] * n, table, 3 * n)
    assert int(t["state_out"][3]) == n - 1
    pool = torch.randn(layers, n + 1, 2, kvh, bs, hd, device="cuda").half()
    want = pool.clone()
    want[:, n, :, :, 1] = want[:, n, :, :, 2]  # the first's: position 18 to 17
    mask = torch.as_tensor(np.array([[1], [3], [5]] * n, np.int32)).cuda()
    path, count, after, new = i32(np.zeros((n, 3))), i32([0] * n), i32([0] * n), i32([0] * n)
    gpu.pass_().tree_accept(i32([9, 8, 3] * n), i32([5, 4, 9] * n), mask, t["row_start"],
                            i32([16] * n), t["table"], pool, path, count, after, new)
    gpu.sync()
    assert path[0].tolist() == [0, 2, -1] and new.tolist() == [18] * n
    assert torch.equal(pool.view(torch.int16), want.view(torch.int16))


def test_a_decoder_without_blocks_keeps_every_cache(gpu):
    from wavo_b200 import GGML_F16
    from wavo_b200.blocks import TreeDecoder
    w = D.encode(D.weights(np.random.default_rng(2)))
    p = gpu.pass_()
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, D.VOCAB, 16).tolist() for _ in range(2)]

    def decoder(blocks):
        dec = TreeDecoder(gpu, GGML_F16, D.D, D.HEADS, D.D_FF, D.VOCAB, D.CONTEXT, D.FRAMES, 2, w, 32,
                          blocks=blocks)
        dec.record_cross(p, torch.zeros(2, D.FRAMES, D.D, device="cuda"))
        return dec, dec.start(p, prompts)
    dec, first = decoder(0)
    after = [g[0] for g in dec.verify(p, [([t], [-1]) for t in first])]
    dec, again = decoder(3)
    assert again == first
    gpu.sync()

    def held(b):
        return dec.pool[:, int(dec.table[b, 0])].clone()
    before = [held(b) for b in range(2)]
    # Segment 1 is refused. Its right token is behind a wrong one, off its place.
    wrong = [(t + 1) % D.VOCAB for t in after]
    trees = [([first[b], wrong[b], after[b]], [-1, 0, 0]) for b in range(2)]
    wide = ([first[1]] + list(range(D.VOCAB - 31, D.VOCAB)), [-1] + [0] * 31)
    for tree in (trees[1], wide):
        with pytest.raises(RuntimeError, match="1 segments"):
            dec.verify(p, [trees[0], tree])
        gpu.sync()
        assert all(torch.equal(held(b), before[b]) for b in range(2))
    # The first goes on alone as it would have.
    assert dec.verify(p, [trees[0], None])[0][0] == after[0]
