"""Row strides of tensors that share memory between rows, or that a single row makes arbitrary, on
the GPU: the entry points take a row's stride as torch has it or refuse it."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    from wavo_b200.gpu import Gpu
    g = Gpu(0)
    yield g
    g.close()


def i32(a):
    return torch.as_tensor(np.ascontiguousarray(a).astype(np.int64).astype(np.int32)).cuda()


def attend(gpu, q, o, pool, rows):
    gpu.pass_().attend_tree(q, pool, i32([[0, 1]]), i32([20]), o, 32, row_start=i32([0, rows]),
                            max_rows=rows)
    gpu.sync()


def test_attention_rows_that_share_memory_are_refused(gpu):
    # A stride of 0 is the ABI's default (dense rows): rows past the tensor would be read.
    pool = torch.randn(2, 2, 2, 16, 64, device="cuda").half()
    row = torch.randn(1, 128, device="cuda")
    for q, o in ((row.expand(4, 128), torch.empty(4, 128, device="cuda")),
                 (torch.randn(4, 128, device="cuda"), torch.empty(1, 128, device="cuda").expand(4, 128)),
                 (torch.randn(300, device="cuda").as_strided((4, 128), (50, 1)),
                  torch.empty(4, 128, device="cuda"))):
        with pytest.raises(ValueError, match="stride"):
            attend(gpu, q, o, pool, 4)


def test_a_single_row_may_have_any_stride(gpu):
    pool = torch.randn(2, 2, 2, 16, 64, device="cuda").half()
    q = torch.randn(1, 128, device="cuda")
    want, got = torch.empty_like(q), torch.zeros(128, device="cuda")
    attend(gpu, q, want, pool, 1)
    attend(gpu, q.flatten().as_strided((1, 128), (1, 1)), got.as_strided((1, 128), (3, 1)), pool, 1)
    assert torch.equal(got, want[0])


def test_logits_that_share_memory_between_rows(gpu):
    from wavo_b200.gpu import LogitRules
    p = gpu.pass_()
    rules = LogitRules(100, n=3)
    x = torch.randn(1, 100, device="cuda")
    picks = i32([-7] * 3)
    for logits, out in ((x.expand(3, 100), None),
                        (torch.randn(3, 100, device="cuda"), torch.empty(1, 100, device="cuda").expand(3, 100)),
                        (torch.randn(150, device="cuda").as_strided((3, 100), (25, 1)), None)):
        with pytest.raises(ValueError, match="stride"):
            p.shape_logits(logits, rules, picks, out=out)
    # One row: any stride.
    out = torch.zeros(100, device="cuda")
    p.shape_logits(x.flatten().as_strided((1, 100), (1, 1)), LogitRules(100, n=1), picks,
                   out=out.as_strided((1, 100), (2, 1)))
    gpu.sync()
    assert torch.equal(out, x[0]) and int(picks[0]) == int(x.argmax())


def test_packed_rows_end_with_the_memory_of_x(gpu):
    # x is rows in memory: what counts is what lies behind its first element, not its shape.
    p = gpu.pass_()
    pool = torch.zeros(2, 2, 1, 16, 8, dtype=torch.float16, device="cuda")
    slots = i32([3, 20, 7])
    row = torch.randn(16, device="cuda")
    with pytest.raises(ValueError, match="fewer rows"):
        p.pack_slots(row.expand(3, 16), (0, 16), slots, pool)
    with pytest.raises(ValueError, match="fewer rows"):
        p.pack_slots(torch.randn(3, 24, device="cuda")[:, ::2], (20, 24), slots, pool)
    for before in (-1, 24):
        with pytest.raises(ValueError, match="fewer rows"):
            p.pack_slots(torch.randn(3, 24, device="cuda"), (before, 24 if before < 0 else -8), slots, pool)
    x = torch.randn(3, 24, device="cuda")
    p.pack_slots(x[:, 8:], (0, 24), slots, pool)  # a view whose last row ends with x
    gpu.sync()
    for r, s in enumerate([3, 20, 7]):
        assert torch.equal(pool[s // 16, :, 0, s % 16].flatten(), x[r, 8:].half())
