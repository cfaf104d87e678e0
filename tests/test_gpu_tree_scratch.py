"""The scratch that attend_tree says it needs, against calls that reach less than they were asked for
(fewer positions, fewer rows), in a capture, where it cannot grow."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.as_tensor(np.ascontiguousarray(a).astype(np.int64).astype(np.int32)).cuda()


@pytest.mark.parametrize("rows,asked", [(1, 64), (4096, 1)])
def test_scratch_is_enough_for_shorter_tables_and_fewer_rows(rows, asked):
    from wavo_b200.gpu import Gpu
    g = Gpu(0)
    # Ranges of 256 positions where the tables end, 320 one position on; fewer if one row were 64.
    per = 3 * g.sm_count // 4
    reach = per * 256
    need = g.attend_tree_scratch(1, rows, asked, reach + 1, 4, 4, 64)
    assert need >= g.attend_tree_scratch(1, rows, 1, reach, 4, 4, 64)
    assert need <= 2 * g.attend_tree_scratch(1, rows, 1, reach, 4, 4, 64)
    g.reserve(need)
    bs = 256
    pool = torch.randn(per, 2, 4, bs, 64, device="cuda").half()
    table = i32(np.arange(per)[None])
    q = torch.randn(rows, 256, device="cuda")
    o, want = torch.zeros_like(q), torch.zeros_like(q)
    lens, starts = i32([reach]), i32([0, 1])
    go = lambda p, to: p.attend_tree(q, pool, table, lens, to, reach + 1, row_start=starts,  # noqa: E731
                                     max_rows=asked)
    graph = g.capture(lambda p: go(p, o))
    graph.launch()
    go(g.pass_(), want)
    g.sync()
    assert torch.equal(o, want) and bool((o[0] != 0).any()) and not bool(o[1:].any())
    del graph
    g.close()
