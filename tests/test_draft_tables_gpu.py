"""Block tables of drafted continuations that are no contiguous tensors of their own: a row ends where its columns do, whatever lies
behind them, and rows may lie at any distance."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_drafts_gpu import Trees, caches, i32

pytestmark = pytest.mark.gpu

I32 = torch.int32


def within_a_wider_one(table, pages):
    """``table`` as a view whose neighbours on all sides are numbers of pages that are there."""
    rows, columns = table.shape
    wide = torch.randint(0, pages, (rows + 2, columns + 9), dtype=I32, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    view = wide[1:rows + 1, 4:4 + columns]
    view.copy_(i32(table))
    return view


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,page", [(64, 16), (20, 16), (128, 5), (256, 32)])
def test_tree_attention_ends_at_the_columns_of_a_table(dim, page, dtype):
    t = Trees([(6, 40), (4, 20)], 4, 2, dim, page, dtype, seed=dim)
    view = within_a_wider_one(t.table, t.pages)
    want = t.want(0.2)
    out, flag = t.run(0.2, table=view)
    assert flag == 0
    t.check(out, want)
    places = t.table.shape[1] * page
    for span, nodes in ((0, slice(0, 6)), (1, slice(6, 10))):
        for behind in (1, 2, page, 4 * page):                 # the neighbours in this row, and the next row's first
            t.context = [40, 20]
            t.context[span] = places - t.nodes[span] + behind
            out, flag = t.run(0.2, table=view)
            assert flag == 2 and bool((out[nodes] == 7.0).all())
            whole = want.copy()
            whole[nodes] = 7.0
            t.check(out, whole)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_kept_drafts_end_at_the_columns_of_a_table(dtype):
    """The path's third row lies behind the table's row: it stays, and so does the page that the neighbouring column names."""
    from celeg_b200 import kernels
    rng = np.random.default_rng(1)
    k, v = caches(2, 9, 2, 16, 24, 24, dtype, rng)
    want = k.clone(), v.clone()
    table = np.array([[3, 7, 1], [2, 4, 6]], dtype=np.int32)
    view = within_a_wider_one(table, 9)
    parents, tokens, chosen = i32([-1, 0, 0, 0, 2, -1, 0]), i32([0, 9, 5, 9, 6, 0, 1]), i32([5, 0, 6, 0, 8, 3, 4])
    path, accepted, following = (torch.zeros(shape, dtype=I32, device="cuda") for shape in ((2, 5), (2,), (2,)))
    flag = torch.zeros(1, dtype=I32, device="cuda")
    kernels.keep_drafts(k, v, parents, tokens, chosen, i32([0, 5, 7]), i32([44, 3]), view, 2, 5, path, accepted, following, flag)
    assert path.tolist() == [[0, 2, 4, -1, -1], [0, -1, -1, -1, -1]] and accepted.tolist() == [3, 1] and following.tolist() == [8, 3]
    assert int(flag.item()) == 1
    for got, cache in zip((k, v), want):
        cache[:, 1, :, 13] = cache[:, 1, :, 14]               # place 46 to 45; 48 is behind the row
        assert torch.equal(got, cache)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tables_whose_rows_are_one_and_tables_of_one_column(dtype):
    """Two spans that read the same pages through one row; and one page each, from a table that was stored by columns."""
    t = Trees([(6, 40), (6, 40)], 4, 2, 64, 16, dtype, seed=2)
    t.table[1] = t.table[0]
    out, flag = t.run(0.2, table=i32(t.table[:1]).expand(2, -1))
    assert flag == 0
    t.check(out, t.want(0.2))
    t = Trees([(6, 9), (4, 12), (1, 0)], 4, 2, 64, 16, dtype, seed=2)
    assert t.table.shape == (3, 1)
    for table in (i32(t.table.reshape(1, 3)).t(), i32(np.repeat(t.table, 4, 1))[:, :1]):
        out, flag = t.run(0.2, table=table)
        assert flag == 0
        t.check(out, t.want(0.2))
