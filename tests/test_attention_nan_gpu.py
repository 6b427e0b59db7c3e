"""Attention over scores that are NaN: a row that sees one is NaN, however its keys are cut, and no other row is."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import plain_drafts as plain
from test_drafts_gpu import Trees

pytestmark = pytest.mark.gpu

NAN = float("nan")


def tree_outputs(t, scale, window=0, sinks=None):
    """Without scratch, and with room for all pieces."""
    from celeg_b200 import kernels
    for scratch in (None, kernels.attention_tree_scratch("cuda")):
        out, flag = t.run(scale, window, sinks, scratch=scratch)
        assert flag == 0
        yield out


def check_tree(t, out, want, rows):
    """``rows`` [nodes, heads]: which are NaN; the others as they would be."""
    got = out[:t.total].double().cpu().numpy().reshape(want.shape)
    assert np.isnan(got[rows]).all() and np.isfinite(got[~rows]).all()
    out = out.clone()
    out[:t.total] = torch.where(torch.from_numpy(rows).cuda()[:, :, None], 0.0, out[:t.total].view(want.shape)).reshape(t.total, -1)
    t.check(out, np.where(rows[:, :, None], 0.0, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spans", [[(3, 0), (2, 40)], [(5, 700), (9, 90)], [(7, 20011)], [(64, 300)]])
@pytest.mark.parametrize("heads,dim", [(4, 64), (4, 128), (4, 256), (4, 40)])
@pytest.mark.parametrize("sinks", [False, True])
def test_tree_attention_of_queries_with_nan(heads, dim, spans, dtype, sinks):
    t = Trees(spans, heads, 2, dim, 16, dtype, seed=dim)
    values = t.rng.normal(size=heads).astype(np.float32) if sinks else None
    want = t.want(dim ** -0.5, 0, values)
    rows = np.zeros((t.total, heads), dtype=bool)
    for node, head in ((0, 1), (t.total - 1, 0), (t.total // 2, heads - 1)):
        t.q[node, head * dim + 3] = NAN
        rows[node, head] = True
    for out in tree_outputs(t, dim ** -0.5, 0, values):
        check_tree(t, out, want, rows)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256, 40])
def test_tree_attention_of_a_root_whose_only_key_is_nan(dim, dtype):
    """No cached positions; the root sees itself alone, and nobody else sees it."""
    t = Trees([(5, 0)], 4, 2, dim, 16, dtype, seed=dim)
    t.seen[0][1:, 0] = False
    t.masks = plain.mask_words(t.seen[0], 1)
    want = t.want(0.2)
    t.k[t.table[0, 0], 0, 0] = NAN                    # of the first kv head: query heads 0 and 1
    rows = np.zeros((5, 4), dtype=bool)
    rows[0, :2] = True
    for out in tree_outputs(t, 0.2):
        check_tree(t, out, want, rows)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256, 40])
@pytest.mark.parametrize("context", [100, 130, 190, 250, 700, 20011])
def test_tree_attention_of_a_run_of_keys_that_are_all_nan(context, dim, dtype):
    """All keys that one piece holds, and all that one team or block takes; every row sees them."""
    t = Trees([(4, context), (3, 100)], 4, 2, dim, 16, dtype, seed=dim)
    want = t.want(dim ** -0.5)
    keep = t.k.clone()
    rows = np.zeros((7, 4), dtype=bool)
    rows[:4, 2:] = True                               # the second kv head's
    for first, behind in ((0, 64), (64, 128), (128, 192), (256, context // 2), (context - 30, context), (0, context)):
        if behind > context or first >= behind:
            continue
        t.k = keep.clone()
        for place in range(first, behind):
            t.k[t.table[0, place // 16], 1, place % 16] = NAN
        for out in tree_outputs(t, dim ** -0.5):
            check_tree(t, out, want, rows)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tree_attention_rows_that_see_nothing_are_zeros_still(dtype):
    """... beside rows of NaN, with sinks and without, in pieces and whole, and where all that is seen scores -inf."""
    for sinks in (None, np.array([0.5, -1.0, 30.0, 2.0], dtype=np.float32)):
        t = Trees([(70, 0)], 4, 2, 64, 16, dtype, seed=3)
        t.seen[0][9] = False
        t.seen[0][69] = False
        t.seen[0][33] = np.arange(70) == 33
        t.masks = plain.mask_words(t.seen[0], 3)
        t.q[33, :128], t.q[33, 128:256] = 1.0, NAN    # row 33: heads 0 and 1 score -inf, heads 2 and 3 NaN
        t.seen[0][:, 33] &= np.arange(70) == 33       # (nobody else sees it)
        t.masks = plain.mask_words(t.seen[0], 3)
        t.k[t.table[0, 2], 0, 1] = 0.0
        t.k[t.table[0, 2], 0, 1, 5] = -float("inf")
        for out in tree_outputs(t, 0.125, 0, sinks):
            assert bool((out[9] == 0).all()) and bool((out[69] == 0).all()) and bool((out[33, :128] == 0).all())
            assert bool(out[33, 128:].isnan().all()) and bool(out[:70].isfinite().any())
