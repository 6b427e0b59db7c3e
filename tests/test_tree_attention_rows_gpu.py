"""Attention of drafted trees row by row: the error of a (node, query head)'s output relative to it, which a lost block of keys, piece or
key exceeds however long the context is.

Values are independent normal numbers. An output is sum(w v) / sum(w); weights that are rounded by shares d_i, |d_i| <= u, make its
error sum(w d v) / sum(w): the same form with coefficients that are smaller by u at least, so that over a row's columns its root
mean square is at most u times the output's. bfloat16: u = 2^-8, and the output is rounded by 2^-8 of itself once more: 2^-7 together
(uniform roundings are 3^-1/2 of that). float32: u from a score's sum of `dim` products and its exponential, as in
test_drafts_gpu.py, and one rounding of the output."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import plain_drafts as plain
from test_drafts_gpu import SHAPES, SPANS, Trees

pytestmark = pytest.mark.gpu


def limit(t):
    return 2.0 ** -7 if t.dtype == torch.bfloat16 else t.dim * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -24


def relative(got, want):
    """[nodes, heads]: the error's root mean square over a row's columns, relative to the row's."""
    size = np.sqrt((want ** 2).mean(-1))
    error = np.sqrt(((got - want) ** 2).mean(-1))
    assert (error[size == 0] == 0).all()
    return error / np.where(size == 0, 1.0, size)


def check(t, scale, window=0, sinks=None, softcap=0.0):
    from celeg_b200 import kernels
    want = t.want(scale, window, sinks, softcap)
    for scratch in (None, kernels.attention_tree_scratch("cuda")):
        out, flag = t.run(scale, window, sinks, softcap, scratch=scratch)
        assert flag == 0
        error = relative(out[:t.total].double().cpu().numpy().reshape(want.shape), want)
        assert error.max(initial=0.0) <= limit(t), error.max()
    return want


def without(t, span, first, behind, scale, sinks=None):
    """The rows of a span as they would be if these cached positions were lost."""
    n, c = t.spans[span]
    a, b = t.begin[span], t.begin[span + 1]
    keep = np.r_[0:first, behind:n + c]
    k, v = (plain.gather(x.double().numpy(), t.table[span], n + c)[keep] for x in (t.k, t.v))
    q = t.q[a:b, :t.heads * t.dim].double().numpy().reshape(n, t.heads, t.dim)
    return plain.attention(q, k, v, t.seen[span], t.positions[span], c - (behind - first), scale, 0, sinks, 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spans", SPANS)
@pytest.mark.parametrize("shape", SHAPES)
def test_rows(shape, spans, dtype):
    heads, kv_heads, dim, page = shape
    check(Trees(SPANS[spans], heads, kv_heads, dim, page, dtype, seed=heads * 10 + dim), dim ** -0.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,dim,nodes", [(4, 64, 3), (4, 128, 3), (2, 256, 5), (4, 72, 3), (32, 64, 8), (32, 128, 8)])
def test_rows_over_many_positions(heads, dim, nodes, dtype):
    """... and what the limit finds: a block of 64 keys, or a piece of the keys, that is lost."""
    t = Trees([(nodes, 20011)], heads, 1, dim, 16, dtype, seed=dim + heads)
    values = t.rng.normal(size=heads).astype(np.float32)
    want = check(t, dim ** -0.5, 0, values)
    for first, behind in ((0, 64), (64 * 37, 64 * 38), (64 * 100, 64 * 110), (20011 - 43, 20011)):
        assert relative(without(t, 0, first, behind, dim ** -0.5, values), want).min() > 2.0 * limit(t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window,sinks,softcap", [(7, True, 0.0), (64, False, 5.0), (400, True, 20.0), (0, True, 30.0)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (16, 1, 128), (16, 2, 256), (12, 2, 136), (3, 3, 20)])
def test_rows_under_windows_sinks_and_caps(heads, kv_heads, dim, window, sinks, softcap, dtype):
    t = Trees([(40, 500), (33, 0), (17, 129)], heads, kv_heads, dim, 16, dtype, seed=window + dim)
    check(t, dim ** -0.5, window, t.rng.normal(size=heads).astype(np.float32) if sinks else None, softcap)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_of_full_trees_and_ragged_requests(dim, dtype):
    check(Trees([(256, 300), (1, 5), (31, 64), (0, 9), (77, 1000)], 4, 2, dim, 16, dtype, seed=dim), dim ** -0.5)


def test_a_key_that_is_lost_is_found():
    """The limit itself, in float64: one key of seven hundred."""
    for dtype in (torch.float32, torch.bfloat16):
        t = Trees([(5, 700)], 4, 2, 64, 16, dtype, seed=1)
        want = t.want(0.125)
        for place in (0, 63, 350, 699):
            assert np.median(relative(without(t, 0, place, place + 1, 0.125), want)) > limit(t)
