"""Attention of drafted trees, kept paths, page copies and log probabilities against float64."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import plain_drafts as plain

pytestmark = pytest.mark.gpu

I32 = torch.int32


def i32(x):
    return torch.tensor(np.ascontiguousarray(x, dtype=np.int32), device="cuda")


def rounded(shape, rng, dtype, scale=1.0):
    return torch.tensor(rng.normal(size=shape) * scale, dtype=torch.float32).to(dtype)


class Trees:
    """A step's trees over a random cache, on the host in the operator's type and on the device."""

    def __init__(self, spans, heads, kv_heads, dim, page, dtype, seed, layers=1, max_nodes=None, words=None, value_scale=1.0):
        """``spans``: (nodes, context) of each."""
        rng = np.random.default_rng(seed)
        self.spans, self.heads, self.kv_heads, self.dim, self.page, self.dtype = spans, heads, kv_heads, dim, page, dtype
        self.nodes = [n for n, _ in spans]
        self.context = [c for _, c in spans]
        self.begin = np.concatenate([[0], np.cumsum(self.nodes)]).astype(np.int32)
        self.total = int(self.begin[-1])
        self.max_nodes = max_nodes or max(max(self.nodes), 1)
        words = words or (self.max_nodes + 31) // 32
        self.table, self.pages = plain.block_tables([n + c for n, c in spans], page, rng)
        self.parents = [plain.random_parents(n, rng) for n in self.nodes]
        self.seen, self.positions = [], []
        for up, c in zip(self.parents, self.context):
            seen, depth = plain.closure(up)
            self.seen.append(seen)
            self.positions.append(c + depth)
        self.masks = np.concatenate([plain.mask_words(s, words) for s in self.seen]) if self.total else np.zeros((0, words), np.int32)
        self.k = rounded((self.pages, kv_heads, page, dim), rng, dtype)
        self.v = rounded((self.pages, kv_heads, page, dim), rng, dtype, value_scale)
        self.q = rounded((self.total, (heads + 2 * kv_heads) * dim), rng, dtype)
        self.rng = rng

    def want(self, scale, window=0, sinks=None, softcap=0.0):
        out = np.zeros((self.total, self.heads, self.dim))
        k, v = self.k.double().numpy(), self.v.double().numpy()
        for s, (n, c) in enumerate(self.spans):
            a, b = self.begin[s], self.begin[s + 1]
            q = self.q[a:b, :self.heads * self.dim].double().numpy().reshape(n, self.heads, self.dim)
            out[a:b] = plain.attention(q, plain.gather(k, self.table[s], n + c), plain.gather(v, self.table[s], n + c), self.seen[s],
                                       self.positions[s], c, scale, window, sinks, softcap)
        return out

    def run(self, scale, window=0, sinks=None, softcap=0.0, scratch=None, out=None, q=None, max_keys=None, k=None, v=None,
            table=None):
        from celeg_b200 import kernels
        out = torch.full((self.total + 2, self.heads * self.dim), 7.0, dtype=self.dtype, device="cuda") if out is None else out
        flag = torch.zeros(1, dtype=I32, device="cuda")
        q = self.q.cuda() if q is None else q
        k, v = (self.k.cuda(), self.v.cuda()) if k is None else (k, v)
        kernels.attention_tree(q, q.stride(0), out, k, v, i32(np.concatenate(self.positions)), i32(self.begin), i32(self.context),
                               i32(self.masks), i32(self.table) if table is None else table, self.total, len(self.spans),
                               self.max_nodes, max_keys if max_keys is not None else max(n + c for n, c in self.spans), self.heads,
                               self.kv_heads, self.dim, self.page, window, scale, scratch, flag,
                               sinks=None if sinks is None else torch.tensor(sinks, dtype=torch.float32, device="cuda"), softcap=softcap)
        return out, int(flag.item())

    def check(self, out, want):
        got = out[:self.total].double().cpu().numpy().reshape(want.shape)
        most = float(self.v[torch.isfinite(self.v)].abs().max())
        if self.dtype == torch.float32:
            # scores are sums of `dim` products (each rounding at most 2^-24 of partial sums below dim), the weighted sum one of
            # non-negative weights: relative errors of the weights up to dim 2^-24 + 2^-21 of exponentials, times values
            bound = most * (self.dim * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -23 * np.abs(want)
        else:
            # weights rounded to bfloat16 (2^-8 of each at most, numerator and denominator), the output once more
            bound = 2.0 ** -8 * (np.abs(want) + most * 0.5)
        error = np.abs(got - want)
        assert (error <= bound).all(), (error - bound).max()
        assert bool((out[self.total:] == 7.0).all()), "rows behind the last span were written"


SHAPES = [(4, 1, 64, 16), (8, 2, 64, 16), (6, 2, 128, 16), (3, 3, 40, 12), (5, 1, 20, 5), (16, 1, 64, 32), (2, 1, 256, 16), (7, 1, 96, 8), (24, 8, 64, 16)]
SPANS = {
    "one": [(1, 0)],
    "edges": [(1, 63), (5, 64), (13, 0), (31, 65), (2, 1)],
    "wide": [(33, 100), (64, 300), (100, 17)],
    "long": [(9, 1500), (3, 40)],
    "empty_between": [(4, 20), (0, 5), (6, 33)],
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spans", SPANS)
@pytest.mark.parametrize("shape", SHAPES)
def test_tree_attention(shape, spans, dtype):
    heads, kv_heads, dim, page = shape
    t = Trees(SPANS[spans], heads, kv_heads, dim, page, dtype, seed=heads * 100 + dim)
    scale = dim ** -0.5
    from celeg_b200 import kernels
    for scratch in (None, kernels.attention_tree_scratch("cuda")):
        out, flag = t.run(scale, scratch=scratch)
        assert flag == 0
        t.check(out, t.want(scale))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window,sinks,softcap", [(1, False, 0.0), (7, True, 0.0), (64, False, 5.0), (400, True, 2.0), (0, True, 0.0), (0, False, 20.0)])
@pytest.mark.parametrize("shape", [(8, 2, 64, 16), (4, 1, 128, 8), (3, 3, 40, 12)])
def test_tree_attention_window_sinks_cap(shape, window, sinks, softcap, dtype):
    heads, kv_heads, dim, page = shape
    t = Trees([(20, 500), (3, 0), (40, 129), (1, 64)], heads, kv_heads, dim, page, dtype, seed=window + dim)
    values = t.rng.normal(size=heads).astype(np.float32) if sinks else None
    if window:       # pages that no node's window reaches have been given back
        for s, c in enumerate(t.context):
            t.table[s, :max(0, c - window + 1) // page] = -1
    from celeg_b200 import kernels
    for scratch in (None, kernels.attention_tree_scratch("cuda")):
        out, flag = t.run(dim ** -0.5, window, values, softcap, scratch=scratch)
        assert flag == 0
        t.check(out, t.want(dim ** -0.5, window, values, softcap))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("context", [0, 70])
@pytest.mark.parametrize("dim", [64, 128, 40])
def test_tree_attention_masks_of_any_kind(context, dim, dtype):
    """Masks that are no trees: random ones, and rows that see no node at all."""
    t = Trees([(70, context)], 4, 2, dim, 16, dtype, seed=dim)
    t.seen[0] = t.rng.random((70, 70)) < 0.3
    t.seen[0][5] = False
    t.seen[0][69] = False
    t.masks = plain.mask_words(t.seen[0], 3)
    for scratch in (None, torch.empty(1 << 22, device="cuda")):
        out, flag = t.run(0.2, scratch=scratch)
        assert flag == 0
        want = t.want(0.2)
        t.check(out, want)
        if context == 0:
            assert bool((out[5] == 0).all()) and bool((out[69] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim", [64, 128, 40])
def test_tree_attention_what_a_row_does_not_see_cannot_reach_it(dim, bad, dtype):
    """Numbers that are not finite in another branch's keys and values, in places behind the last node and before the window."""
    t = Trees([(12, 37), (40, 90)], 4, 2, dim, 16, dtype, seed=3)
    window = 50
    for s, (n, c) in enumerate(t.spans):
        leaf = n - 1
        t.seen[s][:leaf, leaf] = False                       # nobody but itself sees the last node
        for place in (c + leaf, c + n, c + n + 1):
            if place // 16 < t.table.shape[1] and t.table[s, place // 16] >= 0:
                t.k[t.table[s, place // 16], :, place % 16] = bad
                t.v[t.table[s, place // 16], :, place % 16] = bad
        first = c - window + 1
        for place in range(max(0, first)):
            t.k[t.table[s, place // 16], :, place % 16] = bad
            t.v[t.table[s, place // 16], :, place % 16] = bad
    t.masks = np.concatenate([plain.mask_words(x, 2) for x in t.seen])
    for scratch in (None, torch.empty(1 << 22, device="cuda")):
        out, flag = t.run(dim ** -0.5, window, scratch=scratch)
        assert flag == 0
        leaves = [t.begin[1] - 1, t.begin[2] - 1]
        with np.errstate(all="ignore"):
            want = t.want(dim ** -0.5, window)
        keep = np.setdiff1d(np.arange(t.total), leaves)
        got = out.double().cpu().numpy()
        assert np.isfinite(got[keep]).all()
        for row in leaves:                                   # ... and what it sees does
            assert not np.isfinite(got[row]).any()
        want[leaves] = 0.0
        out[leaves] = 0.0
        t.check(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tree_attention_only_a_value_is_not_finite(dtype):
    """Infinite and NaN values under finite scores: a row that sees one has it in that column, the others have not."""
    t = Trees([(10, 30)], 4, 1, 64, 16, dtype, seed=8)
    for node, column, bad in ((3, 5, float("inf")), (4, 5, float("nan")), (6, 9, -float("inf"))):
        place = 30 + node
        t.v[t.table[0, place // 16], 0, place % 16, column] = bad
    out, flag = t.run(0.125)
    assert flag == 0
    got = out[:10].double().cpu().numpy().reshape(10, 4, 64)
    with np.errstate(all="ignore"):
        want = t.want(0.125)
    for kind in (np.isnan, np.isposinf, np.isneginf):
        assert np.array_equal(kind(got), kind(want)), kind
    bad = ~np.isfinite(want)
    want[bad] = 0.0
    got[bad] = 0.0
    assert np.abs(got - want).max() < 0.03


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_tree_attention_scores_that_grow_and_outliers(dim, dtype):
    """Maxima that grow with every tile, and a first key far above the others."""
    t = Trees([(16, 700), (16, 700)], 8, 2, dim, 16, dtype, seed=5)
    for i, place in enumerate(range(0, 716)):
        page = t.table[0, place // 16]
        t.k[page, :, place % 16] = (t.q[0, :dim].float() * (i / 716.0) * 3.0 / dim ** 0.5).to(dtype)
    t.k[t.table[1, 0], :, 0] = (t.q[t.begin[1], :dim].float() * 2.0).to(dtype)
    for scratch in (None, torch.empty(1 << 22, device="cuda")):
        out, flag = t.run(dim ** -0.5 * 2.0, scratch=scratch)
        assert flag == 0
        t.check(out, t.want(dim ** -0.5 * 2.0))


def test_tree_attention_bad_pages_and_sizes_are_reported():
    t = Trees([(6, 40), (4, 20)], 4, 1, 64, 16, torch.bfloat16, seed=1)
    good, _ = t.run(0.125)
    table = t.table.copy()
    for page in (-1, t.pages, 1 << 30):
        t.table = table.copy()
        t.table[0, 1] = page
        out, flag = t.run(0.125)
        assert flag == 2 and torch.equal(out[6:10], good[6:10])
    t.table = table
    begin = t.begin.copy()
    for bad in ([0, 6, 11], [0, -1, 10], [0, 10, 10]):        # past the tokens, backwards, more nodes than max_nodes
        t.begin = np.array(bad, dtype=np.int32)
        _, flag = t.run(0.125, out=torch.zeros((12, 256), dtype=torch.bfloat16, device="cuda"))
        assert flag == 4
    t.begin = begin
    t.context = [-1, 20]
    _, flag = t.run(0.125)
    assert flag == 4


def test_tree_attention_same_bits_again_on_another_stream_and_in_a_graph():
    t = Trees([(32, 900), (20, 333)], 8, 2, 64, 16, torch.bfloat16, seed=2)
    from celeg_b200 import kernels
    scratch = kernels.attention_tree_scratch("cuda")
    first, _ = t.run(0.125, scratch=scratch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, _ = t.run(0.125, scratch=scratch)
    side.synchronize()
    assert torch.equal(first, again)
    q, k, v, out = t.q.cuda(), t.k.cuda(), t.v.cuda(), torch.zeros_like(first)
    fixed = [i32(np.concatenate(t.positions)), i32(t.begin), i32(t.context), i32(t.masks), i32(t.table)]
    flag = torch.zeros(1, dtype=I32, device="cuda")

    def call():
        kernels.attention_tree(q, q.stride(0), out, k, v, *fixed, t.total, 2, t.max_nodes, 1000, 8, 2, 64, 16, None, 0.125, scratch, flag)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    out.zero_()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[:t.total], first[:t.total])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [33, 34, 64])
def test_tree_attention_scratch_of_any_size_and_address(dim, dtype):
    """Odd numbers of pieces of odd heads, scratch that begins anywhere and holds hardly anything."""
    from celeg_b200 import kernels
    whole = kernels.attention_tree_scratch("cuda")
    for context in (130, 330, 500, 700):
        t = Trees([(1, context)], 1, 1, dim, 16, dtype, seed=context)
        want = t.want(0.2)
        for offset, size in ((0, 1 << 20), (1, 1 << 20), (2, 1 << 20), (3, 200), (1, 3), (2, 0), (1, 3 * (dim + 2)), (0, 5 * (dim + 2))):
            out, flag = t.run(0.2, scratch=whole[offset:offset + size])
            assert flag == 0
            t.check(out, want)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 3, 8, 64, 128, 256])
def test_tree_attention_pages_of_all_sizes(page, dim):
    t = Trees([(5, 2100), (40, 700), (2, 63)], 4, 2, dim, page, torch.bfloat16, seed=page + dim)
    out, flag = t.run(dim ** -0.5)
    assert flag == 0
    t.check(out, t.want(dim ** -0.5))
    t.table[0, 3] = t.pages                                  # a page that is missing is reported by all forms
    assert t.run(dim ** -0.5)[1] == 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window,sinks,softcap", [(0, True, 0.0), (33, False, 0.0), (500, True, 30.0)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 64), (16, 2, 128), (16, 1, 80), (16, 2, 256), (12, 2, 136)])
def test_tree_attention_of_many_rows(heads, kv_heads, dim, window, sinks, softcap, dtype):
    """More rows than a tile of either size, the last one nearly empty."""
    t = Trees([(40, 500), (33, 0), (17, 129)], heads, kv_heads, dim, 16, dtype, seed=window + dim)
    values = t.rng.normal(size=heads).astype(np.float32) if sinks else None
    if window:
        for s, c in enumerate(t.context):
            t.table[s, :max(0, c - window + 1) // 16] = -1
    out, flag = t.run(dim ** -0.5, window, values, softcap)
    assert flag == 0
    t.check(out, t.want(dim ** -0.5, window, values, softcap))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,dim,nodes", [(4, 64, 3), (4, 128, 3), (2, 256, 5), (4, 72, 3), (32, 64, 8), (32, 128, 8)])
def test_tree_attention_of_few_rows_over_many_positions(heads, dim, nodes, dtype):
    """Cut into more pieces than a cluster holds; and into as many as it holds, or as scratch does."""
    from celeg_b200 import kernels
    t = Trees([(nodes, 20011)], heads, 1, dim, 16, dtype, seed=dim + heads)
    values = t.rng.normal(size=heads).astype(np.float32)
    want = t.want(dim ** -0.5, 0, values)
    for scratch in (None, kernels.attention_tree_scratch("cuda"), torch.empty(11 * t.total * heads * (dim + 2), device="cuda")):
        out, flag = t.run(dim ** -0.5, 0, values, scratch=scratch)
        assert flag == 0
        t.check(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tree_attention_of_256_nodes_and_of_many_spans(dtype):
    t = Trees([(256, 300), (1, 5)], 4, 2, 64, 16, dtype, seed=1, words=11)
    out, flag = t.run(0.125)
    assert flag == 0
    t.check(out, t.want(0.125))
    t = Trees([(i % 3, i % 41) for i in range(400)], 4, 2, 64, 16, dtype, seed=2)
    out, flag = t.run(0.125, max_keys=0)                     # (max_keys is a hint)
    assert flag == 0
    t.check(out, t.want(0.125))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_tree_attention_strides_and_shared_pages(dim, dtype):
    """Queries at odd addresses, a table that is part of a wider one, caches that are part of larger pages; and two spans that
    share their first pages."""
    t = Trees([(12, 200), (9, 230)], 4, 2, dim, 16, dtype, seed=4)
    t.table[1, :12] = t.table[0, :12]
    want = t.want(0.1)
    wide_q = torch.zeros((t.total, t.q.shape[1] + 5), dtype=dtype, device="cuda")
    wide_table = torch.full((2, t.table.shape[1] + 7), -1, dtype=I32, device="cuda")
    wide_table[:, 3:3 + t.table.shape[1]] = i32(t.table)
    large_k, large_v = (torch.full((t.pages, 5, 16, dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    large_k[:, 1:3], large_v[:, 1:3] = t.k.cuda(), t.v.cuda()
    for offset in (0, 1, 4, 5):
        q = wide_q[:, offset:offset + t.q.shape[1]]
        q.copy_(t.q)
        out, flag = t.run(0.1, q=q, table=wide_table[:, 3:], k=large_k[:, 1:3], v=large_v[:, 1:3])
        assert flag == 0
        t.check(out, want)


def test_tree_attention_contexts_past_the_table_are_refused():
    """... with their rows left alone, and nothing behind the table read, whatever the context is."""
    for dtype in (torch.float32, torch.bfloat16):
        t = Trees([(6, 40), (4, 20)], 4, 1, 64, 16, dtype, seed=1)
        good, _ = t.run(0.125)
        places = t.table.shape[1] * 16
        for context in (places - 5, places, 1 << 30, 2 ** 31 - 1100, 2 ** 31 - 300, 2 ** 31 - 2, 2 ** 31 - 1):
            t.context = [context, 20]
            out, flag = t.run(0.125)
            assert flag == 2 and torch.equal(out[6:10], good[6:10]) and bool((out[:6] == 7.0).all())


def test_tree_attention_two_calls_at_once():
    from celeg_b200 import kernels
    t = Trees([(9, 20011)], 4, 1, 64, 16, torch.bfloat16, seed=2)
    scratch = [kernels.attention_tree_scratch("cuda") for _ in range(2)]
    want, _ = t.run(0.125, scratch=scratch[0])
    q, k, v = t.q.cuda(), t.k.cuda(), t.v.cuda()
    fixed = [i32(np.concatenate(t.positions)), i32(t.begin), i32(t.context), i32(t.masks), i32(t.table)]
    flag = torch.zeros(1, dtype=I32, device="cuda")
    outs = [torch.zeros((9, 256), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, out, own in zip(streams, outs, scratch):
            with torch.cuda.stream(stream):
                kernels.attention_tree(q, q.stride(0), out, k, v, *fixed, 9, 1, 9, 20020, 4, 1, 64, 16, None, 0.125, own, flag)
    torch.cuda.synchronize()
    assert int(flag.item()) == 0
    for out in outs:
        assert torch.equal(out, want[:9])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_caches_larger_than_32_bit_offsets(dtype):
    """Pages behind the first 2^32 elements: read by attention, moved by keep_drafts, copied."""
    from celeg_b200 import kernels
    t = Trees([(12, 200), (9, 1300)], 16, 8, 64, 16, dtype, seed=6)
    per_page = 8 * 16 * 64
    pages = (1 << 32) // per_page + t.pages + 100
    large = [torch.empty((1, pages, 8, 16, 64), dtype=dtype, device="cuda") for _ in range(2)]
    at = pages - t.pages
    large[0][0, at:], large[1][0, at:] = t.k.cuda(), t.v.cuda()
    table = i32(np.where(t.table >= 0, t.table + at, -1))
    want, _ = t.run(0.125)
    got, flag = t.run(0.125, k=large[0][0], v=large[1][0], table=table)
    assert flag == 0 and torch.equal(got, want)
    small = [t.k.cuda()[None].clone(), t.v.cuda()[None].clone()]
    tokens, chosen = (t.rng.integers(0, 2, t.total) for _ in range(2))
    results = []
    for (k, v), rows in ((small, i32(t.table)), (large, table)):
        path, accepted, following = (torch.zeros(shape, dtype=I32, device="cuda") for shape in ((2, 12), (2,), (2,)))
        flag = torch.zeros(1, dtype=I32, device="cuda")
        kernels.keep_drafts(k, v, i32(np.concatenate(t.parents)), i32(tokens), i32(chosen), i32(t.begin), i32(t.context), rows, 2, 12, path,
                            accepted, following, flag)
        first = 0 if k is small[0] else at
        kernels.copy_pages(k, v, [(first + int(t.table[1, 2]), first + int(t.table[0, 1]), 11)])
        assert int(flag.item()) == 0
        results.append((path.tolist(), accepted.tolist(), following.tolist()))
    assert results[0] == results[1]
    for one, other in zip(small, large):
        assert torch.equal(one[0], other[0, at:])


# ------------------------------------------------------------------------------------------- kept drafts, pages
def caches(layers, pages, heads, page, dim, value_dim, dtype, rng):
    make = lambda d: torch.tensor(rng.normal(size=(layers, pages, heads, page, d)), dtype=torch.float32).to(dtype).cuda()      # noqa: E731
    return make(dim), make(value_dim)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,page,dim,value_dim", [(2, 16, 64, 64), (1, 5, 20, 12), (3, 8, 7, 7), (1, 16, 128, 0)])
@pytest.mark.parametrize("alphabet", [1, 2, 3])
def test_keep_drafts(alphabet, heads, page, dim, value_dim, dtype):
    from celeg_b200 import kernels
    rng = np.random.default_rng(dim + alphabet)
    spans = [(13, 40), (1, 0), (0, 9), (64, 17), (200, 3), (30, 15)]
    nodes = [n for n, _ in spans]
    begin = np.concatenate([[0], np.cumsum(nodes)])
    table, pages = plain.block_tables([n + c for n, c in spans], page, rng)
    parents = [plain.random_parents(n, rng) for n in nodes]
    tokens, chosen = (rng.integers(0, alphabet, begin[-1]).astype(np.int32) for _ in range(2))
    k, v = caches(3, pages, heads, page, dim, value_dim, dtype, rng)
    want_k, want_v = k.clone(), v.clone()
    max_nodes = 203
    want_path = np.full((len(spans), max_nodes), -1)
    want_count, want_next = [], []
    for s, (n, c) in enumerate(spans):
        part = slice(begin[s], begin[s + 1])
        path, following = plain.accepted_path(parents[s], tokens[part], chosen[part])
        want_path[s, :len(path)] = path
        want_count.append(len(path))
        want_next.append(following)
        for at, node in enumerate(path):
            for cache in (want_k, want_v):
                cache[:, table[s, (c + at) // page], :, (c + at) % page] = cache[:, table[s, (c + node) // page], :, (c + node) % page].clone()
    path, accepted, following = (torch.full(shape, 99, dtype=I32, device="cuda") for shape in ((6, max_nodes), (7,), (7,)))
    flag = torch.zeros(1, dtype=I32, device="cuda")
    kernels.keep_drafts(k, v, i32(np.concatenate(parents)), i32(tokens), i32(chosen), i32(begin), i32([c for _, c in spans]), i32(table),
                        6, max_nodes, path, accepted, following, flag)
    assert int(flag.item()) == 0
    assert path.tolist() == want_path.tolist()
    assert accepted.tolist() == want_count + [99] and following.tolist() == want_next + [99]
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_keep_drafts_a_chain_of_256_and_bad_tables():
    from celeg_b200 import kernels
    rng = np.random.default_rng(0)
    k, v = caches(1, 20, 1, 16, 8, 8, torch.bfloat16, rng)
    before = k.clone()
    parents = np.arange(-1, 255)
    path, accepted, following = (torch.zeros(shape, dtype=I32, device="cuda") for shape in ((1, 256), (1,), (1,)))
    flag = torch.zeros(1, dtype=I32, device="cuda")
    tokens = np.arange(256)
    args = lambda table, begin=(0, 256), context=30: (k, v, i32(parents), i32(tokens), i32(tokens + 1), i32(begin), i32([context]),    # noqa: E731
                                                      i32(table), 1, 256, path, accepted, following, flag)
    table = np.arange(20)[None]
    kernels.keep_drafts(*args(table))
    assert int(flag.item()) == 0 and path[0].tolist() == list(range(256)) and accepted.item() == 256 and following.item() == 256
    assert torch.equal(k, before)                              # (every row is in its place)
    # every second node is off the path: pages that are missing are reported, nothing outside is touched
    parents = np.array([-1] + [max(0, (i - 1) // 2 * 2 if i % 2 else i - 2) for i in range(1, 256)])
    tokens = np.array([i // 2 if i % 2 == 0 else 1000 for i in range(256)])
    kernels.keep_drafts(k, v, i32(parents), i32(tokens), i32(np.arange(256) // 2 + 1), i32([0, 256]), i32([30]),
                        i32(np.where(table % 2 == 0, table, 77)), 1, 256, path, accepted, following, flag)
    assert int(flag.item()) == 1 and accepted.item() == 128
    flag.zero_()
    kernels.keep_drafts(*args(table, begin=(0, 300)))
    assert int(flag.item()) == 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,page,dim,value_dim,count", [(2, 16, 64, 64, 1), (1, 5, 20, 12, 40), (3, 8, 7, 7, 9), (1, 16, 128, 0, 3), (2, 4, 8, 8, 1500)])
def test_copy_pages(heads, page, dim, value_dim, count, dtype):
    from celeg_b200 import kernels
    rng = np.random.default_rng(count)
    k, v = caches(2, count * 2 + 3, heads, page, dim, value_dim, dtype, rng)
    want = [k.clone(), v.clone()]
    order = rng.permutation(count * 2 + 3)
    moves = [(int(order[0 if i % 3 == 0 else i]), int(order[count + i]), int(rng.integers(0, page + 1)) if i % 2 else page) for i in range(count)]
    for cache in want:
        for source, target, rows in moves:
            cache[:, target, :, :rows] = cache[:, source, :, :rows]
    kernels.copy_pages(k, v, moves)
    kernels.copy_pages(k, v, [])
    kernels.copy_pages(k, v, [(2, 2, page)])                   # a page onto itself
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_keep_drafts_refused_spans_have_no_path():
    from celeg_b200 import kernels
    rng = np.random.default_rng(0)
    k, v = caches(1, 20, 1, 16, 8, 8, torch.bfloat16, rng)
    before = k.clone(), v.clone()
    for begin, context in (((0, 5, 9), (2 ** 31 - 1, 3)), ((0, 5, 9), (-1, 3)), ((0, 5, 9), (2 ** 31 - 200, 3)), ((0, 11, 12), (0, 3))):
        path, accepted, following = (torch.full(shape, 99, dtype=I32, device="cuda") for shape in ((2, 10), (2,), (2,)))
        flag = torch.zeros(1, dtype=I32, device="cuda")
        tokens = np.zeros(12, dtype=np.int32)
        kernels.keep_drafts(k, v, i32([-1, 0, 0, 0, 0, -1, 0, 0, 0, 0, 0, -1]), i32(tokens), i32(tokens + 1), i32(begin), i32(context),
                            i32(np.arange(20)[None].repeat(2, 0)), 2, 10, path, accepted, following, flag)
        assert int(flag.item()) == 4
        assert path[0].tolist() == [-1] * 10 and accepted.tolist() == [0, 1] and following.tolist() == [-1, 1]
        assert path[1].tolist() == [0] + [-1] * 9
    # parents that are no tree: only children behind their parent count
    tokens = i32([5, 5, 5, 5])
    kernels.keep_drafts(k, v, i32([3, 1, 0, 9]), tokens, tokens, i32([0, 4]), i32([0]), i32(np.arange(20)[None]), 1, 10, path, accepted,
                        following, flag)
    assert path[0].tolist() == [0, 2] + [-1] * 8
    before[0][0, 0, :, 1], before[1][0, 0, :, 1] = before[0][0, 0, :, 2], before[1][0, 0, :, 2]
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])


def test_pages_and_scores_in_a_graph_on_another_stream():
    from celeg_b200 import kernels
    rng = np.random.default_rng(3)
    k, v = caches(2, 40, 2, 16, 64, 64, torch.bfloat16, rng)
    start = k.clone(), v.clone()
    parents, tokens = i32([-1, 0, 0, 2, 3, 3]), i32([9, 1, 2, 3, 4, 5])
    chosen, begin, context, table = i32([2, 0, 3, 5, 0, 7]), i32([0, 6]), i32([30]), i32([[4, 9, 2]])
    path, accepted, following = (torch.zeros(shape, dtype=I32, device="cuda") for shape in ((1, 6), (1,), (1,)))
    flag = torch.zeros(1, dtype=I32, device="cuda")
    logits = torch.randn((6, 30000), device="cuda")
    outs = [torch.zeros(6, device="cuda"), torch.zeros(6, device="cuda"), torch.zeros((6, 3), device="cuda"),
            torch.zeros((6, 3), dtype=I32, device="cuda")]

    def call():
        kernels.token_logprobs(logits, 6, tokens, *outs)
        kernels.keep_drafts(k, v, parents, tokens, chosen, begin, context, table, 1, 6, path, accepted, following, flag)
        kernels.copy_pages(k, v, [(4, 20, 16), (9, 21, 3)])

    call()
    torch.cuda.synchronize()
    want = [x.clone() for x in (k, v, path, accepted, following, *outs)]
    assert path.tolist() == [[0, 2, 3, 5, -1, -1]] and following.item() == 7
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    for _ in range(2):
        k.copy_(start[0]), v.copy_(start[1])
        for x in (path, accepted, following, *outs):
            x.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        for x, y in zip((k, v, path, accepted, following, *outs), want):
            assert torch.equal(x, y)


# --------------------------------------------------------------------------------------------- log probabilities
def score(logits, tokens, top, rows=None):
    from celeg_b200 import kernels
    rows = logits.shape[0] if rows is None else rows
    logprobs, entropy = torch.full((rows + 1,), 9.0, device="cuda"), torch.full((rows + 1,), 9.0, device="cuda")
    top_logprobs, top_tokens = torch.full((rows, top), 9.0, device="cuda"), torch.full((rows, top), -5, dtype=I32, device="cuda")
    kernels.token_logprobs(logits, rows, i32(tokens), logprobs, entropy, top_logprobs, top_tokens)
    assert logprobs[rows] == 9.0 and entropy[rows] == 9.0
    return logprobs[:rows].double().cpu().numpy(), entropy[:rows].double().cpu().numpy(), top_logprobs.double().cpu().numpy(), top_tokens.cpu().numpy()


@np.errstate(invalid="ignore")
def check_scores(logits, tokens, top):
    got, entropy, top_logprobs, top_tokens = score(logits, tokens, top)
    x = logits.double().cpu().numpy()
    for r in range(x.shape[0]):
        log_p, want_entropy = plain.log_probabilities(x[r])
        # x - m is rounded once (2^-24 of it), the sum of exponentials is off by 2^-21 of itself at most (exponentials 2^-22,
        # their sums by lanes), one rounding of the result; the entropy's sum likewise
        bound = 2.0 ** -22 * np.abs(log_p).clip(max=1e30) + 2.0 ** -21 * min(1.0, max(want_entropy, 2.0 ** -30)) + 1e-30
        assert abs(got[r] - log_p[tokens[r]]) <= bound[tokens[r]], (r, got[r], log_p[tokens[r]])
        assert abs(entropy[r] - want_entropy) <= 2.0 ** -19 * want_entropy + 1e-30, (r, entropy[r], want_entropy)
        order = plain.best(x[r], top)
        assert top_tokens[r].tolist() == order.tolist(), r
        wanted = log_p[order]
        out_of_reach = np.isneginf(wanted)
        assert np.array_equal(np.isneginf(top_logprobs[r]), out_of_reach)
        assert (np.abs(top_logprobs[r] - wanted)[~out_of_reach] <= bound[order][~out_of_reach]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (2, 7, 7), (5, 300, 128), (1, 65536, 20), (2, 65537, 128), (33, 4099, 5), (700, 1000, 1), (1, 150001, 3), (64, 8192, 0)])
@pytest.mark.parametrize("spread", [0.0, 2.5, 40.0])
def test_token_logprobs(spread, rows, vocab, top, dtype):
    rng = np.random.default_rng(vocab + rows)
    logits = torch.tensor(rng.normal(size=(rows, vocab)) * spread + 3.0, dtype=torch.float32).to(dtype).cuda()
    check_scores(logits, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1000, 65536])
def test_token_logprobs_of_masked_and_peaked_rows(vocab, dtype):
    rng = np.random.default_rng(vocab)
    lowest = torch.finfo(dtype).min
    logits = torch.tensor(rng.normal(size=(8, vocab)), dtype=torch.float32).to(dtype)
    logits[0, 10:] = -float("inf")                    # a grammar that allows ten tokens
    logits[1, :vocab - 3] = lowest                    # ... or three, masked with the lowest number
    logits[2] = lowest                                # nothing but the lowest number: all alike
    logits[3, 77] = 60.0                              # nearly all weight on one
    logits[4, 5] = 17.0
    logits[5] = -float("inf")
    logits[5, vocab - 1] = -4.0                       # a single token
    logits[6, ::2] = 0.0                              # ties, with -0 among them
    logits[6, 1::2] = -0.0
    logits[7, 100:400] = 30.0                         # more equal ones than are asked for
    tokens = np.array([3, vocab - 2, 12, 77, 5, vocab - 1, 8, 120])
    check_scores(logits.cuda(), tokens, 9)


def test_token_logprobs_strides_and_large_logits_in_few_threads():
    """Rows at odd strides and offsets; and large logits 1,024 apart, which all lie with the same threads."""
    rng = np.random.default_rng(4)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.tensor(rng.normal(size=(6, 5003)), dtype=torch.float32).to(dtype).cuda()
        check_scores(wide[:, 3:4800], rng.integers(0, 4797, 6), 16)
        check_scores(wide[:, 1:2], np.zeros(6, dtype=int), 1)
        rows = torch.tensor(rng.normal(size=(300, 40960)), dtype=torch.float32).to(dtype).cuda()
        step = 1024 * (2 if dtype == torch.bfloat16 else 1)
        for offset in range(0, step, max(1, step // 128)):
            rows[:2, offset::step] += 20.0
        check_scores(rows[:2], rng.integers(0, 40960, 2), 128)
        full = score(rows, rng.integers(0, 40960, 300), 128)      # (one block a row)
        x = rows[:2].double().cpu().numpy()
        for r in range(2):
            assert full[3][r].tolist() == plain.best(x[r], 128).tolist()


def test_token_logprobs_rows_without_a_distribution():
    x = torch.zeros((5, 300), device="cuda")
    x[0] = -float("inf")
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    x[3] = float("nan")
    got, entropy, top_logprobs, top_tokens = score(x, [0, 1, 9, 3, -1], 4)
    assert np.isnan(got).all() and np.isnan(entropy[:4]).all() and np.isnan(top_logprobs[:4]).all()
    assert abs(entropy[4] - np.log(300)) < 1e-5
    assert top_tokens[0].tolist() == [0, 1, 2, 3] and top_tokens[1].tolist() == [0, 1, 2, 3]
    assert top_tokens[2].tolist() == [9, 0, 1, 2] and top_tokens[3].tolist() == [0, 1, 2, 3]
    got, *_ = score(x[4:], [300], 0)
    assert np.isnan(got).all()


def test_token_logprobs_rows_behind_32_bit_offsets():
    rows, vocab = 66000, 65541
    logits = torch.empty((rows, vocab), dtype=torch.bfloat16, device="cuda")
    logits[:-3] = 0.0
    logits[-3:] = torch.randn((3, vocab), device="cuda")
    from celeg_b200 import kernels
    tokens = torch.arange(rows, dtype=I32, device="cuda") % vocab
    logprobs, entropy = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    top_logprobs, top_tokens = torch.empty((rows, 2), device="cuda"), torch.empty((rows, 2), dtype=I32, device="cuda")
    kernels.token_logprobs(logits, rows, tokens, logprobs, entropy, top_logprobs, top_tokens)
    assert bool(((logprobs[:-3] + np.log(vocab)).abs() < 1e-5).all()) and bool(((entropy[:-3] - np.log(vocab)).abs() < 1e-4).all())
    assert bool((top_tokens[:-3] == torch.tensor([0, 1], device="cuda")).all())
    x = logits[-3:].double().cpu().numpy()
    for r in range(3):
        log_p, want = plain.log_probabilities(x[r])
        assert abs(logprobs[rows - 3 + r].item() - log_p[int(tokens[rows - 3 + r])]) < 1e-5
        assert abs(entropy[rows - 3 + r].item() - want) < 1e-4
        assert top_tokens[rows - 3 + r].tolist() == plain.best(x[r], 2).tolist()
