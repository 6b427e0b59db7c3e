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

    def run(self, scale, window=0, sinks=None, softcap=0.0, scratch=None, out=None, q=None, stream=None, max_keys=None):
        from celeg_b200 import kernels
        out = torch.full((self.total + 2, self.heads * self.dim), 7.0, dtype=self.dtype, device="cuda") if out is None else out
        flag = torch.zeros(1, dtype=I32, device="cuda")
        q = self.q.cuda() if q is None else q
        kernels.attention_tree(q, q.stride(0), out, self.k.cuda(), self.v.cuda(), i32(np.concatenate(self.positions)),
                               i32(self.begin), i32(self.context), i32(self.masks), i32(self.table), self.total, len(self.spans),
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
