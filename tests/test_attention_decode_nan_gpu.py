"""Decode attention over scores that are NaN: a row that sees one is NaN, however its keys are shared among warps and pieces."""
from __future__ import annotations

import pytest
import torch

from test_attention_generic_nan_gpu import Decoded, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("chunk", [64, 256, 1024])             # pieces; one stage a warp; two
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 2, 128), (16, 1, 96), (2, 1, 256)])
def test_decode_attention_of_scores_that_are_nan(heads, kv_heads, dim, sinks, chunk):
    from celeg_b200 import kernels
    lengths = [1, 33, 40, 100, 129, 700, 640, 128]
    d = Decoded(lengths, heads, kv_heads, dim, 16, torch.bfloat16, seed=dim + chunk)
    d.break_keys(0, 0, 1)                                      # a token's only key
    d.break_keys(1, 32, 33)                                    # one warp's only key
    d.break_query(2, heads - 1)
    d.break_keys(3, 0, 32)                                     # all keys of the first warp
    d.break_keys(4, 128, 129, kv_head=kv_heads - 1)            # a second tile of one key
    d.break_query(5, 0)
    d.break_keys(6, 256, 512)                                  # whole pieces
    tokens, splits = len(lengths), -(-max(lengths) // chunk)
    out, flag, counters = torch.zeros((tokens, heads * dim), dtype=torch.bfloat16, device="cuda"), i32([0]), i32([0] * tokens * kv_heads)
    scratch = torch.empty(tokens * heads * splits * dim, device="cuda"), torch.empty(tokens * heads * splits * 2, device="cuda")
    kernels.attention_decode(d.q.cuda().view(tokens, -1), heads * dim, out, d.k.cuda(), d.v.cuda(), i32([n - 1 for n in lengths]),
                             i32(range(tokens)), i32(d.table), tokens, heads, kv_heads, dim, 16, None, dim ** -0.5, chunk, splits, *scratch,
                             counters, flag, sinks=torch.tensor(d.sinks, device="cuda") if sinks else None)
    assert int(flag.item()) == 0 and not bool(counters.any())
    d.check(out, sinks)


@pytest.mark.parametrize("sinks", [False, True])
def test_decode_attention_of_scores_that_are_nan_with_a_warp_an_item(sinks):
    """Hundreds of requests of short contexts."""
    from celeg_b200 import kernels
    tokens, heads, kv_heads, dim = 400, 8, 4, 64
    d = Decoded([1 + (7 * r) % 90 for r in range(tokens)], heads, kv_heads, dim, 16, torch.bfloat16, seed=1)
    for r in range(0, tokens, 5):
        d.break_keys(r, 0, min(d.lengths[r], 32))
        d.break_query(r + 1, r % heads)
    out, flag, counters = torch.zeros((tokens, heads * dim), dtype=torch.bfloat16, device="cuda"), i32([0]), i32([0] * tokens * kv_heads)
    scratch = torch.empty(tokens * heads * dim, device="cuda"), torch.empty(tokens * heads * 2, device="cuda")
    kernels.attention_decode(d.q.cuda().view(tokens, -1), heads * dim, out, d.k.cuda(), d.v.cuda(), i32([n - 1 for n in d.lengths]),
                             i32(range(tokens)), i32(d.table), tokens, heads, kv_heads, dim, 16, None, dim ** -0.5, 128, 1, *scratch,
                             counters, flag, sinks=torch.tensor(d.sinks, device="cuda") if sinks else None)
    assert int(flag.item()) == 0
    d.check(out, sinks)
