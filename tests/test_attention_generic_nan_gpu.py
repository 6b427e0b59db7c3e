"""General attention over scores that are NaN: a row that sees one is NaN, and no other row is."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import plain_drafts as plain

pytestmark = pytest.mark.gpu

NAN = float("nan")
I32 = torch.int32


def i32(x):
    return torch.tensor(np.ascontiguousarray(x, dtype=np.int32), device="cuda")


class Decoded:
    """One query for each request, at its last position."""

    def __init__(self, lengths, heads, kv_heads, dim, page, dtype, seed):
        rng = np.random.default_rng(seed)
        self.lengths, self.heads, self.kv_heads, self.dim, self.page, self.dtype = lengths, heads, kv_heads, dim, page, dtype
        self.table, pages = plain.block_tables(lengths, page, rng)
        make = lambda *shape: torch.tensor(rng.normal(size=shape), dtype=torch.float32).to(dtype)      # noqa: E731
        self.k, self.v = make(pages, kv_heads, page, dim), make(pages, kv_heads, page, dim)
        self.q = make(len(lengths), heads, dim)
        self.sinks = rng.normal(size=heads).astype(np.float32)
        self.nan = np.zeros((len(lengths), heads), dtype=bool)

    def break_query(self, request, head):
        self.q[request, head, 1] = NAN
        self.nan[request, head] = True

    def break_keys(self, request, first, behind, kv_head=0):
        for place in range(first, behind):
            self.k[self.table[request, place // self.page], kv_head, place % self.page] = NAN
        group = self.heads // self.kv_heads
        self.nan[request, kv_head * group:(kv_head + 1) * group] = True

    def want(self, sinks):
        out = np.zeros((len(self.lengths), self.heads, self.dim))
        k, v, q = self.k.double().numpy(), self.v.double().numpy(), self.q.double().numpy()
        for r, n in enumerate(self.lengths):
            keys, values = plain.gather(k, self.table[r], n), plain.gather(v, self.table[r], n)
            for h in range(self.heads):
                s = keys[:, h * self.kv_heads // self.heads] @ q[r, h] * self.dim ** -0.5
                w = np.exp(s - s.max())
                out[r, h] = (w @ values[:, h * self.kv_heads // self.heads]) / (w.sum() + (np.exp(self.sinks[h] - s.max()) if sinks else 0.0))
        return out

    def check(self, out, sinks):
        got, want = out.double().cpu().numpy().reshape(self.nan.shape + (self.dim,)), self.want(sinks)
        assert np.isnan(want[self.nan]).all() and np.isfinite(want[~self.nan]).all()
        assert np.isnan(got[self.nan]).all() and np.isfinite(got[~self.nan]).all()
        # bfloat16: weights rounded by 2^-9 of themselves at most, numerator and denominator, and the output; float32: sums of `dim`
        # products under exponentials
        step = 2.0 ** -8 if self.dtype == torch.bfloat16 else self.dim * 2.0 ** -24 + 2.0 ** -20
        most = float(self.v.abs().max())
        assert (np.abs(got - want)[~self.nan] <= step * (np.abs(want)[~self.nan] + most)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (3, 1, 20)])
def test_general_attention_of_scores_that_are_nan(heads, kv_heads, dim, sinks, dtype):
    from celeg_b200 import kernels
    d = Decoded([1, 32, 33, 70, 200, 64], heads, kv_heads, dim, 16, dtype, seed=dim)
    d.break_keys(0, 0, 1)                                      # a token's only key
    d.break_query(1, heads - 1)
    d.break_keys(2, 32, 33)                                    # a block of 32 keys, the second with one
    d.break_keys(3, 0, 32)                                     # ... the first
    d.break_query(4, 0)
    out, flag = torch.zeros((6, heads * dim), dtype=dtype, device="cuda"), i32([0])
    kernels.attention_generic(d.q.cuda().view(6, -1), heads * dim, out, d.k.cuda(), d.v.cuda(), i32([n - 1 for n in d.lengths]), i32(range(6)),
                              i32(d.table), 6, heads, kv_heads, dim, 16, None, dim ** -0.5, flag,
                              sinks=torch.tensor(d.sinks, device="cuda") if sinks else None)
    assert int(flag.item()) == 0
    d.check(out, sinks)
