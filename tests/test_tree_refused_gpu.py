"""Spans that attention of drafted trees refuses, with keys cut into pieces that meet in scratch: their rows stay as they were."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_drafts_gpu import Trees

pytestmark = pytest.mark.gpu


# (nodes of both spans, cached positions, query heads, head size): cut into pieces of a join in float32, and in bfloat16 into
# more than a cluster holds
@pytest.mark.parametrize("dtype,context", [(torch.float32, 1500), (torch.bfloat16, 20011)])
@pytest.mark.parametrize("dim", [64, 40])
def test_rows_of_refused_spans_are_left_alone_by_the_join(dim, dtype, context):
    def trees():
        return Trees([(6, context), (4, context - 77)], 4, 1, dim, 16, dtype, seed=dim)

    t = trees()
    want = t.want(0.2)
    places = t.table.shape[1] * 16
    cases = [(2, dict(context=[places, context - 77]), (0, 6)), (2, dict(context=[context, 2 ** 31 - 2]), (6, 10)),
             (4, dict(context=[-1, context - 77]), (0, 6)), (4, dict(max_nodes=5), (0, 6)),
             (4, dict(begin=np.array([0, 6, 11], dtype=np.int32)), (6, 10)), (4, dict(begin=np.array([0, -1, 10], dtype=np.int32)), (0, 10))]
    for error, changes, (first, behind) in cases:
        t = trees()
        for name, value in changes.items():
            setattr(t, name, value)
        # (numbers of an earlier call, which a join would make a plausible row of)
        scratch = torch.full((1 << 23,), 3.0, device="cuda")
        out, flag = t.run(0.2, scratch=scratch, max_keys=context + 6)
        if behind - first < t.total:                     # (a refused span leaves nothing in scratch)
            assert not bool((scratch == 3.0).all()), "the keys were not cut into pieces"
        assert flag == error, changes
        assert bool((out[first:behind] == 7.0).all()), changes
        whole = want.copy()
        whole[first:behind] = 7.0
        t.check(out, whole)
