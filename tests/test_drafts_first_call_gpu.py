"""Calls of drafted continuations that a process makes for the first time inside a capture, and on two streams at once: nothing that they
set up once may need an ordinary call before."""
from __future__ import annotations

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from test_drafts_gpu import Trees, caches, i32

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
# (heads, kv heads, head size, spans, element type): every form of the kernels, pieces in clusters and in scratch
FORMS = [(4, 1, 64, [(9, 2000), (3, 70)], "bfloat16"), (32, 2, 64, [(40, 600)], "bfloat16"), (4, 2, 128, [(9, 700)], "bfloat16"),
         (32, 2, 128, [(40, 600)], "bfloat16"), (4, 2, 256, [(9, 700)], "bfloat16"), (4, 1, 64, [(3, 20011)], "bfloat16"),
         (4, 2, 20, [(9, 300)], "bfloat16"), (4, 2, 64, [(9, 900)], "float32"), (4, 2, 128, [(9, 900)], "float32"), (2, 2, 200, [(9, 300)], "float32")]

SCRIPT = """
import sys
sys.path[:0] = [{here!r}, {root!r}]
import torch
from test_drafts_first_call_gpu import captured_first
captured_first()
print("captured")
"""


def captured_first():
    from celeg_b200 import kernels
    scratch = kernels.attention_tree_scratch("cuda")
    for heads, kv_heads, dim, spans, dtype in FORMS:
        t = Trees(spans, heads, kv_heads, dim, 16, getattr(torch, dtype), seed=dim)
        q, k, v = t.q.cuda(), t.k.cuda(), t.v.cuda()
        fixed = [i32(np.concatenate(t.positions)), i32(t.begin), i32(t.context), i32(t.masks), i32(t.table)]
        out, flag = torch.zeros((t.total, heads * dim), dtype=t.dtype, device="cuda"), i32([0])

        def call():
            kernels.attention_tree(q, q.stride(0), out, k, v, *fixed, t.total, len(spans), t.max_nodes, max(n + c for n, c in spans), heads, kv_heads,
                                   dim, 16, None, dim ** -0.5, scratch, flag)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        call()
        assert int(flag.item()) == 0 and torch.equal(got, out) and bool(out.any()), (heads, dim, dtype)
    k, v = caches(2, 12, 2, 16, 64, 64, torch.bfloat16, np.random.default_rng(0))
    logits, tokens = torch.randn((3, 70000), device="cuda"), i32([5, 6, 7])
    logprobs, entropy, top, best = (torch.zeros(shape, device="cuda") for shape in ((3,), (3,), (3, 5), (3, 5)))
    best = best.int()
    want = k.clone()
    want[:, 5] = k[:, 3]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.token_logprobs(logits, 3, tokens, logprobs, entropy, top, best)
        kernels.copy_pages(k, v, [(3, 5, 16)])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(k, want)
    log_p = logits.double().log_softmax(1)
    assert (logprobs - log_p.gather(1, tokens.long()[:, None])[:, 0]).abs().max() < 1e-4 and torch.equal(best.long(), log_p.topk(5).indices)


def test_first_calls_inside_a_capture():
    script = SCRIPT.format(here=HERE, root=os.path.dirname(HERE))
    done = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stdout + done.stderr


def test_scores_and_kept_drafts_on_two_streams_at_once():
    from celeg_b200 import kernels
    logits = torch.randn((64, 50257), device="cuda")
    tokens = torch.arange(64, device="cuda", dtype=torch.int32)
    parents, chosen = i32([-1, 0, 0, 2, 3, 3]), i32([2, 0, 3, 5, 0, 7])
    sides = []
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        k, v = caches(2, 40, 2, 16, 64, 64, torch.bfloat16, np.random.default_rng(3))
        outs = [torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda"), torch.zeros((64, 5), device="cuda"), i32(np.zeros((64, 5)))]
        kept = [i32(np.zeros((1, 6))), i32([0]), i32([0]), i32([0])]
        sides.append((stream, k, v, outs, kept))
    begin, context, table, drafts = i32([0, 6]), i32([30]), i32([[4, 9, 2]]), i32([9, 1, 2, 3, 4, 5])
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, k, v, outs, kept in sides:
            with torch.cuda.stream(stream):
                kernels.token_logprobs(logits, 64, tokens, *outs)
                kernels.keep_drafts(k, v, parents, drafts, chosen, begin, context, table, 1, 6, *kept)
                kernels.copy_pages(k, v, [(4, 20, 16), (9, 21, 3)])
    torch.cuda.synchronize()
    log_p = logits.double().log_softmax(1)
    for one, other in zip(sides[0][3] + sides[0][4] + list(sides[0][1:3]), sides[1][3] + sides[1][4] + list(sides[1][1:3])):
        assert torch.equal(one, other)
    assert sides[0][4][0].tolist() == [[0, 2, 3, 5, -1, -1]] and torch.equal(sides[0][3][3].long(), log_p.topk(5).indices)
