"""Float64 restatements of the operators behind drafted continuations, and trees, tables and pages for their tests (numpy)."""
from __future__ import annotations

import numpy as np


def random_parents(nodes: int, rng, spread: int = 5) -> np.ndarray:
    """Node 0 is the root, every other node's parent one of the few before it."""
    return np.array([-1] + [int(rng.integers(max(0, i - spread), i)) for i in range(1, nodes)], dtype=np.int32)[:nodes]


def closure(parents: np.ndarray):
    """(seen [nodes, nodes]: itself and its ancestors, depth [nodes])."""
    n = len(parents)
    seen = np.eye(n, dtype=bool)
    depth = np.zeros(n, dtype=np.int32)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] |= seen[p]
            depth[i] = depth[p] + 1
    return seen, depth


def mask_words(seen: np.ndarray, words: int) -> np.ndarray:
    out = np.zeros((seen.shape[0], words), dtype=np.uint32)
    for i, row in enumerate(seen):
        for j in np.nonzero(row)[0]:
            out[i, j // 32] |= np.uint32(1 << (j % 32))
    return out.view(np.int32)


def block_tables(lengths, page_tokens: int, rng, spare: int = 2):
    """(table, pages): random pages for requests of these many positions, -1 behind them."""
    needs = [-(-n // page_tokens) for n in lengths]
    pages = sum(needs) + spare
    order = rng.permutation(pages).tolist()
    table = np.full((len(lengths), max(needs + [1])), -1, dtype=np.int32)
    for r, need in enumerate(needs):
        table[r, :need] = [order.pop() for _ in range(need)]
    return table, pages


def gather(cache: np.ndarray, table_row: np.ndarray, length: int) -> np.ndarray:
    """[length, heads, dim] of a request's positions in [pages, heads, page_tokens, dim]."""
    if length == 0:
        return np.zeros((0, cache.shape[1], cache.shape[3]))
    page_tokens = cache.shape[2]
    held = cache[table_row[:-(-length // page_tokens)]]
    return held.transpose(0, 2, 1, 3).reshape(-1, cache.shape[1], cache.shape[3])[:length]


def attention(q, k, v, seen, positions, context, scale, window=0, sinks=None, softcap=0.0):
    """q [nodes, heads, dim]; k, v [context + nodes, kv_heads, dim]; seen [nodes, nodes]. Float64 [nodes, heads, dim]. A key
    that a row does not see has no part in it, whatever its numbers are."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    at = np.concatenate([np.arange(context), positions])
    out = np.zeros((n, heads, dim))
    for i in range(n):
        visible = np.concatenate([np.ones(context, dtype=bool), seen[i]])
        if window:
            visible &= at > positions[i] - window
        keys = np.nonzero(visible)[0]
        if not len(keys):
            continue
        for h in range(heads):
            s = k[keys, h // group] @ q[i, h] * scale
            if softcap:
                s = softcap * np.tanh(s / softcap)
            top = s.max()
            w = np.exp(s - top)
            total = w.sum() + (np.exp(sinks[h] - top) if sinks is not None else 0.0)
            out[i, h] = (w[:, None] * v[keys, h // group]).sum(0) / total
    return out


def accepted_path(parents, tokens, chosen):
    """(path, token chosen after it)."""
    if len(parents) == 0:
        return [], -1
    path = [0]
    while True:
        node = path[-1]
        after = [c for c in range(node + 1, len(parents)) if parents[c] == node and tokens[c] == chosen[node]]
        if not after:
            return path, int(chosen[node])
        path.append(after[0])


def log_probabilities(x: np.ndarray):
    """(log softmax, entropy) of a row in float64."""
    x = x.astype(np.float64)
    m = x.max()
    e = np.exp(x - m)
    # (the largest's own 1 apart, so that a sum close to 1 keeps its small part)
    rest = e.sum() - 1.0 if (x == m).sum() > 1 else np.delete(e, int(x.argmax())).sum()
    log_p = x - m - np.log1p(rest)
    p = np.exp(log_p)
    return log_p, -(p[p > 0] * log_p[p > 0]).sum()


def best(x: np.ndarray, count: int) -> np.ndarray:
    """Indices of the largest, equal ones by the lower index."""
    return np.lexsort((np.arange(len(x)), -x))[:count]
