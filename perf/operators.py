"""The operators behind drafted continuations of a request, measured: attention of a tree of drafted tokens over the paged
cache, keeping the accepted path of such a tree, copies of cache pages (a request forked into several), and log probabilities
of given tokens with entropy and top alternatives.

Sizes are those of this package's own models: 32 query heads on 8 kv heads of 64 (LFM2-1.2B), 16 on 4 of 128, pages of 16
positions, a vocabulary of 65,536."""
import math

import numpy as np
import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _tree(name, requests, nodes, context, heads=32, kv_heads=8, dim=64, dtype="bf16", ragged=False, window=0, sinks=False, cap=0.0):
    return {"name": name, "kind": "tree", "requests": requests, "nodes": nodes, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "ragged": ragged, "window": window, "sinks": sinks, "cap": cap}


def _keep(name, requests, nodes, context, layers, kv_heads=8, dim=64, dtype="bf16"):
    return {"name": name, "kind": "keep", "requests": requests, "nodes": nodes, "context": context, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def _copy(name, pairs, layers, partial, kv_heads=8, dim=64, dtype="bf16"):
    return {"name": name, "kind": "copy", "pairs": pairs, "layers": layers, "partial": partial, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype}


def _score(name, rows, vocab, top, dtype="f32"):
    return {"name": name, "kind": "score", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype}


def listed():
    return [
        # one user, a small tree behind a short conversation: latency
        _tree("tree_one_user", 1, 13, 601),
        # a server's ordinary step: eight users of unequal lengths, 32 drafts each
        _tree("tree_batch8", 8, 32, 4096, ragged=True),
        # heads of 128 under a window with a sink per head, odd sizes
        _tree("tree_window_128", 12, 21, 5003, heads=16, kv_heads=4, dim=128, ragged=True, window=1024, sinks=True),
        # wide trees over long contexts: the largest
        _tree("tree_long", 4, 64, 65536),
        # the float32 path of the same model
        _tree("tree_float32", 2, 24, 1500, dtype="f32", ragged=True),
        # one user's accepted path, six attention layers: latency
        _keep("keep_one_user", 1, 13, 601, 6),
        # a full server's step: 64 users, 32 drafts each, sixteen layers
        _keep("keep_batch64", 64, 32, 200, 16),
        # a request forked once: its last page, partly filled
        _copy("fork_one", 1, 6, True),
        # beams reordered, many requests forked: whole pages over sixteen layers
        _copy("copy_pages_768", 768, 16, False),
        # a decoded token with its twenty best alternatives
        _score("logprobs_one_row", 1, 65536, 20),
        # a batch of users asking for five alternatives, an odd vocabulary
        _score("logprobs_batch64", 64, 50257, 5),
        # a document scored: every token's log probability and the model's own choice
        _score("logprobs_document", 4095, 65536, 1),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "keep", "copy", "score", "score"])
    if kind == "tree":
        heads, kv_heads, dim = rng.choice([(32, 8, 64), (16, 4, 128), (24, 8, 64), (16, 2, 64), (8, 8, 128), (32, 4, 64), (12, 4, 80), (8, 2, 256)])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        requests, nodes = _log_int(rng, 1, 32), _log_int(rng, 1, 150)
        most = min(65536.0, 1.6e7 / (requests * nodes), 2.6e5 / requests * min(1.0, 512 / (kv_heads * dim)))
        if dtype == "f32":
            most = min(most, 3e5 / (requests * nodes))
        context = _log_int(rng, 1, max(2.0, most))
        return dict(_tree("", requests, nodes, context, heads, kv_heads, dim, dtype, rng.random() < 0.6,
                          rng.choice([0, 0, _log_int(rng, 4, 2000)]), rng.random() < 0.3, rng.choice([0.0, 0.0, 30.0])))
    if kind == "keep":
        return dict(_keep("", _log_int(rng, 1, 64), _log_int(rng, 1, 64), _log_int(rng, 1, 200), _log_int(rng, 1, 16),
                          rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 80, 20]), rng.choice(["bf16", "f32"])))
    if kind == "copy":
        layers, kv_heads, dim, dtype = _log_int(rng, 1, 16), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 80, 20]), rng.choice(["bf16", "f32"])
        most = 768 * 16 * 8 * 64 * 2 // (layers * kv_heads * dim * (4 if dtype == "f32" else 2))
        return dict(_copy("", _log_int(rng, 1, min(768, most)), layers, rng.random() < 0.5, kv_heads, dim, dtype))
    vocab = _log_int(rng, 300, 150000)
    rows = min(_log_int(rng, 1, 4095), int(2.6e8 / vocab))
    return dict(_score("", rows, vocab, rng.choice([0, 1, 5, 20, 64]), rng.choice(["f32", "f32", "bf16"])))


# ------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Nodes and cached positions of every request. They follow from the case alone: inputs of another seed have the same sizes."""
    n = case["requests"]
    if not case.get("ragged"):
        return [case["nodes"]] * n, [case["context"]] * n
    rng = np.random.default_rng([n, case["nodes"], case["context"]])
    nodes = [case["nodes"]] + [int(rng.integers(max(1, case["nodes"] // 2), case["nodes"] + 1)) for _ in range(n - 1)]
    context = [case["context"]] + [int(rng.integers(case["context"] // 4, case["context"] + 1)) for _ in range(n - 1)]
    return nodes, context


def _parents(nodes, rng):
    """A tree as drafters make them: every node hangs on one of the few before it, node 0 is the root."""
    return np.array([-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, nodes)], dtype=np.int32)


def _closure(parents, words):
    """Per node the bits of itself and its ancestors, and its depth."""
    bits = np.zeros((len(parents), words), dtype=np.uint32)
    depth = np.zeros(len(parents), dtype=np.int32)
    for i, p in enumerate(parents):
        if p >= 0:
            bits[i] = bits[p]
            depth[i] = depth[p] + 1
        bits[i, i // 32] |= np.uint32(1 << (i % 32))
    return bits.view(np.int32), depth


def _prefix(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _drafts(case, rng, device):
    """Trees, tables and positions of a step: what a server holds on the host and sends along."""
    nodes, context = _lengths(case)
    words = (max(nodes) + 31) // 32
    parents, masks, positions = [], [], []
    for n, c in zip(nodes, context):
        up = _parents(n, rng)
        bits, depth = _closure(up, words)
        parents.append(up)
        masks.append(bits)
        positions.append(c + depth)
    per = [(n + c + PAGE - 1) // PAGE for n, c in zip(nodes, context)]
    pages = sum(per) + 3
    order = rng.permutation(pages)
    table = np.full((len(nodes), max(per)), -1, dtype=np.int32)
    at = 0
    for r, count in enumerate(per):
        table[r, :count] = order[at:at + count]
        at += count
    send = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(device)  # noqa: E731
    return {"nodes": nodes, "context": context, "words": words, "pages": pages, "table": send(table),
            "span_begin": send(_prefix(nodes)), "span_context": send(context), "parents": send(np.concatenate(parents)),
            "ancestors": send(np.concatenate(masks)), "positions": send(np.concatenate(positions)),
            "total": int(sum(nodes)), "max_nodes": max(nodes), "max_keys": max(n + c for n, c in zip(nodes, context))}


def _normal(shape, generator, dtype, scale=1.0):
    """Normal numbers in `dtype`, made a slice at a time (a large cache need not exist in float32 too)."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 26
    for at in range(0, flat.numel(), step):
        part = flat[at:at + step]
        part.copy_(torch.randn(part.numel(), generator=generator, device="cuda").mul_(scale))
    return out


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "tree":
        s.update(_drafts(case, rng, "cuda"))
        shape = (s["pages"], case["kv_heads"], PAGE, case["dim"])
        s["k"], s["v"] = _normal(shape, generator, dtype), _normal(shape, generator, dtype)
        # rows as the projection leaves them: queries, then the step's own keys and values
        width = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        s["qkv"] = _normal((s["total"], width), generator, dtype)
        s["sinks"] = torch.randn(case["heads"], generator=generator, device="cuda") if case["sinks"] else None
        s["out"] = torch.empty((s["total"], case["heads"] * case["dim"]), dtype=dtype, device="cuda")
        s["error"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["scale"] = case["dim"] ** -0.5
        s["scratch"] = torch.empty(1 << 24, device="cuda")       # a workspace that all layers of a model share
    elif case["kind"] == "keep":
        s.update(_drafts(case, rng, "cuda"))
        shape = (case["layers"], s["pages"], case["kv_heads"], PAGE, case["dim"])
        s["k"], s["v"] = _normal(shape, generator, dtype), _normal(shape, generator, dtype)
        # a drafter is often right: with tokens of two values a path of some three nodes is accepted
        s["tokens"] = torch.from_numpy(rng.integers(0, 2, s["total"]).astype(np.int32)).cuda()
        s["chosen"] = torch.from_numpy(rng.integers(0, 2, s["total"]).astype(np.int32)).cuda()
        n = case["requests"]
        s["path"] = torch.empty((n, s["max_nodes"]), dtype=torch.int32, device="cuda")
        s["accepted"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["next"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["error"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    elif case["kind"] == "copy":
        pages = 2 * case["pairs"] + 1
        shape = (case["layers"], pages, case["kv_heads"], PAGE, case["dim"])
        s["k"], s["v"] = _normal(shape, generator, dtype), _normal(shape, generator, dtype)
        order = rng.permutation(pages)
        count = case["pairs"]
        rows = rng.integers(1, PAGE + 1, count) if case["partial"] else np.full(count, PAGE)
        s["copies"] = np.stack([order[:count], order[count:2 * count], rows], axis=1).astype(np.int32)
        s["copies_device"] = torch.from_numpy(s["copies"].astype(np.int64)).cuda()
    else:
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        # logits of a language model: a normal bulk and a few tokens far above it
        logits = torch.randn((rows, vocab), generator=generator, device="cuda").mul_(2.5)
        high = torch.randint(0, vocab, (rows, 8), generator=generator, device="cuda")
        logits.scatter_add_(1, high, torch.rand((rows, 8), generator=generator, device="cuda").mul_(14.0))
        s["logits"] = logits.to(dtype)
        s["tokens"] = torch.where(torch.rand(rows, generator=generator, device="cuda") < 0.7, high[:, 0],
                                  torch.randint(0, vocab, (rows,), generator=generator, device="cuda")).to(torch.int32)
        s["logprobs"] = torch.empty(rows, device="cuda")
        s["entropy"] = torch.empty(rows, device="cuda")
        s["top_logprobs"] = torch.empty((rows, top), device="cuda")
        s["top_tokens"] = torch.empty((rows, top), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------------------------- a pass
def run(s):
    return {"tree": _run_tree, "keep": _run_keep, "copy": _run_copy, "score": _run_score}[s["case"]["kind"]](s)


def _run_tree(s):
    c = s["case"]
    if own:
        from celeg_b200 import kernels
        kernels.attention_tree(s["qkv"], s["qkv"].stride(0), s["out"], s["k"], s["v"], s["positions"], s["span_begin"],
                               s["span_context"], s["ancestors"], s["table"], s["total"], c["requests"], s["max_nodes"],
                               s["max_keys"], c["heads"], c["kv_heads"], c["dim"], PAGE, c["window"] or None, s["scale"],
                               s["scratch"], s["error"], sinks=s["sinks"], softcap=c["cap"] or None)
        return s["out"]
    r, n, keys, group, dim = c["requests"], s["max_nodes"], s["table"].shape[1] * PAGE, c["heads"] // c["kv_heads"], c["dim"]
    begin, context = s["span_begin"].long(), s["span_context"].long()
    device = begin.device
    table = s["table"].long().clamp(min=0)
    k = s["k"][table].transpose(1, 2).reshape(r, c["kv_heads"], keys, dim).float()
    v = s["v"][table].transpose(1, 2).reshape(r, c["kv_heads"], keys, dim).float()
    # nodes of all requests side by side, short trees filled up with their first node
    local = torch.arange(n, device=device)
    count = begin[1:] - begin[:-1]
    real = local < count[:, None]
    token = torch.where(real, begin[:-1, None] + local, begin[:-1, None])
    q = s["qkv"][:, :c["heads"] * dim][token].float().view(r, n, c["kv_heads"], group, dim).permute(0, 2, 3, 1, 4)
    place = torch.arange(keys, device=device)
    cached = place < context[:, None]                                                       # [r, keys]
    draft = place - context[:, None]
    drafted = (draft >= 0) & (draft < count[:, None])
    bit = draft.clamp(0, n - 1)
    position = s["positions"].long()
    key_position = torch.where(drafted, position[(begin[:-1, None] + bit).clamp(max=s["total"] - 1)], place)
    words = s["ancestors"].long()[token]                                                    # [r, n, words]
    is_ancestor = (torch.gather(words, 2, (bit // 32)[:, None].expand(r, n, keys)) >> (bit % 32)[:, None]) & 1
    seen = cached[:, None] | (drafted[:, None] & (is_ancestor == 1))
    if c["window"]:
        seen &= key_position[:, None] > position[token][:, :, None] - c["window"]
    score = torch.matmul(q.reshape(r, c["kv_heads"], group * n, dim), k.transpose(2, 3)) * s["scale"]
    score = score.view(r, c["kv_heads"], group, n, keys)
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, c["kv_heads"], group, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    out = torch.matmul(weight.view(r, c["kv_heads"], group * n, keys), v).view(r, c["kv_heads"], group, n, dim)
    out = out / torch.where(total > 0, total, 1.0)
    return out.permute(0, 3, 1, 2, 4).reshape(r, n, c["heads"] * dim)[real].to(s["qkv"].dtype)


def _run_keep(s):
    c = s["case"]
    if own:
        from celeg_b200 import kernels
        kernels.keep_drafts(s["k"], s["v"], s["parents"], s["tokens"], s["chosen"], s["span_begin"], s["span_context"],
                            s["table"], c["requests"], s["max_nodes"], s["path"], s["accepted"], s["next"], s["error"])
        return {"k": s["k"], "v": s["v"], "path": s["path"], "accepted": s["accepted"], "next": s["next"]}
    r, n = c["requests"], s["max_nodes"]
    begin, context = s["span_begin"].long(), s["span_context"].long()
    device = begin.device
    local = torch.arange(n, device=device)
    count = begin[1:] - begin[:-1]
    real = local < count[:, None]
    at = torch.where(real, begin[:-1, None] + local, begin[:-1, None])
    parent, token, chosen = (s[name].long()[at] for name in ("parents", "tokens", "chosen"))
    follows = (token == torch.gather(chosen, 1, parent.clamp(min=0))) | (local == 0)
    # of children of one node with the same token the first counts
    same = (parent[:, :, None] == parent[:, None, :]) & (token[:, :, None] == token[:, None, :])
    first = ~(same & (local[None, None, :] < local[None, :, None])).any(-1)
    taken = follows & first & real
    bit = ((s["ancestors"].long()[at][:, :, local // 32] >> (local % 32)) & 1) == 1           # [r, node, ancestor]
    taken = (taken[:, None, :] | ~bit).all(-1) & real
    accepted = taken.sum(1)
    path = torch.where(taken, local, n).sort(1).values
    path = torch.where(path < n, path, -1)
    last = torch.gather(path, 1, (accepted - 1)[:, None])
    following = torch.gather(chosen, 1, last)[:, 0]
    request, step = torch.nonzero(path >= 0, as_tuple=True)
    table = s["table"].long()
    source, target = context[request] + path[request, step], context[request] + step
    from_page, to_page = table[request, source // PAGE], table[request, target // PAGE]
    for cache in (s["k"], s["v"]):
        cache[:, to_page, :, target % PAGE] = cache[:, from_page, :, source % PAGE]
    return {"k": s["k"], "v": s["v"], "path": path.int(), "accepted": accepted.int(), "next": following.int()}


def _run_copy(s):
    c = s["case"]
    if own:
        from celeg_b200 import kernels
        kernels.copy_pages(s["k"], s["v"], s["copies"])
        return {"k": s["k"], "v": s["v"]}
    source, target, rows = s["copies_device"].unbind(1)
    fresh = (torch.arange(PAGE, device=rows.device) < rows[:, None])[None, :, None, :, None]
    for cache in (s["k"], s["v"]):
        moved = cache[:, source]
        cache[:, target] = torch.where(fresh, moved, cache[:, target]) if c["partial"] else moved
    return {"k": s["k"], "v": s["v"]}


def _run_score(s):
    c = s["case"]
    if own:
        from celeg_b200 import kernels
        kernels.token_logprobs(s["logits"], c["rows"], s["tokens"], s["logprobs"], s["entropy"], s["top_logprobs"], s["top_tokens"])
        return {"logprobs": s["logprobs"], "entropy": s["entropy"], "top_logprobs": s["top_logprobs"], "top_tokens": s["top_tokens"]}
    x = s["logits"].float()
    above = x - x.amax(1, keepdim=True)
    weight = above.exp()
    total = weight.sum(1, keepdim=True)
    log_total = total.log()
    entropy = log_total[:, 0] - (weight * above).sum(1) / total[:, 0]
    given = torch.gather(above, 1, s["tokens"].long()[:, None])[:, 0] - log_total[:, 0]
    if c["top"] == 0:
        tokens = torch.empty((c["rows"], 0), dtype=torch.int64, device=x.device)
    elif c["top"] == 1:
        tokens = x.argmax(1, keepdim=True)
    else:
        tokens = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
    return {"logprobs": given, "entropy": entropy, "top_logprobs": torch.gather(above, 1, tokens) - log_total, "top_tokens": tokens.int()}


# ------------------------------------------------------------------------------------- 64 bits, apart
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tree":
        return _exact_tree(case, s)
    if case["kind"] == "score":
        x = s["logits"].double()
        log_p = torch.log_softmax(x, dim=1)
        p = log_p.exp()
        entropy = -(p * log_p).sum(1)
        del p, x
        rows = torch.arange(case["rows"], device="cuda")
        return {"logprobs": log_p[rows, s["tokens"].long()], "entropy": entropy,
                "top_logprobs": torch.topk(log_p, case["top"], dim=1).values, "top_tokens": None}
    # copies: the same numbers at other places, walked on the host
    k, v = s["k"].double(), s["v"].double()
    if case["kind"] == "copy":
        for source, target, rows in s["copies"].tolist():
            for cache in (k, v):
                cache[:, target, :, :rows] = cache[:, source, :, :rows]
        return {"k": k, "v": v}
    table = s["table"].cpu().numpy()
    parents, tokens, chosen = (s[name].cpu().numpy() for name in ("parents", "tokens", "chosen"))
    begin, moves = 0, []
    for request, (n, c) in enumerate(zip(s["nodes"], s["context"])):
        node, path = 0, [0]
        while node is not None:
            after = [i for i in range(node + 1, n) if parents[begin + i] == node and tokens[begin + i] == chosen[begin + node]]
            node = after[0] if after else None
            path += after[:1]
        for step, node in enumerate(path):
            moves.append((table[request, (c + node) // PAGE], (c + node) % PAGE, table[request, (c + step) // PAGE], (c + step) % PAGE))
        begin += n
    from_page, from_row, to_page, to_row = (torch.tensor(part, device="cuda") for part in zip(*moves))
    for cache in (k, v):
        cache[:, to_page, :, to_row] = cache[:, from_page, :, from_row].clone()
    return {"k": k, "v": v, "path": None, "accepted": None, "next": None}


def _exact_tree(case, s):
    group, dim, heads = case["heads"] // case["kv_heads"], case["dim"], case["heads"]
    out = torch.zeros((s["total"], heads, dim), dtype=torch.float64, device="cuda")
    masks = s["ancestors"].cpu().numpy().view(np.uint32)
    positions = s["positions"].cpu().numpy().astype(np.int64)
    begin = 0
    for request, (n, c) in enumerate(zip(s["nodes"], s["context"])):
        held = s["table"][request, :(n + c + PAGE - 1) // PAGE].long()
        k = s["k"][held].double().permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, dim)[:, :n + c]
        v = s["v"][held].double().permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, dim)[:, :n + c]
        at = np.concatenate([np.arange(c), positions[begin:begin + n]])
        seen = np.ones((n, n + c), dtype=bool)
        for i in range(n):
            seen[i, c:] = [(int(masks[begin + i, j // 32]) >> (j % 32)) & 1 for j in range(n)]
            if case["window"]:
                seen[i] &= at > positions[begin + i] - case["window"]
        seen = torch.from_numpy(seen).cuda()
        for head in range(heads):
            q = s["qkv"][begin:begin + n, head * dim:(head + 1) * dim].double()
            score = q @ k[head // group].T * s["scale"]
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            score = score.masked_fill(~seen, -math.inf)
            if s["sinks"] is not None:
                score = torch.cat([score, s["sinks"][head].double().expand(n, 1)], dim=1)
            weight = torch.softmax(score, dim=1)[:, :n + c]
            out[begin:begin + n, head] = weight @ v[head // group]
        begin += n
    return out.view(s["total"], heads * dim)


# ---------------------------------------------------------------------------------- what it has to move
def work(case):
    size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    if case["kind"] == "tree":
        nodes, context = _lengths(case)
        reach = [min(c, case["window"] - 1) if case["window"] else c for c in context]
        # (every draft sees itself and some six ancestors beside what is cached)
        pairs = sum(n * (c + min(7, n)) for n, c in zip(nodes, reach))
        return {"bytes": 2 * (sum(nodes) + sum(reach)) * case["kv_heads"] * case["dim"] * size
                + 2 * sum(nodes) * case["heads"] * case["dim"] * size, "flops": 4.0 * pairs * case["heads"] * case["dim"]}
    if case["kind"] == "keep":
        # (about one node in two moves on: a path of some three nodes, of which two move)
        row = case["layers"] * 2 * case["kv_heads"] * case["dim"] * size
        return {"bytes": 2 * 2 * case["requests"] * row + 5 * 4 * case["requests"] * case["nodes"], "flops": 1}
    if case["kind"] == "copy":
        rows = (PAGE + 1) / 2 if case["partial"] else PAGE
        return {"bytes": 2 * case["pairs"] * rows * case["layers"] * 2 * case["kv_heads"] * case["dim"] * size, "flops": 1}
    return {"bytes": case["rows"] * case["vocab"] * size + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * case["rows"] * case["vocab"]}
