"""Forked requests and scored prompts through the engine, and a run of the operators together: trees drafted, attended, scored,
kept and forked, against the same model fed token by token."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

import plain_drafts as plain
import plain_lfm2
import tiny_models

pytestmark = pytest.mark.gpu


def engine_of(tmp_path, name, dtype, **options):
    from celeg_b200 import Engine, EngineOptions
    return Engine(tiny_models.write_tiny(tmp_path, name), dtype=dtype, options=EngineOptions(**options))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
@pytest.mark.parametrize("prompt_tokens", [1, 16, 37])
def test_a_fork_goes_on_as_the_request_itself_would(tmp_path, name, dtype, prompt_tokens):
    engine = engine_of(tmp_path, name, dtype)
    rng = np.random.default_rng(prompt_tokens)
    vocab = engine.loaded.model.vocab_size
    prompt = rng.integers(0, vocab, prompt_tokens).tolist()
    ways = [rng.integers(0, vocab, 20).tolist() for _ in range(3)]
    want = []
    for way in ways:                                            # alone, from the beginning
        rows = [engine.forward([{"id": "alone", "tokens": prompt}])]
        rows = [engine.forward([{"id": "alone", "tokens": [token], "want": [0]}]).clone() for token in way]
        want.append(torch.cat(rows))
        engine.end("alone")
    engine.forward([{"id": 0, "tokens": prompt}])
    engine.fork(0, 1)
    first = engine.forward([{"id": 1, "tokens": ways[1][:1], "want": [0]}]).clone()
    engine.fork(0, 2)                                           # (request 1 has gone on: request 0 has not)
    got = [[], [first], []]
    for step in range(20):
        batch = [(r, ways[r][step]) for r in range(3) if len(got[r]) <= step]
        logits = engine.forward([{"id": r, "tokens": [token], "want": [0]} for r, token in batch])
        for row, (r, _) in enumerate(batch):
            got[r].append(logits[row:row + 1].clone())
        engine.loaded.manager.check_invariants()
        if step == 9:
            engine.fork(2, 3)                                   # a fork of a fork, ended at once
            engine.end(3)
    for r in range(3):
        # (products of 1 and of 3 rows add up in another order)
        bound = 1e-4 if dtype == "float32" else 6e-2
        assert (torch.cat(got[r]) - want[r]).abs().max().item() <= bound * max(1.0, want[r].abs().max().item())
        engine.end(r)
    engine.loaded.step.raise_on_device_error()
    engine.loaded.manager.check_invariants()
    assert all(group.pool.used_pages == 0 for group in engine.loaded.manager.groups)


@pytest.mark.parametrize("design", ["ramosun", "kedesun", "naselorn", "liverax", "kodupel", "fovezen"])
def test_forks_of_every_design_carry_its_caches_and_states(tmp_path, design):
    """Windows whose first pages are gone, values of another size than keys or of none, matrix states, convolutions' tails, layers
    that repeat with caches of their own."""
    from celeg_b200.engine.loading import load_model
    from celeg_b200.engine.step import StepEntry
    module = importlib.import_module(f"{design}_models")
    for name, (raw, seed) in module.CONFIGS.items():
        folder = str(tmp_path / name)
        module.write_model(folder, raw, seed)
        loaded = load_model(folder, dtype="float32", max_requests=4, cache_tokens=1024, max_batched_tokens=512, max_context=512)
        rng = np.random.default_rng(seed)
        vocab = loaded.model.vocab_size
        prompt, ways = rng.integers(0, vocab, 70).tolist(), rng.integers(0, vocab, (2, 9)).tolist()

        def feed(request, tokens):
            logits = loaded.step.run([StepEntry(request, tokens, list(range(len(tokens))))], auto_begin=True).clone()
            loaded.step.raise_on_device_error()
            return logits

        want = []
        for way in ways:
            feed("alone", prompt[:41])
            feed("alone", prompt[41:])
            want.append(torch.cat([feed("alone", way[:3])] + [feed("alone", [token]) for token in way[3:]]))
            loaded.step.end("alone")
        feed("a", prompt[:41])
        feed("a", prompt[41:])
        loaded.step.fork("a", "b")
        got = [[feed("a", ways[0][:3])], [feed("b", ways[1][:3])]]
        for a, b in zip(ways[0][3:], ways[1][3:]):
            got[1].append(feed("b", [b]))
            got[0].append(feed("a", [a]))
        loaded.manager.check_invariants()
        for rows, whole in zip(got, want):
            assert (torch.cat(rows) - whole).abs().max().item() <= 1e-4 * max(1.0, whole.abs().max().item()), name
        loaded.step.end("a")
        loaded.step.end("b")
        assert all(group.pool.used_pages == 0 for group in loaded.manager.groups)


def test_a_fork_refuses_what_it_cannot_hold(tmp_path):
    from celeg_b200.cache import OutOfPages
    engine = engine_of(tmp_path, "A", "float32", max_active_requests=2, logical_kv_pages=4)
    engine.forward([{"id": 0, "tokens": list(range(40))}])
    with pytest.raises(KeyError):
        engine.fork(7, 8)
    with pytest.raises(ValueError):
        engine.fork(0, 0)
    engine.fork(0, 1)
    with pytest.raises(OutOfPages):
        engine.fork(0, 2)
    for r in (0, 1):
        engine.end(r)
    engine.loaded.manager.check_invariants()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "D"])
def test_score(tmp_path, name, dtype):
    engine = engine_of(tmp_path, name, dtype)
    folder = tiny_models.write_tiny(tmp_path, name)
    config, weights = plain_lfm2.load_model_folder(folder)
    rng = np.random.default_rng(5)
    vocab = engine.loaded.model.vocab_size
    prompts = [rng.integers(0, vocab, n).tolist() for n in (1, 2, 33, 100)]
    scores = engine.score(prompts, top=4)
    for prompt, got in zip(prompts, scores):
        assert len(got.logprobs) == len(got.entropy) == len(got.top) == len(prompt) - 1
        if len(prompt) == 1:
            assert got.total == 0.0
            continue
        logits = np.asarray(engine.forward([{"id": "plain", "tokens": prompt, "want": range(len(prompt))}]).double().cpu())
        engine.end("plain")
        for i in range(len(prompt) - 1):
            log_p, entropy = plain.log_probabilities(logits[i])
            # (the logits of a prompt and of a portion without its last token: products of other row counts)
            bound = 1e-3 if dtype == "float32" else 0.1
            assert abs(got.logprobs[i] - log_p[prompt[i + 1]]) <= bound and abs(got.entropy[i] - entropy) <= bound
            if dtype == "float32":
                assert [token for token, _ in got.top[i]] == plain.best(logits[i], 4).tolist()
        assert abs(got.total - sum(got.logprobs)) < 1e-6 * len(prompt)
    one = engine.score(prompts[2])
    assert one.logprobs == scores[2].logprobs and one.top == [[]] * 32
    for bad in ([], [[]], [[1, vocab]]):
        with pytest.raises(ValueError):
            engine.score(bad) if bad else engine.score([[1], []])
    with pytest.raises(ValueError):
        engine.score([1, 2], top=129)
    engine.loaded.manager.check_invariants()
    assert all(group.pool.used_pages == 0 for group in engine.loaded.manager.groups)


def test_score_takes_arrays(tmp_path):
    engine = engine_of(tmp_path, "A", "float32")
    prompt = [3, 1, 4, 1, 5, 9, 2, 6]
    want = engine.score(prompt).logprobs
    for one in (tuple(prompt), np.array(prompt), torch.tensor(prompt), torch.tensor(prompt, device="cuda")):
        assert engine.score(one).logprobs == want
    for several in ([np.array(prompt), torch.tensor(prompt)], np.array([prompt] * 2), torch.tensor([prompt] * 2)):
        assert [scores.logprobs for scores in engine.score(several)] == [want] * 2
    assert engine.score([]) == []


def test_score_in_portions(tmp_path, monkeypatch):
    from celeg_b200.engine import engine as module
    engine = engine_of(tmp_path, "B", "float32")
    prompt = np.random.default_rng(1).integers(0, 1000, 150).tolist()
    whole = engine.score(prompt, top=2)
    monkeypatch.setattr(module, "SCORED_TOKENS", 64)
    parts = engine.score(prompt, top=2)
    assert np.abs(np.array(whole.logprobs) - np.array(parts.logprobs)).max() < 1e-3
    assert [t[0][0] for t in whole.top] == [t[0][0] for t in parts.top]


class Toy:
    """Attention layers alone over a paged cache, in float32 and torch but for the operators under test: enough of a model that a
    token's continuation depends on every token before it."""

    def __init__(self, dtype, dim, layers=2, heads=4, kv_heads=2, vocab=40, page=8, pages=64):
        g = torch.Generator().manual_seed(dim)
        self.heads, self.kv_heads, self.dim, self.page, self.dtype, self.layers = heads, kv_heads, dim, page, dtype, layers
        width = heads * dim
        make = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g) * scale).cuda()      # noqa: E731
        self.embedding, self.places = make(vocab, width), make(600, width, scale=0.5)
        self.qkv = [make(width, (heads + 2 * kv_heads) * dim, scale=width ** -0.5 * 1.5) for _ in range(layers)]
        self.out = [make(width, width, scale=width ** -0.5) for _ in range(layers)]
        self.head = make(width, vocab, scale=width ** -0.5 * 3.0)
        self.k, self.v = (torch.zeros(layers, pages, kv_heads, page, dim, dtype=dtype, device="cuda") for _ in range(2))
        self.flag = torch.zeros(1, dtype=torch.int32, device="cuda")

    def step(self, tokens, positions, places, table, attend):
        """Logits [tokens, vocab]; keys and values go to ``places`` of ``table`` [rows of places]; ``attend(q, layer)`` reads them."""
        x = self.embedding[tokens] + self.places[positions]
        kv_width = self.kv_heads * self.dim
        for layer in range(self.layers):
            qkv = (x / x.square().mean(1, keepdim=True).sqrt()) @ self.qkv[layer]
            q, k, v = qkv.split([self.heads * self.dim, kv_width, kv_width], 1)
            pages, rows = table[places // self.page], places % self.page
            self.k[layer][pages, :, rows] = k.reshape(-1, self.kv_heads, self.dim).to(self.dtype)
            self.v[layer][pages, :, rows] = v.reshape(-1, self.kv_heads, self.dim).to(self.dtype)
            x = x + attend(q.to(self.dtype).contiguous(), layer).float() @ self.out[layer]
        return (x @ self.head).contiguous()


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 24), (torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_drafted_trees_give_the_tokens_that_one_at_a_time_gives(dtype, dim):
    """Trees whose branches hold the right tokens, wrong ones and both; the accepted tokens are those of greedy decoding, and the
    scores those of the step that decodes them. In the middle the request is forked and both go on."""
    from celeg_b200 import kernels
    from celeg_b200.cache import CacheManager, PagedNeed, StateLayout
    toy = Toy(dtype, dim)
    i32 = lambda a: torch.tensor(np.ascontiguousarray(a, dtype=np.int32), device="cuda")      # noqa: E731
    prompt = [3, 17, 8, 25, 25, 1, 39, 12, 30, 2, 5]
    need = PagedNeed(2, dim)
    manager = CacheManager(8, [64], [(need.group_key(), need)], StateLayout(), 4)
    scratch = kernels.attention_tree_scratch("cuda")

    def tree_step(cache, parents, tokens):
        n, context = len(parents), cache.tokens
        seen, depth = plain.closure(np.array(parents))
        manager.reserve(cache, context + n)
        table = i32(cache.table_array(0))
        positions = context + depth
        fixed = [i32(positions), i32([0, n]), i32([context]), i32(plain.mask_words(seen, 2)), table[None]]

        def attend(q, layer):
            out = torch.empty_like(q)
            kernels.attention_tree(q, q.stride(0), out, toy.k[layer], toy.v[layer], *fixed, n, 1, 64, 300, 4, 2, dim, 8, None, dim ** -0.5,
                                   scratch, toy.flag)
            return out
        logits = toy.step(i32(tokens).long(), i32(positions).long(), i32(context + np.arange(n)).long(), table.long(), attend)
        top, log_p = torch.empty(n, 1, dtype=torch.int32, device="cuda"), torch.empty(n, 1, device="cuda")
        kernels.token_logprobs(logits, n, None, None, None, log_p, top)
        path, accepted, following = (torch.empty(shape, dtype=torch.int32, device="cuda") for shape in ((1, 64), (1,), (1,)))
        kernels.keep_drafts(toy.k, toy.v, i32(parents), i32(tokens), top.view(-1), fixed[1], fixed[2], fixed[4], 1, 64, path, accepted,
                            following, toy.flag)
        count = int(accepted.item())
        manager.advance(cache, context + count)
        manager.check_invariants()
        nodes = path[0, :count].tolist()
        return [tokens[node] for node in nodes[1:]] + [int(following.item())], [log_p[node, 0].item() for node in nodes]

    def chain(cache, tokens):                                     # a prompt: a tree that is one branch
        return tree_step(cache, list(range(-1, len(tokens) - 1)), tokens)

    # one token at a time
    cache = manager.open("plain")
    tokens, scores = chain(cache, prompt)
    decoded, log_ps = tokens[-1:], scores[-1:]
    for _ in range(40):
        tokens, scores = tree_step(cache, [-1], decoded[-1:])
        decoded += tokens
        log_ps += scores
    manager.close("plain")

    rng = np.random.default_rng(1)

    def speculate(cache, got, got_p, until):
        while len(got) < until:
            # the root, three branches of which one may be right for some tokens, and wrong leaves everywhere
            parents, tokens = [-1], got[-1:]
            for branch in range(3):
                at, good = 0, rng.integers(0, 5)
                for depth in range(4):
                    right = decoded[len(got) + depth] if len(got) + depth < len(decoded) else 0
                    parents.append(at)
                    tokens.append(int(right) if depth < good else int(rng.integers(0, 40)))
                    at = len(tokens) - 1
                    if rng.random() < 0.4:
                        parents.append(at)
                        tokens.append(int(rng.integers(0, 40)))
            new, new_p = tree_step(cache, parents, tokens)
            got += new
            got_p += new_p
        return got, got_p

    cache = manager.open("a")
    tokens, scores = chain(cache, prompt)
    got, got_p = speculate(cache, tokens[-1:], scores[-1:], 15)
    other, copies = manager.fork("a", "b")
    if copies[0]:
        kernels.copy_pages(toy.k, toy.v, copies[0])
    second = (list(got), list(got_p))
    got, got_p = speculate(cache, got, got_p, 35)
    second = speculate(other, *second, 35)
    assert int(toy.flag.item()) == 0
    for tokens, scores in ((got, got_p), second):
        same = min(len(tokens), len(decoded))
        if dtype == torch.float32:
            assert tokens[:same] == decoded[:same]
            assert np.abs(np.array(scores[:same]) - np.array(log_ps[:same])).max() < 1e-3
        else:
            # (rounded attention of another split: a nearly tied arg-max may go the other way, and all behind it)
            equal = next((i for i, (x, y) in enumerate(zip(tokens, decoded)) if x != y), same)
            assert equal >= 10 and np.abs(np.array(scores[:equal]) - np.array(log_ps[:equal])).max() < 0.2
    manager.close("a")
    manager.close("b")
    manager.check_invariants()
