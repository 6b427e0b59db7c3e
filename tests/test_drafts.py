"""What the operators behind drafted continuations refuse, without a GPU."""
import numpy as np
import pytest
import torch

from celeg_b200 import kernels
from celeg_b200.kernels import KernelLibraryError

I32 = torch.int32


def tree_arguments(**changes):
    tokens, spans, heads, kv_heads, dim, page = 5, 2, 4, 2, 64, 16
    a = dict(q=torch.zeros(tokens, heads * dim), q_row_stride=heads * dim, out=torch.zeros(tokens, heads * dim),
             k_cache=torch.zeros(4, kv_heads, page, dim), v_cache=torch.zeros(4, kv_heads, page, dim),
             positions=torch.zeros(tokens, dtype=I32), span_begin=torch.tensor([0, 3, 5], dtype=I32),
             span_context=torch.zeros(spans, dtype=I32), ancestors=torch.zeros(tokens, 1, dtype=I32),
             block_table=torch.zeros(spans, 2, dtype=I32), tokens=tokens, spans=spans, max_nodes=3, max_keys=8, q_heads=heads,
             kv_heads=kv_heads, head_dim=dim, page_tokens=page, window=None, scale=0.1, scratch=None,
             error_flag=torch.zeros(1, dtype=I32))
    a.update(changes)
    return a


@pytest.mark.parametrize("changes", [
    dict(q=torch.zeros(5, 256, dtype=torch.float16)), dict(q=torch.zeros(5, 256, dtype=torch.bfloat16)), dict(out=torch.zeros(4, 256)),
    dict(q=torch.zeros(4, 256)), dict(q=torch.zeros(5, 255)), dict(q=torch.zeros(256, 5).t()), dict(q_row_stride=300),
    dict(k_cache=torch.zeros(4, 2, 16, 32)), dict(v_cache=torch.zeros(5, 2, 16, 64)), dict(page_tokens=8),
    dict(k_cache=torch.zeros(4, 16, 2, 64).transpose(1, 2)), dict(positions=torch.zeros(5, dtype=torch.int64)), dict(positions=torch.zeros(4, dtype=I32)),
    dict(span_begin=torch.zeros(2, dtype=I32)), dict(span_context=torch.zeros(1, dtype=I32)), dict(ancestors=torch.zeros(4, 1, dtype=I32)),
    dict(ancestors=torch.zeros(5, dtype=I32)), dict(ancestors=torch.zeros(5, 1)), dict(block_table=torch.zeros(1, 2, dtype=I32)),
    dict(block_table=torch.zeros(2, 2)), dict(sinks=torch.zeros(3)), dict(sinks=torch.zeros(4, dtype=torch.float64)),
    dict(scratch=torch.zeros(8, dtype=torch.bfloat16)), dict(error_flag=torch.zeros(0, dtype=I32)), dict()])
def test_attention_tree_refuses(changes):
    """Wrong types, sizes and strides; and, with all of them right, tensors that are on no GPU."""
    with pytest.raises(KernelLibraryError, match="attention_tree|float32 and bfloat16"):
        kernels.attention_tree(**tree_arguments(**changes))


@pytest.mark.parametrize("moves", [[(0, 1, 4), (2, 1, 4)], [(0, 1, 4), (1, 2, 4)], [(0, 1)], [(-1, 2, 4)], [(0.5, 1, 2)], [(0, 1 << 31, 1)], [(0, 1, 4)]])
def test_copy_pages_refuses(moves):
    cache = torch.zeros(2, 5, 1, 4, 8)
    with pytest.raises(KernelLibraryError, match="copy_pages"):
        kernels.copy_pages(cache, cache.clone(), moves)


def test_copy_pages_refuses_caches():
    cache = torch.zeros(2, 5, 1, 4, 8)
    for k, v in ((cache[0], cache[0]), (cache, cache[:1]), (cache, cache.bfloat16()), (cache.half(), cache.half()), (cache[..., ::2], cache),
                 (cache, cache.transpose(2, 3).contiguous().transpose(2, 3)[:, :, :, ::2])):
        with pytest.raises(KernelLibraryError):
            kernels.copy_pages(k, v, [(0, 1, 2)])


def test_keep_drafts_refuses():
    cache, i = torch.zeros(2, 5, 1, 4, 8), lambda *n: torch.zeros(*n, dtype=I32)      # noqa: E731
    good = dict(k=cache, v=cache.clone(), parents=i(6), tokens=i(6), chosen=i(6), span_begin=i(3), span_context=i(2), block_table=i(2, 3),
                spans=2, max_nodes=4, path=i(2, 4), accepted=i(2), next_token=i(2), error_flag=i(1))
    for changes in (dict(parents=torch.zeros(6)), dict(tokens=i(6).long()), dict(chosen=i(12)[::2]), dict(span_begin=i(2)), dict(span_context=i(1)),
                    dict(path=i(2, 3)), dict(accepted=i(1)), dict(next_token=i(1)), dict(error_flag=i(0)), dict(block_table=i(1, 3)), dict(v=cache[0]), {}):
        with pytest.raises(KernelLibraryError, match="keep_drafts"):
            kernels.keep_drafts(**{**good, **changes})


def test_token_logprobs_refuses():
    x, i, f = torch.zeros(3, 50), lambda *n: torch.zeros(*n, dtype=I32), torch.zeros      # noqa: E731
    for args in ((x.half(), 3, i(3), f(3)), (x[0], 1, i(3), f(3)), (x.t(), 3, i(3), f(3)), (x, 4, i(4), f(4)), (x, -1, i(3), f(3)), (x, 3, None, f(3)),
                 (x, 3, i(2), f(3)), (x, 3, i(3).long(), f(3)), (x, 3, i(3), f(2)), (x, 3, i(3), f(3).double()), (x, 3, None, None, f(2)),
                 (x, 3, None, None, None, f(3, 2)), (x, 3, None, None, None, f(3, 2), i(3, 3)), (x, 3, None, None, None, f(3, 51), i(3, 51)),
                 (torch.zeros(3, 200), 3, None, None, None, f(3, 129), i(3, 129)), (x, 3, None, None, None, f(2, 2), i(2, 2)),
                 (x, 3, None, None, None, f(3, 2), i(3, 2).long()), (x, 3, i(3), f(3))):
        with pytest.raises(KernelLibraryError, match="token_logprobs|float32 and bfloat16"):
            kernels.token_logprobs(*args)


def test_the_library_refuses_sizes():
    """The checks behind the wrappers, which return before anything is launched."""
    lib = kernels.library()

    def tree(**changes):
        a = dict(tokens=5, spans=2, max_nodes=3, max_keys=9, q_heads=4, kv_heads=2, head_dim=64, page_tokens=16, window=0, words=1, softcap=0.0, dtype=0)
        a.update(changes)
        return lib.celeg_attention_tree(kernels._TREE_RECORD.pack(
            *[0] * 11, 1, 0, 256, 2048, 0, 4, a["words"], 2, a["tokens"], a["spans"], a["max_nodes"], a["max_keys"], a["q_heads"], a["kv_heads"],
            a["head_dim"], a["page_tokens"], a["window"], a["dtype"], 0.1, a["softcap"]))
    for changes in (dict(q_heads=5), dict(head_dim=257), dict(head_dim=0), dict(max_nodes=257, words=9), dict(max_nodes=33), dict(max_nodes=0),
                    dict(tokens=-1), dict(spans=-1), dict(window=-2), dict(softcap=-1.0), dict(dtype=7), dict(spans=70000), dict(page_tokens=0)):
        assert tree(**changes) == -1, changes
    assert tree(tokens=0) == 0 and tree(spans=0) == 0
    moves = np.array([[0, 4, 1]], dtype=np.int32)

    def copy(pages=5, element=4, count=1, dim=8):
        return lib.celeg_copy_pages(kernels._COPY_RECORD.pack(16, 16, moves.ctypes.data, 0, 100, 20, 100, 20, dim, 8, 2, pages, 1, 4, element, count))
    for clash in ([[0, 1, 4], [2, 1, 4]], [[0, 1, 4], [1, 2, 4]], [[3, 3, 1], [3, 4, 1]]):
        moves = np.array(clash, dtype=np.int32)
        assert copy(count=2) == -1 and b"another" in lib.celeg_last_error()
    moves = np.array([[i, 4000 + i, 1] for i in range(3000)] + [[5000, 9000, 1]], dtype=np.int32)      # a table beyond the stack's
    assert copy(pages=10000, count=3001) == -1 and b"move 3000" in lib.celeg_last_error()
    moves = np.array([[0, 4, 1]], dtype=np.int32)
    assert copy(pages=4) == -1 and copy(element=1) == -1 and copy(dim=-1) == -1 and copy(count=-1) == -1 and copy(count=0) == 0

    def keep(max_nodes=4, spans=1, element=2):
        return lib.celeg_keep_drafts(kernels._KEEP_RECORD.pack(16, 16, *[0] * 9, 1, 0, 100, 20, 100, 20, 8, 8, 2, 5, 1, 4, element, 6, 3, spans,
                                                               max_nodes))
    assert keep(max_nodes=257) == -1 and keep(max_nodes=0) == -1 and keep(spans=-1) == -1 and keep(element=3) == -1 and keep(spans=0) == 0

    def logprobs(rows=2, vocab=10, top=0, stride=10, dtype=0, at=16):
        return lib.celeg_token_logprobs(kernels._LOGPROBS_RECORD.pack(at, 0, 0, 0, 16, 16, 0, stride, rows, vocab, top, dtype))
    assert logprobs(vocab=0) == -1 and logprobs(top=11) == -1 and logprobs(stride=9) == -1 and logprobs(dtype=3) == -1 and logprobs(at=18) == -1
    assert logprobs(rows=-1) == -1 and logprobs(vocab=500, stride=500, top=129) == -1 and logprobs(rows=0) == 0


def test_numbers_that_do_not_fit_their_kind_are_refused():
    with pytest.raises(KernelLibraryError, match="not a number of its kind"):
        kernels._record("attention_tree", kernels._TREE_RECORD, *[0] * 13, 0, 0, 0, 1 << 31, *[0] * 12, 0.0, 0.0)
    with pytest.raises(KernelLibraryError, match="not a number of its kind"):
        kernels._record("token_logprobs", kernels._LOGPROBS_RECORD, *[0] * 8, 1.5, 0, 0, 0)
