"""What the operators behind drafted continuations refuse, each by the reason that its message gives; without a GPU."""
import pytest
import torch

from celeg_b200 import kernels
from celeg_b200.kernels import KernelLibraryError
from test_drafts import tree_arguments

I32 = torch.int32


def zeros(*shape):
    return torch.zeros(*shape, dtype=I32)


@pytest.mark.parametrize("changes,reason", [
    (dict(q=torch.zeros(5, 256, dtype=torch.float16)), "float32 and bfloat16"),
    (dict(q=torch.zeros(5, 256, dtype=torch.bfloat16)), "q torch.bfloat16, caches torch.float32"),
    (dict(v_cache=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)), "caches torch.float32 and torch.bfloat16"),
    (dict(out=torch.zeros(4, 256)), "out must be .* at least 1280 elements"),
    (dict(out=torch.zeros(5, 256, dtype=torch.bfloat16)), "out must be a contiguous tensor of torch.float32"),
    (dict(out=torch.zeros(5, 512)[:, :256]), "out must be .* contiguous=False"),
    (dict(q=torch.zeros(4, 256)), "does not hold 5 rows of 4 x 64"),
    (dict(q=torch.zeros(5, 255)), "does not hold 5 rows of 4 x 64"),
    (dict(q=torch.zeros(256, 5).t()), "does not hold 5 rows of 4 x 64"),
    (dict(q_row_stride=300), "300 apart"),
    (dict(k_cache=torch.zeros(4, 2, 16, 32)), "in one piece are needed"),
    (dict(v_cache=torch.zeros(5, 2, 16, 64)), "in one piece are needed"),
    (dict(page_tokens=8), r"with pages \(2, 8, 64\)"),
    (dict(kv_heads=1), r"with pages \(1, 16, 64\)"),
    (dict(k_cache=torch.zeros(4, 16, 2, 64).transpose(1, 2)), "in one piece are needed"),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), "positions must be a contiguous tensor of torch.int32"),
    (dict(positions=zeros(4)), "positions must be .* at least 5 elements"),
    (dict(span_begin=zeros(2)), "span_begin must be .* at least 3 elements"),
    (dict(span_context=zeros(1)), "span_context must be .* at least 2 elements"),
    (dict(ancestors=zeros(4, 1)), r"ancestors \(4, 1\) for 5 tokens"),
    (dict(ancestors=zeros(5)), r"ancestors \(5,\) for 5 tokens"),
    (dict(ancestors=torch.zeros(5, 1)), "ancestors must be a contiguous tensor of torch.int32"),
    (dict(ancestors=zeros(5, 2)[:, :1]), "ancestors must be .* contiguous=False"),
    (dict(block_table=zeros(1, 2)), r"a block table \(1, 2\) of torch.int32 .* for 2 spans"),
    (dict(block_table=zeros(4)), r"a block table \(4,\)"),
    (dict(block_table=torch.zeros(2, 2)), r"a block table \(2, 2\) of torch.float32"),
    (dict(block_table=zeros(2, 4)[:, ::2]), r"with strides \(4, 2\)"),
    (dict(error_flag=zeros(0)), "error_flag must be .* at least 1 elements"),
    (dict(), "tensors of CUDA device -1"),
])
def test_attention_tree_says_what_is_wrong(changes, reason):
    with pytest.raises(KernelLibraryError, match=reason):
        kernels.attention_tree(**tree_arguments(**changes))


@pytest.mark.parametrize("moves,reason", [
    ([(0, 1)], "triples of whole numbers"), ([0, 1, 2], "triples of whole numbers"), ([(0.5, 1, 2)], "triples of whole numbers"),
    ([(-1, 2, 4)], "negative or too large"), ([(0, 1 << 31, 1)], "negative or too large"), ([(0, 1, 4)], "tensors of CUDA device -1"),
])
def test_copy_pages_says_what_is_wrong(moves, reason):
    cache = torch.zeros(2, 5, 1, 4, 8)
    with pytest.raises(KernelLibraryError, match=reason):
        kernels.copy_pages(cache, cache.clone(), moves)


def keep_arguments(**changes):
    cache = torch.zeros(2, 5, 1, 4, 8)
    return {**dict(k=cache, v=cache.clone(), parents=zeros(6), tokens=zeros(6), chosen=zeros(6), span_begin=zeros(3), span_context=zeros(2),
                   block_table=zeros(2, 3), spans=2, max_nodes=4, path=zeros(2, 4), accepted=zeros(2), next_token=zeros(2),
                   error_flag=zeros(1)), **changes}


@pytest.mark.parametrize("k,v,reason", [
    (torch.zeros(5, 1, 4, 8), torch.zeros(5, 1, 4, 8), "of one type are needed"),
    (torch.zeros(2, 5, 1, 4, 8), torch.zeros(1, 5, 1, 4, 8), "of one type are needed"),
    (torch.zeros(2, 5, 1, 4, 8), torch.zeros(2, 5, 1, 4, 8, dtype=torch.bfloat16), "of one type are needed"),
    (torch.zeros(2, 5, 1, 4, 8, dtype=torch.float16), torch.zeros(2, 5, 1, 4, 8, dtype=torch.float16), "float32 and bfloat16"),
    (torch.zeros(2, 5, 1, 4, 16)[..., ::2], torch.zeros(2, 5, 1, 4, 8), "must lie side by side"),
    (torch.zeros(2, 5, 1, 4, 8), torch.zeros(2, 5, 1, 8, 8)[:, :, :, ::2], "must lie side by side"),
])
def test_caches_that_cannot_be_moved(k, v, reason):
    with pytest.raises(KernelLibraryError, match=reason):
        kernels.copy_pages(k, v, [(0, 1, 2)])
    with pytest.raises(KernelLibraryError, match=reason):
        kernels.keep_drafts(**keep_arguments(k=k, v=v))


@pytest.mark.parametrize("changes,reason", [
    (dict(parents=torch.zeros(6)), "parents must be a contiguous tensor of torch.int32"), (dict(tokens=zeros(6).long()), "tokens must be"),
    (dict(chosen=zeros(12)[::2]), "chosen must be .* contiguous=False"), (dict(span_begin=zeros(2)), "span_begin must be .* at least 3"),
    (dict(span_context=zeros(1)), "span_context must be .* at least 2"), (dict(path=zeros(2, 3)), "path must be .* at least 8"),
    (dict(accepted=zeros(1)), "accepted must be .* at least 2"), (dict(next_token=zeros(1)), "next_token must be .* at least 2"),
    (dict(error_flag=zeros(0)), "error_flag must be .* at least 1"), (dict(block_table=zeros(1, 3)), r"a block table \(1, 3\)"),
    (dict(block_table=zeros(2, 3).long()), "a block table .* of torch.int64"), (dict(), "tensors of CUDA device -1")])
def test_keep_drafts_says_what_is_wrong(changes, reason):
    with pytest.raises(KernelLibraryError, match=reason):
        kernels.keep_drafts(**keep_arguments(**changes))


X, F = torch.zeros(3, 50), torch.zeros


@pytest.mark.parametrize("arguments,reason", [
    ((X.half(), 3, zeros(3), F(3)), "float32 and bfloat16"), ((X[0], 1, zeros(3), F(3)), r"logits \(50,\)"),
    ((X.t(), 3, zeros(3), F(3)), r"with strides \(1, 50\)"), ((X, 4, zeros(4), F(4)), "for 4 rows"), ((X, -1, zeros(3), F(3)), "for -1 rows"),
    ((X, 3, None, F(3)), "log probabilities of no tokens"), ((X, 3, zeros(2), F(3)), "tokens must be .* at least 3"),
    ((X, 3, zeros(3).long(), F(3)), "tokens must be a contiguous tensor of torch.int32"), ((X, 3, zeros(3), F(2)), "logprobs must be .* at least 3"),
    ((X, 3, zeros(3), F(3).double()), "logprobs must be a contiguous tensor of torch.float32"),
    ((X, 3, None, None, F(2)), "entropy must be .* at least 3"), ((X, 3, None, None, None, F(3, 2)), "come together"),
    ((X, 3, None, None, None, None, zeros(3, 2)), "come together"),
    ((X, 3, None, None, None, F(3, 2), zeros(3, 3)), r"top_logprobs \(3, 2\) and top_tokens \(3, 3\)"),
    ((X, 3, None, None, None, F(3, 51), zeros(3, 51)), "51 alternatives"),
    ((F(3, 200), 3, None, None, None, F(3, 129), zeros(3, 129)), "129 alternatives"),
    ((X, 3, None, None, None, F(2, 2), zeros(2, 2)), "top_logprobs must be .* at least 6"),
    ((X, 3, None, None, None, F(3, 2), zeros(3, 2).long()), "top_tokens must be a contiguous tensor of torch.int32"),
    ((X, 3, zeros(3), F(3)), "tensors of CUDA device -1")])
def test_token_logprobs_says_what_is_wrong(arguments, reason):
    with pytest.raises(KernelLibraryError, match=reason):
        kernels.token_logprobs(*arguments)
