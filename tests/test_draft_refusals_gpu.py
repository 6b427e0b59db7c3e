"""What the operators behind drafted continuations refuse of tensors that are on a GPU: checks that come behind the device's, and
those of the library behind the wrappers. Nothing is launched, and nothing is written."""
import numpy as np
import pytest
import torch

from celeg_b200.kernels import KernelLibraryError
from test_draft_refusals import keep_arguments
from test_drafts import tree_arguments

pytestmark = pytest.mark.gpu

I32 = torch.int32


def there(arguments):
    return {name: value.cuda() if isinstance(value, torch.Tensor) else value for name, value in arguments.items()}


@pytest.mark.parametrize("changes,reason", [
    (dict(sinks=torch.zeros(3)), "sinks must be .* at least 4 elements"),
    (dict(sinks=torch.zeros(4, dtype=torch.float64)), "sinks must be a contiguous tensor of torch.float32"),
    (dict(scratch=torch.zeros(8, dtype=torch.bfloat16)), "scratch must be a contiguous tensor of torch.float32"),
    (dict(max_nodes=33), "need masks of 2 words, got 1"), (dict(max_nodes=0), "trees of up to 0 nodes"),
    (dict(max_nodes=257, ancestors=torch.zeros(5, 9, dtype=I32)), "at most 256"),
    (dict(kv_heads=3, k_cache=torch.zeros(4, 3, 16, 64), v_cache=torch.zeros(4, 3, 16, 64)), "4 query heads are not a multiple of 3"),
    (dict(window=-1), "window -1"), (dict(softcap=-2.0), "softcap -2"), (dict(max_keys=-1), "invalid sizes"), (dict(max_keys=1 << 31), "not a number"),
])
def test_attention_tree_says_what_is_wrong(changes, reason):
    from celeg_b200 import kernels
    arguments = there(tree_arguments(**changes))
    arguments["out"].fill_(7.0)
    with pytest.raises(KernelLibraryError, match=reason):
        kernels.attention_tree(**arguments)
    torch.cuda.synchronize()
    assert bool((arguments["out"] == 7.0).all()) and int(arguments["error_flag"].item()) == 0


@pytest.mark.parametrize("name", ["q", "out", "k_cache", "v_cache", "positions", "span_begin", "span_context", "ancestors", "block_table", "error_flag",
                                  "sinks", "scratch"])
def test_attention_tree_refuses_a_tensor_that_is_elsewhere(name):
    from celeg_b200 import kernels
    arguments = there(tree_arguments(sinks=torch.zeros(4), scratch=torch.zeros(8)))
    arguments[name] = arguments[name].cpu()
    with pytest.raises(KernelLibraryError, match="attention_tree: .* (on|and) cpu"):
        kernels.attention_tree(**arguments)


@pytest.mark.parametrize("name", ["sinks", "scratch"])
def test_attention_tree_refuses_every_second_number(name):
    from celeg_b200 import kernels
    arguments = there(tree_arguments())
    arguments[name] = torch.zeros(8, device="cuda")[::2]
    with pytest.raises(KernelLibraryError, match=f"{name} must be .* contiguous=False"):
        kernels.attention_tree(**arguments)


@pytest.mark.parametrize("moves,reason", [
    ([(0, 1, 4), (2, 1, 4)], r"move 1 \(page 2 to 1\) writes a page that another one writes"), ([(0, 1, 4), (1, 2, 4)], "reads one that another one writes"),
    ([(3, 3, 1), (3, 4, 1)], "another one writes"), ([(5, 1, 4)], "outside 5 pages of 4"), ([(0, 5, 4)], "outside 5 pages of 4"),
    ([(0, 1, 5)], "outside 5 pages of 4"), ([(0, 1, 4)] * 3000, "another one writes")])
def test_copy_pages_says_what_is_wrong(moves, reason):
    from celeg_b200 import kernels
    k = torch.randn(2, 5, 1, 4, 8, device="cuda")
    v, want = k.clone(), k.clone()
    for given in (moves, np.array(moves), np.array(moves, dtype=np.int32)):
        with pytest.raises(KernelLibraryError, match=reason):
            kernels.copy_pages(k, v, given)
    with pytest.raises(KernelLibraryError, match="keys on cuda:0, values on cpu"):
        kernels.copy_pages(k, v.cpu(), [(0, 1, 4)])
    torch.cuda.synchronize()
    assert torch.equal(k, want) and torch.equal(v, want)


@pytest.mark.parametrize("name", ["parents", "tokens", "chosen", "span_begin", "span_context", "block_table", "path", "accepted", "next_token", "error_flag"])
def test_keep_drafts_refuses_a_tensor_that_is_elsewhere(name):
    from celeg_b200 import kernels
    arguments = there(keep_arguments())
    arguments[name] = arguments[name].cpu()
    with pytest.raises(KernelLibraryError, match="keep_drafts: .* on cpu"):
        kernels.keep_drafts(**arguments)


@pytest.mark.parametrize("changes,reason", [(dict(max_nodes=257, path=torch.zeros(2, 257, dtype=I32)), "at most 65535 and 256"),
                                            (dict(max_nodes=0), "up to 0 nodes"), (dict(spans=-1), "-1 spans")])
def test_keep_drafts_says_what_is_wrong(changes, reason):
    from celeg_b200 import kernels
    with pytest.raises(KernelLibraryError, match=reason):
        kernels.keep_drafts(**there(keep_arguments(**changes)))


def test_token_logprobs_says_what_is_wrong():
    from celeg_b200 import kernels
    x, tokens, out = torch.zeros(3, 50, device="cuda"), torch.zeros(3, dtype=I32, device="cuda"), torch.zeros(3, device="cuda")
    for arguments, reason in (((x, 3, tokens.cpu(), out), "tokens on cpu"), ((x, 3, tokens, out.cpu()), "logprobs on cpu"),
                              ((x, 3, tokens, out, out.cpu()), "entropy on cpu"), ((x.cpu(), 3, tokens, out), "on cuda:0, other tensors on device -1"),
                              ((x[:1].expand(3, 50), 3, tokens, out), "row_stride=0")):
        with pytest.raises(KernelLibraryError, match=reason):
            kernels.token_logprobs(*arguments)
