"""What the drafted trees' front end does on the host, and what the C ABI refuses."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests import tree_ref as R
from vllm_webgpu_amd import _lib
from vllm_webgpu_amd.v1.kv_cache import PagedKVCache
from vllm_webgpu_amd.v1.sample.tree_sampler import DraftTree

FAKE = 0x10000          # stand-in addresses: validation never dereferences them


def test_trees():
    g = torch.Generator().manual_seed(0)
    parents = [R.random_tree(n, g) for n in (1, 70, 256, 3)]
    t = DraftTree.make(parents, torch.device("cpu"))
    assert t.cu_nodes.tolist() == [0, 1, 71, 327, 330] and t.max_nodes == 256 and t.num_nodes == [1, 70, 256, 3]
    assert t.parents.tolist() == [p for tree in parents for p in tree]
    assert t.requests.tolist() == [0] + [1] * 70 + [2] * 256 + [3] * 3
    for i, tree in enumerate(parents):
        lo = int(t.cu_nodes[i])
        see = R.sees(tree)
        assert torch.equal(t.visible[lo:lo + len(tree)], R.pack(see, 256))
        assert t.depths[lo:lo + len(tree)].tolist() == (see.sum(1) - 1).tolist()
        assert t.numbers[lo:lo + len(tree)].tolist() == list(range(len(tree)))
    assert t.max_depth == int(t.depths.max())


@pytest.mark.parametrize("parents", [[], [[]], [[0]], [[-1, 1]], [[-1, -1]], [[-1] + [0] * 256], [[-1, 0], [-1, 2, 0]]])
def test_trees_that_are_none(parents):
    with pytest.raises(ValueError):
        DraftTree.make(parents, torch.device("cpu"))


def test_pages():
    c = PagedKVCache(2, 10, 2, 64, page_size=8, device="cpu")
    assert len(c.k) == 2 and c.k[0].shape == (10, 2, 8, 64) and c.v[1].shape == (10, 2, 64, 8)
    c.reserve("a", 17)
    c.reserve("b", 1)
    c.reserve("a", 18)
    c.reserve("b", 16)
    assert c.block_table(["b", "a"]).tolist() == [[3, 4, -1], [0, 1, 2]]
    with pytest.raises(RuntimeError):
        c.reserve("c", 48)
    assert "c" not in c._pages
    tree = DraftTree.make([[-1, 0, 0], [-1, 0]], torch.device("cpu"))
    slots = c.slots(c.block_table(["a", "b"]), torch.tensor([7, 14]), tree)
    assert slots.tolist() == [7, 8, 9, 4 * 8 + 6, 4 * 8 + 7] and slots.dtype == torch.int32
    c.release("a")
    c.reserve("d", 8 * 8)
    assert sorted(c._pages["d"] + c._pages["b"]) == list(range(10))
    assert c.block_table([]).shape == (0, 1)


def cache(**over):
    c = _lib.KvCache(FAKE, FAKE, 2 * 16 * 64, 2 * 16 * 64, 10, 16, 2, 64, _lib.DTYPE_BF16)
    for k, v in over.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [
    (dict(k=None), _lib.ERR_INVALID_ARGUMENT), (dict(v=FAKE + 8), _lib.ERR_INVALID_ARGUMENT), (dict(dtype=_lib.DTYPE_F32), _lib.ERR_UNSUPPORTED_DTYPE),
    (dict(page_size=12), _lib.ERR_LIMIT), (dict(page_size=4), _lib.ERR_LIMIT), (dict(page_size=512), _lib.ERR_LIMIT),
    (dict(head_dim=80), _lib.ERR_LIMIT), (dict(kv_heads=0), _lib.ERR_LIMIT), (dict(num_pages=0), _lib.ERR_LIMIT),
    (dict(num_pages=2 ** 28), _lib.ERR_LIMIT), (dict(k_page_stride=2 * 16 * 64 - 8), _lib.ERR_INVALID_ARGUMENT),
    (dict(v_page_stride=2 * 16 * 64 + 4), _lib.ERR_INVALID_ARGUMENT),
]


def append_args(c, **over):
    a = _lib.AppendArgs(ctypes.sizeof(_lib.AppendArgs), 5, c, FAKE, 128, 64, FAKE, 128, 64, FAKE, FAKE, FAKE, 64, 0, 1.0, 4, FAKE, 256, 64,
                        FAKE, 256, 64, None)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def tree_args(L, c, **over):
    a = _lib.TreeAttentionArgs(ctypes.sizeof(_lib.TreeAttentionArgs), 3, c, 9, 4, 4, FAKE, 256, 64, FAKE, 256, 64, FAKE, 7, 7, FAKE, FAKE,
                               FAKE, 1, 0.125, 0x100000, L.vws_tree_attention_workspace_size(3, 4, 4, 2, 64, 16, 7), None)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def score_args(L, **over):
    a = _lib.TokenLogprobsArgs(ctypes.sizeof(_lib.TokenLogprobsArgs), 6, 1000, _lib.DTYPE_F32, FAKE, 1000, FAKE, 1.0, 5, FAKE, FAKE, FAKE,
                               FAKE, FAKE, FAKE, 6 * 32, FAKE, FAKE, 0x4000000, 1000, 0x100000, L.vws_token_logprobs_workspace_size(6, 1000, 5), None)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_the_abi_refuses():
    L = _lib.lib()

    def refused(status, want):
        assert status == want and L.vws_last_error(), (status, want, L.vws_last_error())

    for change, want in BAD_CACHES:
        c = cache(**change)
        refused(L.vws_append_kv(ctypes.byref(append_args(c))), want)
        refused(L.vws_compact_kv(ctypes.byref(c), 1, FAKE, 4, 4, FAKE, FAKE, 3, 3, None), want)
        refused(L.vws_tree_attention(ctypes.byref(tree_args(L, c))), want)
    I, M, W = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_LIMIT, _lib.ERR_WORKSPACE_TOO_SMALL
    for change, want in ((dict(struct_size=4), I), (dict(tokens=0), I), (dict(k=None), I), (dict(slots=None), I), (dict(inv_freq=None), I),
                         (dict(rotary_dim=8), M), (dict(rotary_dim=128), M), (dict(rotary_dim=40), M), (dict(rope_scale=float("nan")), I),
                         (dict(heads=-1), M), (dict(q=None), I), (dict(q_out=None), I), (dict(tokens=2 ** 24), M)):
        refused(L.vws_append_kv(ctypes.byref(append_args(cache(), **change))), want)
    refused(L.vws_append_kv(None), I)
    for change, want in ((dict(struct_size=4), I), (dict(batch=0), I), (dict(nodes=0), I), (dict(max_nodes=0), M), (dict(max_nodes=257), M),
                         (dict(heads=3), I), (dict(heads=0), I), (dict(q=None), I), (dict(cu_nodes=None), I), (dict(max_pages=0), I),
                         (dict(block_table_row_stride=6), I), (dict(visible_row_stride=0), I), (dict(scale=0.0), I),
                         (dict(scale=float("nan")), I), (dict(workspace=None), W), (dict(workspace_bytes=8), W), (dict(workspace=0x100010), I),
                         (dict(batch=2 ** 24), M)):
        refused(L.vws_tree_attention(ctypes.byref(tree_args(L, cache(), **change))), want)
    for args, want in (((0, FAKE, 4, 4, FAKE, FAKE, 3, 3), I), ((2 ** 24, FAKE, 4, 4, FAKE, FAKE, 3, 3), M), ((1, None, 4, 4, FAKE, FAKE, 3, 3), I),
                       ((1, FAKE, 3, 4, FAKE, FAKE, 3, 3), I), ((1, FAKE, 4, 0, FAKE, FAKE, 3, 3), I), ((1, FAKE, 4, 4, FAKE, FAKE, 257, 257), M),
                       ((1, FAKE, 4, 4, FAKE, FAKE, 2, 3), I)):
        refused(L.vws_compact_kv(ctypes.byref(cache()), *args, None), want)
    refused(L.vws_compact_kv(None, 1, FAKE, 4, 4, FAKE, FAKE, 3, 3, None), I)
    for args, want in (((0, 5, FAKE, FAKE, FAKE, FAKE, 3, FAKE, FAKE, FAKE), M), ((1, -1, FAKE, FAKE, FAKE, FAKE, 3, FAKE, FAKE, FAKE), I),
                       ((1, 5, None, FAKE, FAKE, FAKE, 3, FAKE, FAKE, FAKE), I), ((1, 5, FAKE, FAKE, FAKE, None, 3, FAKE, FAKE, FAKE), I),
                       ((1, 5, FAKE, FAKE, FAKE, FAKE, 0, FAKE, FAKE, FAKE), M), ((1, 5, FAKE, FAKE, FAKE, FAKE, 257, FAKE, FAKE, FAKE), M)):
        refused(L.vws_accept_tree(*args, None), want)
    for change, want in ((dict(struct_size=4), I), (dict(rows=0), I), (dict(vocab=2 ** 20), M), (dict(dtype=9), _lib.ERR_UNSUPPORTED_DTYPE),
                         (dict(temperature=0.0), I), (dict(temperature=float("inf")), I), (dict(token_ids=None), I), (dict(saved_bytes=8), W),
                         (dict(saved=FAKE + 4), I)):
        a = score_args(L, **change)
        refused(L.vws_token_logprobs_forward(ctypes.byref(a)), want)
        refused(L.vws_token_logprobs_backward(ctypes.byref(a)), want)
    for change, want in ((dict(num_logprobs=65), M), (dict(num_logprobs=-2), M), (dict(logprobs=None), I), (dict(logprob_ids=None), I),
                         (dict(workspace_bytes=8), W), (dict(workspace=0x100010), I), (dict(vocab=4), I)):
        refused(L.vws_token_logprobs_forward(ctypes.byref(score_args(L, **change))), want)
    for change, want in ((dict(saved=None), W), (dict(grad=None), I), (dict(grad_row_stride=999), I), (dict(grad=FAKE + 64), I)):
        refused(L.vws_token_logprobs_backward(ctypes.byref(score_args(L, **change))), want)


def test_workspace_sizes():
    L = _lib.lib()
    fixed = L.vws_sample_workspace_size(1, 1, 0)
    assert L.vws_token_logprobs_saved_size(7) == 7 * 32 and L.vws_token_logprobs_saved_size(0) == 0
    few, many = L.vws_token_logprobs_workspace_size(3, 128256, 20), L.vws_token_logprobs_workspace_size(5000, 128256, 20)
    assert few > fixed and few % 256 == 0 and many > fixed
    # the last of several launches may be split further than the others
    assert L.vws_token_logprobs_workspace_size(8193, 128256, 64) >= L.vws_token_logprobs_workspace_size(1, 128256, 64)
    for bad in ((0, 10, 1), (1, 0, 1), (1, 10, 65), (1, 10, -2), (1, 2 ** 20, 0)):
        assert L.vws_token_logprobs_workspace_size(*bad) == 0
    one = L.vws_tree_attention_workspace_size(1, 16, 32, 8, 128, 16, 512)
    assert one > fixed and one % 256 == 0
    assert L.vws_tree_attention_workspace_size(2000, 16, 32, 8, 128, 16, 4) == fixed       # (nothing to join)
    for bad in ((0, 1, 8, 8, 64, 16, 1), (1, 0, 8, 8, 64, 16, 1), (1, 257, 8, 8, 64, 16, 1), (1, 1, 8, 3, 64, 16, 1), (1, 1, 8, 8, 64, 16, 0)):
        assert L.vws_tree_attention_workspace_size(*bad) == 0


def test_keys_and_values_share_no_element():
    L = _lib.lib()
    page = 2 * 16 * 64
    for v, ks, vs in ((0, page, page), (2 * 8, page, page), (9 * 2 * page, page, page), (page, 2 * page, 2 * page), (2 * page, 2 * page, 3 * page),
                      (-2 * page + 16, 3 * page, 3 * page)):
        c = cache(k=1 << 30, v=(1 << 30) + v, k_page_stride=ks, v_page_stride=vs)
        for status in (L.vws_append_kv(ctypes.byref(append_args(c))), L.vws_tree_attention(ctypes.byref(tree_args(L, c))),
                       L.vws_compact_kv(ctypes.byref(c), 1, FAKE, 4, 4, FAKE, FAKE, 3, 3, None)):
            assert status == _lib.ERR_INVALID_ARGUMENT and b"overlap" in L.vws_last_error()


def test_slots_past_a_requests_pages():
    """Nodes behind the pages that a request holds have no slot."""
    c = PagedKVCache(1, 10, 1, 64, page_size=16, device="cpu")
    c.reserve("a", 20)
    c.reserve("b", 40)
    tree = DraftTree.make([[-1, 0, 1], [-1, 0, 1]], torch.device("cpu"))
    t = c.block_table(["a", "b"])
    slots = c.slots(t, torch.tensor([31, 46]), tree).tolist()
    assert slots == [int(t[0, 1]) * 16 + 15, -1, -1, int(t[1, 2]) * 16 + 14, int(t[1, 2]) * 16 + 15, -1]
