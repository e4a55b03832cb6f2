"""Attention of drafted trees whose rows share the keys' tiles (more than 32 rows a request, many workgroups), and what
outputs may overlap, against 64-bit forms."""
from __future__ import annotations

import pytest
import torch

from tests import tree_ref as R
from tests.test_gpu_tree import check
from tests.test_gpu_tree import setup as arguments
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def widen(args, columns):
    """More columns in the table: the call is laid out for longer contexts."""
    t = args["block_table"]
    args["block_table"] = torch.cat([t, torch.full((t.shape[0], columns - t.shape[1]), -1, device=t.device).int()], 1)


# requests of 256, 4, 48, 80 and 132 rows: waves that share eight, four, two or no rows' tiles, idle ones, a second workgroup
@pytest.mark.parametrize("dim,page,dtype", [(64, 8, "f16"), (96, 32, "bf16"), (128, 16, "bf16"), (128, 256, "f16"), (192, 16, "f16"), (256, 8, "bf16")])
@pytest.mark.parametrize("chain", [False, True])
def test_rows_of_all_counts(cuda, dim, page, dtype, chain):
    contexts = [0, 1, 33, 511, 3000]
    args, see, cu = arguments(cuda, contexts, [64, 1, 12, 20, 33], 8, 2, dim, page, dtype, seed=dim + page, chain=chain)
    check(args, see, cu, contexts)


@pytest.mark.parametrize("B,dim,dtype", [(200, 128, "bf16"), (300, 64, "f16"), (200, 256, "f16"), (300, 96, "bf16")])
def test_many_requests(cuda, B, dim, dtype):
    """Undivided requests, ordered by their length up to 256 of them."""
    g = torch.Generator().manual_seed(B + dim)
    contexts, nodes = torch.randint(0, 600, (B,), generator=g).tolist(), torch.randint(1, 13, (B,), generator=g).tolist()
    args, see, cu = arguments(cuda, contexts, nodes, 8, 2, dim, 16, dtype, seed=B)
    check(args, see, cu, contexts)


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_hidden_nodes_may_hold_anything(cuda, bad, dim):
    """Node 2 is no number in its value, and nobody but node 30 sees it."""
    contexts = [37, 500]
    args, see, cu = arguments(cuda, contexts, [40, 40], 4, 2, dim, 16, "bf16", seed=dim)
    for s in see:
        s[:, 2] = False
        s[30, 2] = True
    args["visible"] = R.pack(torch.cat(see), 40).to(cuda)
    widen(args, 2400)
    want, bound = R.attention(args["q"], args["k_cache"], args["v_cache"], args["block_table"], contexts, cu, see)
    for b, c in enumerate(contexts):
        page, off = int(args["block_table"][b, (c + 2) // 16]), (c + 2) % 16
        args["v_cache"][page, :, 8:40, off] = bad
    out = ops.tree_attention(**args)
    rows = [i for i in range(80) if i % 40 != 30]
    assert bool(((out[rows].double() - want[rows]).abs() <= bound[rows]).all())
    for r in (30, 70):
        o = out[r].double()
        assert bool(torch.isnan(o[:, 8:40]).all() if bad != bad else (o[:, 8:40] == bad).all())
        assert bool(((o - want[r]).abs() <= bound[r])[:, 40:].all())


@pytest.mark.parametrize("dim", [128, 256])
def test_pages_that_do_not_exist_are_not_seen(cuda, dim):
    """The same as a request without the keys of those pages, whose other keys keep their order."""
    args, see, cu = arguments(cuda, [160], [40], 4, 2, dim, 16, "f16", seed=dim + 1)
    table = args["block_table"]
    short = {**args, "block_table": torch.cat([table[:, :3], table[:, 5:9], table[:, 10:]], 1).contiguous(),
             "context_lens": args["context_lens"] - 48}
    want, bound = R.attention(args["q"], args["k_cache"], args["v_cache"], short["block_table"], [112], cu, see)
    for at, page in ((3, -1), (4, 10 ** 9), (9, args["k_cache"].shape[0])):
        table[0, at] = page
    widen(args, 4800)
    assert bool(((ops.tree_attention(**args).double() - want).abs() <= bound).all())


# one part, parts that are joined, rows that share tiles
@pytest.mark.parametrize("context,nodes,columns,dim", [(20, 3, 2, 64), (3000, 3, 200, 64), (3000, 40, 2400, 128), (700, 40, 2400, 256)])
def test_queries_that_are_no_numbers(cuda, context, nodes, columns, dim):
    args, see, cu = arguments(cuda, [context], [nodes], 4, 2, dim, 16, "bf16", seed=context)
    widen(args, max(columns, args["block_table"].shape[1]))
    want, bound = R.attention(args["q"], args["k_cache"], args["v_cache"], args["block_table"], [context], cu, see)
    args["q"][1, 2, 5] = float("nan")
    out = ops.tree_attention(**args)
    rest = torch.ones(out.shape[:2], dtype=torch.bool)
    rest[1, 2] = False
    assert bool(torch.isnan(out[1, 2]).all()) and bool(((out.double() - want).abs() <= bound)[rest].all())


def test_out_beside_the_queries(cuda):
    """Queries and outputs side by side in one buffer's rows; heads outermost; an overlap is refused."""
    args, see, cu = arguments(cuda, [45, 200], [6, 3], 6, 2, 64, 16, "f16", seed=12)
    want = ops.tree_attention(**args)
    both = torch.zeros((9, 12, 64), dtype=torch.float16, device=cuda)
    both[:, :6] = args["q"]
    assert torch.equal(ops.tree_attention(**{**args, "q": both[:, :6]}, out=both[:, 6:]), want) and torch.equal(both[:, :6], args["q"])
    heads = torch.zeros((6, 9, 64), dtype=torch.float16, device=cuda)
    assert torch.equal(ops.tree_attention(**args, out=heads.transpose(0, 1)).contiguous(), want)
    assert torch.equal(heads.transpose(0, 1), want)
    for out in (both[:, 5:11], both[:, :6]):
        with pytest.raises(ValueError):
            ops.tree_attention(**{**args, "q": both[:, :6]}, out=out)
    cache = args["v_cache"].flatten()[:9 * 6 * 64]
    with pytest.raises(ValueError):
        ops.tree_attention(**args, out=cache.view(9, 6, 64))


def test_append_refuses_overlaps(cuda):
    """Queries may be turned in place beside their keys in one projection's rows, not on them, nor on the cache."""
    T, dim = 5, 64
    kc, vc = R.make_cache(cuda, 4, 2, 16, dim, "bf16")
    rows = torch.randn((T, 8, dim), device=cuda).bfloat16()
    q, k, v = rows[:, :4], rows[:, 4:6], rows[:, 6:]
    slots, pos = torch.arange(T, device=cuda).int(), torch.arange(T, device=cuda).int()
    f = torch.ones(dim // 2, device=cuda)
    want = R.rotate(q, pos, f)[0]
    args = dict(slots=slots, positions=pos, inv_freq=f)
    for out, keys, values in ((q, rows[:, 3:5], v), (q, k, rows[:, 2:4]), (kc.view(-1, 4, dim)[:T], k, v), (vc.view(-1, 4, dim)[:T], k, v),
                              (rows[:, 1:5], k, v), (rows[:, 3:7], k, v)):
        with pytest.raises(ValueError):
            ops.append_kv(keys, values, kc, vc, q=q, out=out, **args)
    with pytest.raises(ops._lib.VwsError):
        both = torch.zeros((4, 2, 64, 64), dtype=torch.bfloat16, device=cuda)
        ops.append_kv(k, v, both, both, slots)
    # (pages of keys and values in turn do not overlap)
    pair = torch.zeros((4, 2, 2 * 16 * dim), dtype=torch.bfloat16, device=cuda)
    kp, vp = pair[:, 0].view(4, 2, 16, dim), pair[:, 1].view(4, 2, dim, 16)
    ops.append_kv(k, v, kp, vp, slots)
    assert torch.equal(kp[0, :, :T], k.transpose(0, 1)) and torch.equal(vp[0, :, :, :T], v.permute(1, 2, 0))
    assert ops.append_kv(k, v, kc, vc, q=q, out=q, **args).data_ptr() == q.data_ptr()
    # (a product, a sum and a rounding: 2^-8 of the result, and less than 2^-20 of values of at most 8)
    assert bool(((q.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -17).all())


def test_gradients_of_logits_saved_elsewhere(cuda):
    """Logits that come back at their address with other rows between them."""
    from vllm_webgpu_amd.ops import token_logprobs
    wide = torch.randn((6, 1032), device=cuda)
    ids = torch.tensor([3, 999, -1, 0, 512, 7], device=cuda)
    x = wide[:, :1000].clone().requires_grad_()
    token_logprobs(x, ids).logprobs.sum().backward()
    leaf = wide.requires_grad_()

    def pack(t):
        return t if t.shape != (6, 1000) else t.detach().clone()

    def unpack(t):
        if t.shape != (6, 1000):
            return t
        with torch.no_grad():
            leaf.data.view(-1)[:6000] = t.reshape(-1)
        return leaf.data.view(-1)[:6000].view(6, 1000)

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        r = token_logprobs(leaf[:, :1000], ids)
    r.logprobs.sum().backward()
    assert torch.equal(leaf.grad[:, :1000], x.grad) and not bool(leaf.grad[:, 1000:].any())
