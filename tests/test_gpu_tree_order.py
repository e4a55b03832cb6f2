"""Which kernel, parts and order of requests a drafted trees' attention takes: every combination against 64-bit forms, and
contexts that reach past their table."""
from __future__ import annotations

import pytest
import torch

from tests import tree_ref as R
from tests.test_gpu_tree import check
from tests.test_gpu_tree import setup as arguments
from tests.test_gpu_tree_wide import widen
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def plan(args):
    """(rows a workgroup, parts, whether requests are taken longest first) as the launcher chooses them; what of it the size of the
    workspace shows is checked against that, so that a changed choice does not go unnoticed."""
    (_, Hk, page, D), (B, W), H, N = args["k_cache"].shape, args["block_table"].shape, args["q"].shape[1], args["max_nodes"]
    need, most = N * (H // Hk), min(W * page, 0x7FFF0000)
    few = 16 if D > 128 else 32
    wide = need > 32 and B * Hk * -(-need // few) * -(-most // 256) > 512
    rows = 128 if wide else 16 if need <= 16 else few
    slots, blocks = 256 if wide or D > 128 else 512, -(-need // rows)
    items = B * Hk * blocks
    s = max(1, min((512 if items * 8 > 256 and (wide or D <= 128) else 256) // items, most // 256, 256))
    chunk = -(-(-(-most // s)) // 128) * 128
    splits = -(-most // chunk)
    L = ops._lib.lib()
    recs = B * splits * Hk * blocks * rows if splits > 1 else 0
    size = L.vws_sample_workspace_size(1, 1, 0) + -(-4 * recs * D // 256) * 256 + -(-8 * recs // 256) * 256
    assert L.vws_tree_attention_workspace_size(B, N, H, Hk, D, page, W) == size
    return rows, splits, 1 < B <= 256 and B * splits * Hk * blocks > slots


def ragged(B, most, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, most, (B,), generator=g).tolist(), g


@pytest.mark.parametrize("B,nodes,heads,kv_heads,dim,columns,dtype,want", [
    (20, 32, 8, 2, 128, 512, "bf16", (128, 11, True)),      # parts of reordered requests
    (16, 40, 4, 2, 256, 640, "f16", (128, 8, False)),
    (50, 1, 8, 4, 64, 256, "f16", (16, 2, False)),
    (40, 6, 16, 4, 96, 512, "bf16", (32, 3, False)),
    (20, 8, 8, 4, 192, 256, "f16", (16, 3, False)),
    (200, 1, 8, 8, 128, 40, "bf16", (16, 1, True)),         # plain decoding of a batch
    (256, 1, 4, 1, 64, 40, "f16", (16, 2, False)),
    (257, 1, 4, 4, 64, 40, "f16", (16, 1, False)),          # one request too many to be ordered
    (256, 1, 4, 4, 64, 40, "f16", (16, 1, True)),
    (100, 6, 32, 8, 128, 40, "f16", (32, 1, True)),
    (90, 2, 16, 4, 256, 40, "bf16", (16, 1, True)),
    (150, 12, 8, 2, 192, 40, "bf16", (128, 1, True)),
    (3, 8, 16, 2, 128, 1200, "bf16", (128, 38, False)),
])
def test_every_plan(cuda, B, nodes, heads, kv_heads, dim, columns, dtype, want):
    contexts, g = ragged(B, 500, B + dim)
    counts = torch.randint(1, nodes + 1, (B,), generator=g).tolist()
    counts[B // 2] = nodes
    args, see, cu = arguments(cuda, contexts, counts, heads, kv_heads, dim, 16, dtype, seed=B)
    widen(args, columns)
    assert plan(args) == want
    check(args, see, cu, contexts)


@pytest.mark.parametrize("B,nodes,heads,kv_heads,dim,columns,want", [
    (200, 5, 8, 8, 64, 40, (16, 1, True)), (60, 6, 16, 4, 128, 256, (32, 2, False)), (40, 32, 8, 2, 128, 256, (128, 6, True)),
    (150, 12, 8, 2, 256, 40, (128, 1, True)),
])
def test_empty_and_ill_bounded_requests_among_the_ordered(cuda, B, nodes, heads, kv_heads, dim, columns, want):
    """Requests without a node and of more nodes than the call is laid out for come last and leave their rows."""
    contexts, g = ragged(B, 400, B)
    counts = torch.randint(1, nodes + 1, (B,), generator=g).tolist()
    empty, long = {1, B // 2, B - 1}, {0, B // 3, B - 5}
    for b in empty:
        counts[b] = 0
    for b in long:
        counts[b] = nodes + 1 + b % 2
    args, see, cu = arguments(cuda, contexts, counts, heads, kv_heads, dim, 16, "bf16", seed=B)
    args["max_nodes"] = nodes
    widen(args, columns)
    assert plan(args) == want
    wanted, bound = R.attention(args["q"], args["k_cache"], args["v_cache"], args["block_table"], contexts, cu, see)
    out = ops.tree_attention(**args, out=torch.full_like(args["q"], 7.0))
    for b in range(B):
        rows = slice(cu[b], cu[b + 1])
        if b in long:
            assert bool((out[rows] == 7.0).all()), b
        else:
            assert bool(((out[rows].double() - wanted[rows]).abs() <= bound[rows]).all()), b


@pytest.mark.parametrize("nodes,heads,kv_heads,dim,columns,want", [
    (5, 4, 2, 64, 8, (16, 1, False)), (5, 4, 2, 64, 200, (16, 9, False)), (9, 8, 2, 128, 400, (32, 10, False)),
    (40, 8, 2, 128, 400, (128, 10, False)), (40, 4, 2, 192, 900, (128, 23, False)),
])
def test_contexts_past_the_table(cuda, nodes, heads, kv_heads, dim, columns, want):
    """Positions behind the table's last are not seen, nodes' own among them; a negative context is none."""
    cap, page = columns * 16, 16
    contexts = [cap - 2, cap + 100, 2 ** 31 - 1, -3, cap]
    g = torch.Generator().manual_seed(columns)
    B, T = len(contexts), len(contexts) * nodes
    kc, vc = R.make_cache(cuda, columns, kv_heads, page, dim, "bf16", seed=1)
    trees = [R.sees(R.random_tree(nodes, g)) for _ in contexts]
    table = torch.stack([torch.randperm(columns, generator=g) for _ in contexts]).int()
    q = torch.randn((T, heads, dim), generator=g).bfloat16().to(cuda)
    args = dict(q=q, k_cache=kc, v_cache=vc, block_table=table.to(cuda), context_lens=torch.tensor(contexts).int().to(cuda),
                cu_nodes=torch.arange(B + 1, device=cuda).int() * nodes, max_nodes=nodes, visible=R.pack(torch.cat(trees), nodes).to(cuda))
    assert plan(args)[:2] == want[:2]
    out = ops.tree_attention(**args).double()
    for b, c in enumerate(contexts):
        c = min(max(c, 0), cap)
        see = torch.ones((nodes, min(c + nodes, cap)), dtype=torch.bool)
        see[:, c:] = trees[b][:, :see.shape[1] - c]
        pos = torch.arange(see.shape[1])
        pages, off, see = table[b][pos // page].long().to(cuda), (pos % page).to(cuda), see.to(cuda).unsqueeze(1)
        for h in range(kv_heads):
            k, v = kc[pages, h, off].double(), vc[pages, h, :, off].double()
            mine = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
            x = q[b * nodes:(b + 1) * nodes, mine].double()
            s = torch.where(see, (x @ k.T) * dim ** -0.5, -float("inf"))
            w = torch.softmax(s, -1)
            score = ((x.abs() @ k.abs().T) * dim ** -0.5 * (dim + 4) * 2.0 ** -24).amax(-1, keepdim=True)
            o = w @ v
            bound = 2.0 ** -8 * o.abs() + (w @ v.abs()) * (2.0 ** -8 + 2.5 * score + see.shape[2] * 2.0 ** -24 / 4 + 2.0 ** -19)
            got = out[b * nodes:(b + 1) * nodes, mine]
            assert bool(((got - o).abs() <= bound).all()), (contexts[b], float(((got - o).abs() / bound).max()))


def test_a_cache_without_heads_is_refused(cuda):
    args, _, _ = arguments(cuda, [20], [4], 4, 2, 64, 16, "bf16")
    none = dict(k_cache=args["k_cache"][:, :0], v_cache=args["v_cache"][:, :0])
    for heads in (0, 4):
        with pytest.raises(ValueError):
            ops.tree_attention(**{**args, **none, "q": args["q"][:, :heads]})
