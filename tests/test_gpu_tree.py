"""Attention of drafted trees over a paged cache and the walk down a tree, against 64-bit and plain forms."""
from __future__ import annotations

import pytest
import torch

from tests import tree_ref as R
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def setup(dev, contexts, nodes, heads, kv_heads, dim, page, dtype, seed=0, chain=False, spare=2):
    """Arguments of a call and the trees' visibility; what lies behind a request's last node is NaN."""
    g = torch.Generator().manual_seed(seed)
    B, cu = len(contexts), [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    need = [(c + n + page - 1) // page for c, n in zip(contexts, nodes)]
    pages, width = sum(need) + spare, max(max(need), 1)
    kc, vc = R.make_cache(dev, pages, kv_heads, page, dim, dtype, seed=seed + 1)
    order, at = torch.randperm(pages, generator=g), 0
    table = torch.full((B, width), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        end = contexts[b] + nodes[b]
        if end % page:
            kc[table[b, n - 1], :, end % page:] = float("nan")
            vc[table[b, n - 1], :, :, end % page:] = float("nan")
    q = torch.randn((cu[-1], heads, dim), generator=g).to(R.DTYPES[dtype]).to(dev)
    most = max(nodes)
    see = None if chain else [R.sees(R.random_tree(n, g)) if n else torch.zeros((0, 0), dtype=torch.bool) for n in nodes]
    words = None
    if not chain:
        rows = [torch.nn.functional.pad(s, (0, most - s.shape[1])) for s in see]
        words = R.pack(torch.cat(rows), most).to(dev)
    args = dict(q=q, k_cache=kc, v_cache=vc, block_table=table.to(dev), context_lens=torch.tensor(contexts).int().to(dev),
                cu_nodes=torch.tensor(cu).int().to(dev), max_nodes=most, visible=words)
    return args, see, cu


def check(args, see, cu, contexts, out=None, scale=None):
    out = ops.tree_attention(**args, **({} if scale is None else {"scale": scale})) if out is None else out
    want, bound = R.attention(args["q"], args["k_cache"], args["v_cache"], args["block_table"], contexts, cu, see, scale)
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    return out


# rows (nodes times query heads of a key head) for every tile of both kinds, contexts that end inside steps and pages
@pytest.mark.parametrize("contexts,nodes,heads,kv_heads,dim,page,dtype,chain", [
    ([0], [1], 1, 1, 64, 8, "bf16", True), ([1], [1], 4, 4, 128, 16, "f16", True), ([31], [2], 8, 1, 64, 8, "bf16", False),
    ([32], [5], 8, 2, 128, 16, "bf16", False), ([100, 3, 0], [7, 1, 12], 12, 3, 128, 32, "f16", False),
    ([517, 1000], [33, 20], 4, 2, 96, 16, "bf16", False), ([255, 256, 257, 700], [64, 1, 40, 3], 7, 1, 64, 64, "f16", False),
    ([90], [256], 2, 1, 64, 16, "bf16", False), ([64, 65], [100, 70], 8, 2, 256, 256, "bf16", False),
    ([300], [16], 16, 1, 256, 16, "f16", False), ([40], [3], 15, 5, 192, 8, "bf16", False), ([2000], [9], 3, 3, 192, 32, "f16", True),
    ([5000, 20], [4, 4], 8, 8, 128, 16, "bf16", True), ([3333], [60], 16, 2, 128, 128, "f16", False), ([77], [17], 2, 2, 96, 8, "f16", False),
    ([1500] * 40, [6] * 40, 8, 4, 64, 16, "bf16", False),
])
def test_trees(cuda, contexts, nodes, heads, kv_heads, dim, page, dtype, chain):
    args, see, cu = setup(cuda, contexts, nodes, heads, kv_heads, dim, page, dtype, seed=sum(contexts) + heads, chain=chain)
    check(args, see, cu, contexts)


def test_long_context_and_scale(cuda):
    args, see, cu = setup(cuda, [40000, 9], [5, 3], 8, 2, 128, 16, "bf16", seed=3)
    check(args, see, cu, [40000, 9], scale=0.5)   # (peaked: scores of some 5 times the default's spread)


def test_reference_rises_many_times(cuda):
    """Keys that grow along the context: every step's scores exceed the ones before."""
    args, see, cu = setup(cuda, [600], [4], 4, 1, 64, 16, "bf16", seed=5, chain=True)
    n = 604
    k = args["k_cache"]
    for pos in range(n):
        page, off = int(args["block_table"][0, pos // 16]), pos % 16
        k[page, 0, off] = args["q"][0, 0] * (pos / n) * 4
    check(args, see, cu, [600])


def test_rows_that_see_nothing(cuda):
    args, see, cu = setup(cuda, [0, 0, 50], [4, 3, 5], 4, 2, 64, 16, "f16", seed=6)
    see[0][2] = False
    see[1][:] = False
    see[2][1] = False
    args["visible"] = R.pack(torch.cat([torch.nn.functional.pad(s, (0, 5 - s.shape[1])) for s in see]), 5).to(cuda)
    out = check(args, see, cu, [0, 0, 50])
    assert not bool(out[2].any()) and not bool(out[4:7].any())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_hidden_nodes_may_hold_anything(cuda, bad):
    """Node 2's key and value are not numbers: nodes that do not see it do not notice, those that do are not numbers."""
    args, see, cu = setup(cuda, [37, 5], [6, 6], 4, 2, 128, 16, "bf16", seed=7)
    for s in see:
        s[:, 2] = False
        s[2, 2] = s[5, 2] = True
    args["visible"] = R.pack(torch.cat(see), 6).to(cuda)
    want, bound = R.attention(args["q"], args["k_cache"], args["v_cache"], args["block_table"], [37, 5], cu, see)
    for b, c in enumerate((37, 5)):
        page, off = int(args["block_table"][b, (c + 2) // 16]), (c + 2) % 16
        args["v_cache"][page, :, 8:40, off] = bad
        if b:
            args["k_cache"][page, :, off] = float("nan")
    out = ops.tree_attention(**args)
    rows = [0, 1, 3, 4, 6, 7, 9, 10]
    assert bool(((out[rows].double() - want[rows]).abs() <= bound[rows]).all())
    for r in (2, 5):
        o = out[r].double()
        assert bool(torch.isnan(o[:, 8:40]).all() if bad != bad else (o[:, 8:40] == bad).all())
        rest = torch.cat([o[:, :8], o[:, 40:]], 1) - torch.cat([want[r, :, :8], want[r, :, 40:]], 1)
        assert bool((rest.abs() <= torch.cat([bound[r, :, :8], bound[r, :, 40:]], 1)).all())
    assert bool(torch.isnan(out[[8, 11]]).all())


def test_nodes_past_the_last_are_not_seen(cuda):
    """Bits past a request's nodes, and a table that is wider than the request."""
    args, see, cu = setup(cuda, [20, 40], [3, 9], 4, 2, 64, 16, "bf16", seed=8)
    args["visible"][:3] |= torch.tensor(~7, device=cuda, dtype=torch.int32)
    args["block_table"] = torch.cat([args["block_table"], torch.full((2, 9), 10 ** 6, device=cuda).int()], 1)
    check(args, see, cu, [20, 40])


def test_pages_that_do_not_exist_are_not_seen(cuda):
    args, see, cu = setup(cuda, [70, 64], [5, 2], 4, 2, 64, 16, "f16", seed=9)
    for b, at, page in ((0, 1, -1), (0, 2, 10 ** 9), (1, 0, -5)):
        args["block_table"][b, at] = page
    out = ops.tree_attention(**args)
    for b in (0, 1):
        n, c = cu[b + 1] - cu[b], [70, 64][b]
        pos = torch.arange(c + n)
        gone = (pos >= 16) & (pos < 48) if b == 0 else pos < 16
        pos = pos[~gone]
        pages, off = args["block_table"][b].cpu()[pos // 16].long().to(cuda), (pos % 16).to(cuda)
        mask = torch.ones((n, c + n), dtype=torch.bool)
        mask[:, c:] = see[b]
        mask = mask[:, ~gone].to(cuda).unsqueeze(1)
        for h in range(2):
            k, v = args["k_cache"][pages, h, off].double(), args["v_cache"][pages, h, :, off].double()
            s = args["q"][cu[b]:cu[b + 1], 2 * h:2 * h + 2].double() @ k.T * 0.125
            want = torch.softmax(torch.where(mask, s, -float("inf")), -1) @ v
            got = out[cu[b]:cu[b + 1], 2 * h:2 * h + 2].double()
            assert bool(((got - want).abs() <= 2.0 ** -10 * 4).all())   # (two roundings of 2^-11 of values of at most 4)


def test_bounds_that_do_not_fit_leave_their_rows(cuda):
    args, see, cu = setup(cuda, [20, 30, 10], [4, 4, 4], 4, 2, 64, 16, "bf16", seed=10)
    want = ops.tree_attention(**args)
    for bounds, kept in (([0, 4, 4, 12], [(0, 4)]), ([0, 4, 2, 6], [(0, 2)]), ([-1, 4, 8, 12], [(4, 8), (8, 12)]),
                         ([0, 4, 8, 13], [(0, 4), (4, 8)]), ([0, 4, 8, 2 ** 31 - 1], [(0, 4), (4, 8)])):
        out = torch.full_like(want, 7.0)
        got = ops.tree_attention(**{**args, "cu_nodes": torch.tensor(bounds, device=cuda)}, out=out)
        assert got is out
        if bounds[1:3] == [4, 4]:
            assert torch.equal(out[:4], want[:4]) and bool((out[4:] == 7.0).all())   # (8 nodes: more than max_nodes)
            continue
        for lo, hi in kept:
            assert torch.equal(out[lo:hi], want[lo:hi]), bounds


def test_rows_of_no_request_stay(cuda):
    args, see, cu = setup(cuda, [20, 30], [4, 4], 4, 2, 64, 16, "bf16", seed=11)
    want = ops.tree_attention(**args)
    more = {**args, "q": torch.cat([args["q"], args["q"][:3]]), "visible": torch.cat([args["visible"], args["visible"][:3]])}
    out = torch.full((11, 4, 64), 5.0, dtype=torch.bfloat16, device=cuda)
    ops.tree_attention(**more, out=out)
    assert torch.equal(out[:8], want) and bool((out[8:] == 5.0).all())


def test_strides(cuda):
    """Queries inside a projection's output, outputs in a wider buffer, a table and words with longer rows."""
    args, see, cu = setup(cuda, [45, 200], [6, 3], 6, 2, 64, 16, "f16", seed=12)
    want = ops.tree_attention(**args)
    wide = torch.zeros((9, 10, 64 + 3), dtype=torch.float16, device=cuda)     # (rows that start unaligned)
    wide[:, 2:8, 1:65] = args["q"]
    out = torch.zeros((9, 7, 64 + 1), dtype=torch.float16, device=cuda)
    table = torch.zeros((2, 30), device=cuda).int()
    table[:, :args["block_table"].shape[1]] = args["block_table"]
    words = torch.zeros((9, 4), device=cuda).int()
    words[:, :1] = args["visible"]
    got = ops.tree_attention(**{**args, "q": wide[:, 2:8, 1:65], "block_table": table[:, :args["block_table"].shape[1]],
                                "visible": words}, out=out[:, 1:, 1:])
    assert torch.equal(got, want) and not bool(out[:, 0].any()) and not bool(out[:, :, 0].any())


def test_the_same_result_in_any_batch(cuda):
    """Repeated calls, and a side stream: the same bits."""
    args, see, cu = setup(cuda, [900, 1700, 5], [12, 30, 2], 8, 2, 128, 16, "bf16", seed=13)
    want = ops.tree_attention(**args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        outs = [ops.tree_attention(**args) for _ in range(5)]
    outs += [ops.tree_attention(**args) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_refusals(cuda):
    args, see, cu = setup(cuda, [20], [4], 4, 2, 64, 16, "bf16")
    q = args["q"]
    for change in (dict(q=q[:, :3]), dict(q=q[0]), dict(q=q[..., :32]), dict(max_nodes=0), dict(max_nodes=257), dict(cu_nodes=args["cu_nodes"][:1]),
                   dict(context_lens=args["context_lens"].repeat(2)), dict(visible=args["visible"].long()), dict(visible=args["visible"][:2]),
                   dict(max_nodes=33), dict(out=q), dict(out=q[:2]), dict(block_table=args["block_table"].cpu()),
                   dict(q=q.clone().requires_grad_()), dict(visible=args["visible"].cpu())):
        with pytest.raises(ValueError):
            ops.tree_attention(**{**args, **change})
    with pytest.raises(TypeError):
        ops.tree_attention(**{**args, "q": q.half()})
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ops._lib.VwsError):
            ops.tree_attention(**args, scale=scale)


# ---- the walk -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("sizes,width,vocab", [([1], 1, 3), ([5, 0, 12], 4, 3), ([64] * 9, 64, 4), ([256, 1, 200], 256, 2), ([30] * 300, 6, 2)])
def test_walk(cuda, sizes, width, vocab):
    g = torch.Generator().manual_seed(len(sizes) + width)
    cu, parents = [0], []
    for n in sizes:
        cu.append(cu[-1] + n)
        parents += R.random_tree(n, g) if n else []
    T = cu[-1]
    tokens, sampled = (torch.randint(vocab, (T,), generator=g).tolist() for _ in range(2))
    out, path, count = R.walk(sampled, tokens, parents, cu, width)
    dev = lambda x: torch.tensor(x, device=cuda)  # noqa: E731
    r = ops.accept_tree(dev(sampled), dev(tokens).int(), dev(parents), dev(cu), width)
    assert r.tokens.tolist() == out and r.path.tolist() == path and r.num_accepted.tolist() == count


def test_walk_of_odd_parents(cuda):
    """Parents at or behind their node lead nowhere, other roots are not reached, bounds that do not fit have no walk."""
    dev = lambda x: torch.tensor(x, device=cuda).int()  # noqa: E731
    r = ops.accept_tree(dev([7] * 5), dev([7] * 5), dev([-1, 1, 3, -1, 0]), dev([0, 5]), 4)
    assert r.path.tolist() == [[0, 4, -1, -1]] and r.tokens.tolist() == [[7, 7, -1, -1]]
    for cu, want in (([0, 3, 2, 5], [2, -1, 2]), ([0, 6, 5, 5], [-1, -1, -1]), ([-1, 2, 5, 2 ** 31 - 1], [-1, 2, -1])):
        r = ops.accept_tree(dev([7] * 5), dev([7] * 5), dev([-1, 0, 1, 2, 3]) if want == 0 else dev([-1, 0, 1, 0, 1]), dev(cu), 4)
        got = r.num_accepted.tolist()
        assert [g < 0 for g in got] == [w < 0 for w in want], (cu, got)
        assert all(t == [-1] * 4 for t, g in zip(r.path.tolist(), got) if g < 0)
    with pytest.raises(ValueError):
        ops.accept_tree(dev([1]), dev([1]), dev([-1]), dev([0, 1]), 0)
    with pytest.raises(ValueError):
        ops.accept_tree(dev([1]), dev([1, 2]), dev([-1]), dev([0, 1]), 2)
    with pytest.raises(ValueError):
        ops.accept_tree(dev([1]), dev([1]).float(), dev([-1]), dev([0, 1]), 2)
