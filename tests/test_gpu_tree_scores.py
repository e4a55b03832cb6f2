"""Attention of drafted trees where scores differ by much or lie far from zero, against 64-bit forms."""
from __future__ import annotations

import pytest
import torch

from tests import tree_ref as R
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def shared(dev, B, nodes, heads, kv_heads, dim, page, n, dtype):
    """Arguments of B requests of `nodes` chained tokens over the same pages of n keys, the nodes' own among them; zeros."""
    kc = torch.zeros((n // page, kv_heads, page, dim), dtype=R.DTYPES[dtype], device=dev)
    vc = torch.zeros((n // page, kv_heads, dim, page), dtype=R.DTYPES[dtype], device=dev)
    table = torch.arange(n // page, dtype=torch.int32, device=dev).expand(B, -1)
    return dict(q=torch.zeros((B * nodes, heads, dim), dtype=R.DTYPES[dtype], device=dev), k_cache=kc, v_cache=vc, block_table=table,
                context_lens=torch.full((B,), n - nodes, dtype=torch.int32, device=dev),
                cu_nodes=torch.arange(B + 1, dtype=torch.int32, device=dev) * nodes, max_nodes=nodes)


def parts(args):
    """Whether the call divides its requests' keys (it needs room for the parts then)."""
    (_, Hk, page, D), L = args["k_cache"].shape, ops._lib.lib()
    B, W = args["block_table"].shape
    return (L.vws_tree_attention_workspace_size(B, args["max_nodes"], args["q"].shape[1], Hk, D, page, W)
            > L.vws_sample_workspace_size(1, 1, 0))


# rows of 16, 32 and 128 a workgroup, of all widths of shared tiles
@pytest.mark.parametrize("B,nodes,heads,dim", [(600, 1, 1, 64), (600, 6, 4, 96), (300, 64, 2, 128), (300, 10, 4, 64), (300, 40, 1, 256),
                                               (300, 1, 2, 192)])
@pytest.mark.parametrize("gap", [14.0, 16.5, 17.0, 20.0])
def test_a_first_token_that_takes_the_weight(cuda, B, nodes, heads, dim, gap):
    """f16: the first key stands e^gap above all others and its value is 0, so that the result is what little weight the others
    have, in one undivided pass."""
    page, n = 64, 131072
    args = shared(cuda, B, nodes, heads, 1, dim, page, n, "f16")
    assert not parts(args)
    g = torch.Generator(device=cuda).manual_seed(int(gap))
    args["q"][:] = 1.0
    args["k_cache"][:] = torch.randn(args["k_cache"].shape, generator=g, device=cuda) * 0.05
    args["k_cache"][0, 0, 0] = 2.0
    args["v_cache"][:] = 0.5 + torch.rand(args["v_cache"].shape, generator=g, device=cuda)
    args["v_cache"][0, 0, :, 0] = 0.0
    scale = gap / (2.0 * dim)
    out = ops.tree_attention(**args, scale=scale).double()
    k, v = args["k_cache"][:, 0].reshape(n, dim).double(), args["v_cache"][:, 0].transpose(1, 2).reshape(n, dim).double()
    s = k.sum(1) * scale
    e = torch.exp(s - s[0])
    near, total = (e[:, None] * v).cumsum(0), e.cumsum(0)
    # A weight is off by 2^-11 of itself, or below 2^-14 by 2^-25, where the largest is at least 2^11; its score by (dim + 4)
    # 2^-24 of the products' sizes; sums of 32 bits and the result's rounding as in tree_ref.attention.
    off = (k.abs().sum(1) * scale * (dim + 4) * 2.0 ** -24).max()
    for node in {0, nodes // 2, nodes - 1}:
        at = n - nodes + node
        want = near[at] / total[at]
        bound = 2.0 ** -11 * want + want * (2.0 ** -11 + 2.5 * off + n * 2.0 ** -24 / 4 + 2.0 ** -19) + 2.0 ** -36 * v[:at + 1].sum(0)
        got = out[node::nodes]
        assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("B,nodes,heads,dim,n", [(1, 1, 1, 64, 128), (1, 5, 4, 128, 4096), (300, 64, 2, 128, 512), (300, 40, 1, 256, 512),
                                                 (3, 9, 2, 192, 8192)])
@pytest.mark.parametrize("size,dtype", [(300.0, "f16"), (3000.0, "f16"), (5000.0, "f16"), (20000.0, "f16"), (60000.0, "f16"), (3e5, "bf16"),
                                        (1e8, "bf16"), (1e15, "bf16")])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_far_from_zero(cuda, B, nodes, heads, dim, n, size, dtype, sign):
    """Equal scores of 1e6 to 1e31, where neighbouring 32-bit numbers lie up to many powers of two apart, have equal weights; keys
    with scores of half of that have none, or all of it where those are negative."""
    args = shared(cuda, B, nodes, heads, 1, dim, 16, n, dtype)
    g = torch.Generator(device=cuda).manual_seed(n + dim)
    args["q"][:] = size
    args["v_cache"][:] = torch.randn(args["v_cache"].shape, generator=g, device=cuda)
    half = torch.rand((n // 16, 1, 16, 1), generator=g, device=cuda) < 0.5
    half[0, 0, 0], half[0, 0, 1] = True, False
    args["k_cache"][:] = torch.where(half, sign * size / 2, sign * size)
    out = ops.tree_attention(**args).double()
    v = args["v_cache"][:, 0].transpose(1, 2).reshape(n, dim).double()
    most = (half.flatten() == (sign < 0)).unsqueeze(1)
    for node in {0, nodes // 2, nodes - 1}:
        end = n - nodes + node + 1
        w = most[:end].double() / most[:end].sum()
        want, near = (w * v[:end]).sum(0), (w * v[:end].abs()).sum(0)
        eps = R.half_step(R.DTYPES[dtype])
        bound = eps * want.abs() + near * (eps + n * 2.0 ** -24 / 4 + 2.0 ** -19)   # (equal weights, rounded; sums; the result)
        got = out[node::nodes]
        assert bool(((got - want).abs() <= bound).all()), (node, got[0, 0, :3], want[:3])


@pytest.mark.parametrize("B,nodes,heads,dim,n", [(1, 1, 1, 64, 512), (1, 5, 4, 128, 4096), (300, 64, 2, 128, 512), (300, 40, 1, 256, 512),
                                                 (3, 9, 2, 192, 8192)])
@pytest.mark.parametrize("size,dtype", [(8000.0, "f16"), (60000.0, "f16"), (3e4, "bf16"), (1e9, "bf16"), (1e15, "bf16")])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("at", [0.1, 0.5, 1.0])
def test_scores_far_from_zero_beside_others(cuda, B, nodes, heads, dim, n, size, dtype, sign, at):
    """Some keys' scores are far above or below the others', which are zero, before and behind them: the larger ones take all weight."""
    args = shared(cuda, B, nodes, heads, 1, dim, 16, n, dtype)
    g = torch.Generator(device=cuda).manual_seed(n + dim)
    args["q"][:] = size
    args["v_cache"][:] = torch.randn(args["v_cache"].shape, generator=g, device=cuda)
    end = n - nodes + 1 if at == 1.0 else int(at * n)      # (the last ones are what the first node sees last)
    far = torch.zeros(n, dtype=torch.bool, device=cuda)
    far[end - 7:end] = True
    far[40:60] |= at == 0.5
    args["k_cache"].view(n // 16, 16, dim)[far.view(n // 16, 16)] = sign * size
    out = ops.tree_attention(**args).double()
    v = args["v_cache"][:, 0].transpose(1, 2).reshape(n, dim).double()
    most = (far == (sign > 0)).unsqueeze(1)
    for node in {0, nodes // 2, nodes - 1}:
        end = n - nodes + node + 1
        w = most[:end].double() / most[:end].sum()
        want, near = (w * v[:end]).sum(0), (w * v[:end].abs()).sum(0)
        eps = R.half_step(R.DTYPES[dtype])
        bound = eps * want.abs() + near * (eps + n * 2.0 ** -24 / 4 + 2.0 ** -19)
        got = out[node::nodes]
        assert bool(((got - want).abs() <= bound).all()), (node, got[0, 0, :3], want[:3])


@pytest.mark.parametrize("B,nodes,heads,dim,columns", [(1, 3, 4, 64, 200), (1, 40, 4, 128, 2400), (1, 20, 2, 256, 400), (1, 3, 4, 64, 8),
                                                       (600, 1, 1, 128, 24)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_no_numbers_count_whatever_their_weight(cuda, B, nodes, heads, dim, columns, bad):
    """A seen value that is not finite makes the result so, though its key stands 300 nats below the others, with the keys divided
    or not."""
    n, at = columns * 16, columns * 5
    args = shared(cuda, B, nodes, heads, 1, dim, 16, n, "bf16")
    assert parts(args) == (columns >= 200)
    args["q"][:] = 1.0
    args["k_cache"][at // 16, 0, at % 16] = 300.0 / dim ** 0.5
    args["v_cache"][:] = 1.0
    args["v_cache"][0, 0, 7, 5] = bad
    out = ops.tree_attention(**args)
    fine = torch.isfinite(out)
    assert not bool(fine[..., 7].any()) and bool(fine[..., :7].all()) and bool(fine[..., 8:].all())
