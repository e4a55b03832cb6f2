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
