"""What the paged cache's, drafted trees' and log-probabilities' operators do with derivatives that they have none of, and gradients
of rows that are not numbers."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from tests import tree_ref as R
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def operands(dev):
    """Arguments of a step of one request of three tokens, whose own keys lie at positions 5 to 7."""
    kc, vc = R.make_cache(dev, 2, 2, 16, 64, "bf16")
    q, k, v = (torch.randn((3, h, 64), device=dev).bfloat16() for h in (4, 2, 2))
    at = lambda *x: torch.tensor(x, device=dev).int()  # noqa: E731
    append = dict(k=k, v=v, k_cache=kc, v_cache=vc, slots=at(5, 6, 7), q=q, positions=at(5, 6, 7), inv_freq=torch.ones(32, device=dev))
    tree = dict(q=q, k_cache=kc, v_cache=vc, block_table=at(0, 1).view(1, 2), context_lens=at(5), cu_nodes=at(0, 3), max_nodes=3)
    return append, tree


@pytest.mark.parametrize("grad", [True, False])
def test_forward_derivatives_are_refused(cuda, grad):
    """Tangents would be lost: the calls raise, with gradients on and off, and take tensors without one as before."""
    append, tree = operands(cuda)
    x, ids = torch.randn((3, 50), device=cuda), torch.tensor([1, 2, 3], device=cuda)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for leaf in (x, x.clone().requires_grad_()):
            with pytest.raises((ValueError, RuntimeError)):
                ops.token_logprobs(dual(leaf), ids)
        for name in ("q", "k", "v", "k_cache", "v_cache", "inv_freq"):
            with pytest.raises(ValueError):
                ops.append_kv(**{**append, name: dual(append[name])})
        for name in ("q", "k_cache", "v_cache"):
            with pytest.raises(ValueError):
                ops.tree_attention(**{**tree, name: dual(tree[name])})
        for name in ("k_cache", "v_cache"):
            with pytest.raises(ValueError):
                ops.compact_kv(**{**{n: tree[n] for n in ("k_cache", "v_cache", "block_table", "context_lens")}, name: dual(tree[name])},
                               path=torch.zeros((1, 1), device=cuda).int())
        for call, args in ((ops.append_kv, append), (ops.tree_attention, tree)):
            out = torch.empty_like(args["q"])
            with pytest.raises(ValueError):
                call(**args, out=dual(out))
            assert call(**args, out=out) is out
        assert ops.token_logprobs(x, ids).logprobs.shape == (3,)


def test_frequencies_that_require_a_gradient_are_refused(cuda):
    append, _ = operands(cuda)
    f = append["inv_freq"].clone().requires_grad_()
    with pytest.raises(ValueError):
        ops.append_kv(**{**append, "inv_freq": f})
    want = ops.append_kv(**append)
    with torch.no_grad():
        assert torch.equal(ops.append_kv(**{**append, "inv_freq": f}), want)


@pytest.mark.parametrize("V", [100, 30000])
@pytest.mark.parametrize("gl,gh", [(0.0, 0.0), (1.5, 0.0), (0.0, -0.5), (1.0, 2.0), (0.0, None), (None, 0.0), (None, 1.0)])
def test_gradients_of_rows_that_are_not_numbers(cuda, V, gl, gh):
    """A row with a NaN or +inf, or without a logit above -inf, has a gradient of NaN whatever its upstream; padding rows and rows of
    numbers with an upstream of 0 have 0."""
    x = torch.randn((6, V), device=cuda, generator=torch.Generator(device=cuda).manual_seed(V))
    x[0, 17], x[1, V - 1], x[2] = float("nan"), float("inf"), -float("inf")
    x[3] = float("nan")
    ids = torch.tensor([3, 4, 5, -1, 6, V], device=cuda)
    x.requires_grad_()
    r = ops.token_logprobs(x, ids, entropy=True)
    outs = [t for t, g in ((r.logprobs, gl), (r.entropy, gh)) if g is not None]
    got, = torch.autograd.grad(outs, [x], [torch.full_like(r.logprobs, g) for g in (gl, gh) if g is not None])
    assert bool(torch.isnan(got[:3]).all()) and not bool(got[[3, 5]].any())
    assert bool(torch.isfinite(got[4]).all()) and bool(got[4].any()) == bool(gl or gh)
