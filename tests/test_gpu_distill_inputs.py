"""What the distillation entry points make of inputs that they cannot take as they are."""
from __future__ import annotations

import pytest
import torch

from tests import speculative_ref as R
from tests.test_gpu_distill import TOL, check, close, make
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def test_inputs_that_would_silently_get_no_gradient_are_refused(cuda):
    x, ids, lp = make(cuda, 4, 900, 6, "f32", seed=1)
    w = torch.ones(4, device=cuda)
    x.requires_grad_(True)
    for bad in (dict(teacher_logprobs=lp.clone().requires_grad_(True)), dict(row_weight=w.clone().requires_grad_(True))):
        args = {**dict(logits=x, teacher_ids=ids, teacher_logprobs=lp, row_weight=w), **bad}
        with pytest.raises(ValueError, match=next(iter(bad))):
            ops.distill_loss(**args)
        with torch.no_grad():               # (nothing is lost here)
            assert torch.equal(ops.distill_loss(**args), ops.distill_loss(x, ids, lp, w))
    loss = ops.distill_loss(x, ids, lp.clone().requires_grad_(True).detach(), w)
    loss.sum().backward()
    assert x.grad is not None


FAR = [-2 ** 63, 2 ** 63 - 1, 2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31 + 3, 2 ** 40]


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_ids_past_32_bits_are_padding(cuda, tail):
    """As any id outside the vocabulary, whatever their lower halves are."""
    x, ids, lp = make(cuda, 5, 900, 12, "f32", seed=2)
    wide, narrow = ids.long(), ids.clone()
    wide[:, 3:9], narrow[:, 3:9] = torch.tensor(FAR, device=cuda), -1
    want, want_grad = ops.distill_loss_and_grad(x, narrow, lp, tail=tail)
    got, grad = ops.distill_loss_and_grad(x, wide, lp, tail=tail)
    assert torch.equal(got, want) and torch.equal(grad, want_grad)
    assert torch.equal(ops.distill_loss(x, wide, lp, tail=tail), ops.distill_loss(x, narrow, lp, tail=tail))


def test_drafts_and_bounds_past_32_bits(cuda):
    """Drafts there are refused, bounds there do not fit."""
    V, n = 300, len(FAR)
    x = torch.zeros((2 * n, V), device=cuda)
    x[:, [0, 3, 5]] = 20.0                                   # the lower halves' tokens are likely
    q = torch.full((n, V), 1e-6, device=cuda)
    cu = torch.arange(n + 1)
    r = ops.verify_drafts(x, torch.tensor(FAR), cu, 1, draft_probs=q, temperature=1.0, rng_key=3)
    assert not r.num_accepted.any()
    ok = ops.verify_drafts(x, torch.tensor([0, 3, 5, 5, 3, 0]), cu, 1, draft_probs=q, temperature=1.0, rng_key=3)
    assert bool((ok.num_accepted == 1).all())
    for far in FAR[:1] + FAR[2:4]:
        bounds = cu.clone()
        bounds[2] = far
        r = ops.verify_drafts(x, torch.zeros(n, dtype=torch.int32), bounds, 1, temperature=1.0, rng_key=3)
        assert r.num_accepted[1:3].tolist() == [-1, -1]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_teacher_whose_probabilities_exceed_one(cuda, dtype):
    """Bucket: no rest is left, and the gradient is the stated loss's, w / T (q sum p - p)."""
    x, ids, lp = make(cuda, 6, 3001, 20, dtype, seed=3)
    lp = lp + torch.linspace(0.5, 1.5, 6, device=cuda).unsqueeze(1)
    p = lp.double().exp()
    assert bool((p.sum(1) > 1.05).all())
    check(x, ids, lp, tail="bucket")
    _, grad = ops.distill_loss_and_grad(x, ids, lp, tail="bucket")
    want = torch.softmax(x.double(), 1) * p.sum(1, keepdim=True)
    want.scatter_add_(1, ids.long(), -p)
    assert ((grad.double() - want).abs() <= 4 * TOL + 2.0 ** -8 * want.abs() * (dtype == "bf16")).all()


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_entries_that_the_student_masks_by_the_types_lowest_value(cuda, dtype, tail):
    """Their loss is as large, and finite while it fits 32 bits; the gradient is -p."""
    x, ids, lp = make(cuda, 4, 3001, 60, dtype, seed=4)
    lp = lp - 0.7
    lp[0] = -5.0                                             # many alike: unnormalised they add up to 60
    x.scatter_(1, ids[:, ::2].long(), torch.finfo(x.dtype).min)
    g = torch.ones(4, device=cuda)
    z = x.double()
    leaf = (z - z.amax(1, keepdim=True)).requires_grad_(True)
    want = R.distill(leaf, ids, lp, None, 1.0, tail)
    (want_grad,) = torch.autograd.grad(want, leaf, g.double())
    assert dtype == "f16" or (want > 1e36).all()
    loss, grad = ops.distill_loss_and_grad(x, ids, lp, tail=tail)
    close(loss, grad, want.detach(), want_grad, None, g, 1.0, x.dtype)
