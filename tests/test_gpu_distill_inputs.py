"""What the distillation entry points make of inputs that they cannot take as they are."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_distill import make
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
