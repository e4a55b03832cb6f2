"""What the paged cache's, drafted trees' and log-probabilities' operators do with derivatives that they have none of, and gradients
of rows that are not numbers."""
from __future__ import annotations

import pytest
import torch

from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


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
