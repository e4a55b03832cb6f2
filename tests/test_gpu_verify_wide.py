"""Top-p alone on long rows of equal logits: more groups at the list's bound than the list is read from,
so every row leaves the list for the masses, and the index alone decides its cut."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_verify import check, make
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [33000, 70001])
@pytest.mark.parametrize("dtype,probs", [("bf16", None), ("f16", "bf16"), ("f32", None)])
def test_long_rows_of_equal_logits(cuda, V, dtype, probs):
    t = make(cuda, [1, 2, 0, 1], V, dtype, probs, seed=V)
    t["logits"][:] = 2.5
    check(t, 2, T=1.0, p=0.9, max_near=0.75)
    check(t, 2, T=0.7, p=0.25, max_near=0.75)


def test_many_long_rows_of_equal_logits(cuda):
    """More of them than the launch sets aside for the masses' own kernel."""
    t = make(cuda, [1] * 170, 33001, "bf16", None, seed=1, spikes=1)
    t["logits"][:] = -1.0
    r = ops.verify_drafts(max_drafts=1, temperature=1.0, top_p=0.6, **t)
    few = dict(logits=t["logits"][:20], draft_tokens=t["draft_tokens"][:10], cu_drafts=t["cu_drafts"][:11],
               draft_probs=None, accept_uniforms=t["accept_uniforms"][:10], uniforms=t["uniforms"][:10])
    check(few, 1, T=1.0, p=0.6, max_near=0.75)
    one = ops.verify_drafts(max_drafts=1, temperature=1.0, top_p=0.6, **few)
    assert torch.equal(one.tokens, r.tokens[:10]) and torch.equal(one.num_accepted, r.num_accepted[:10])
    # of V equal tokens floor(0.4 V) with the lowest indices are gone
    assert int(r.tokens[:, 0][r.num_accepted == 0].min()) >= int(0.4 * 33001)
    assert torch.allclose(r.logprobs[:, 0].exp() * (33001 - int(0.4 * 33001)), torch.ones_like(r.logprobs[:, 0]), rtol=1e-4)
