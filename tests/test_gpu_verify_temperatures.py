"""Draft verification at temperatures from the least that is not greedy to infinity: without drafts it is the
sampler.  At T = inf every finite logit scales to 0, and one of -inf to no number, which is never kept."""
from __future__ import annotations

import pytest
import torch

from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1e-5, 2e-5, 1e-3, 0.02, 50.0, 1e10, 1e38, float("inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [dict(), dict(top_p=0.9), dict(top_k=9), dict(top_k=400, top_p=0.8), dict(min_p=0.05)])
def test_without_drafts_it_is_the_sampler(cuda, T, dtype, kw):
    B, V = 24, 20011
    g = torch.Generator().manual_seed(1)
    x = (torch.randn((B, V), generator=g) * 3).to(dtype).to(cuda)
    for b in range(3, 12):
        x[b, b::2] = -float("inf")
    x[12, :15000] = -1e4
    x[13, 9:] = float("nan")
    u = torch.rand((B, V), generator=g).clamp(2.0 ** -24, 1 - 2.0 ** -24).to(cuda)
    want = ops.sample(x, temperature=T, uniforms=u, **kw)
    got = ops.verify_drafts(x, torch.zeros(0, dtype=torch.int32), torch.zeros(B + 1, dtype=torch.int32), 0, temperature=T,
                            uniforms=u, accept_uniforms=torch.zeros(0), **kw)
    assert torch.equal(got.tokens[:, 0], want.sampled)
    assert torch.isfinite(got.logprobs).all() and bool((got.logprobs <= 1e-5).all())
    if T == float("inf") and kw in (dict(), dict(top_k=9)):     # every token whose logit is finite, alike
        n = torch.isfinite(x).sum(1).double()
        assert torch.allclose(got.logprobs[:, 0].double(), -n.log(), rtol=0, atol=1e-5)
