"""Drafts and verification from seeds that are the same."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_speculative import example
from vllm_webgpu_amd import ops
from vllm_webgpu_amd.v1.sample.rejection_sampler import RejectionSampler, SpecDecodeMetadata
from vllm_webgpu_amd.v1.sample.sampler import KeyStream, Sampler

pytestmark = pytest.mark.gpu

P, Q = [0.3, 0.3, 0.2, 0.1, 0.1], [0.1, 0.15, 0.05, 0.3, 0.4]


def frequencies(tokens, V):
    return torch.bincount(tokens.cpu().long(), minlength=V).double() / tokens.numel()


def fits(f, p, n):
    return bool(((f - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all())


def test_seeded_requests_are_the_targets_whatever_seed_the_draft_has(cuda):
    """Five standard deviations, for the first token and, after an acceptance, the second."""
    B, V = 60000, 5
    p, q = torch.tensor(P, dtype=torch.float64), torch.tensor(Q, dtype=torch.float64)
    md = example().sampling(B, 1.0, 1.0, cuda)
    md.generators = {i: KeyStream(i) for i in range(B)}
    drafts = Sampler()(q.log().float().expand(B, V).contiguous().to(cuda), md).sampled_token_ids.reshape(-1)
    assert fits(frequencies(drafts, V), q, B)
    spec = SpecDecodeMetadata.make([[0]] * B, cuda)
    spec.draft_token_ids = drafts.int()
    md.generators = {i: KeyStream(i) for i in range(B)}
    logits = p.log().float().expand(2 * B, V).contiguous().to(cuda)
    for probs in (q.float().expand(B, V).contiguous().to(cuda), None):
        out = RejectionSampler()(spec, probs, logits, md).sampled_token_ids
        assert fits(frequencies(out[:, 0], V), p, B), frequencies(out[:, 0], V)
        second = out[:, 1][out[:, 1] >= 0]
        assert fits(frequencies(second, V), p, second.numel())
        for g in md.generators.values():
            g.step = 0


def test_other_offsets_of_the_same_seeds(cuda):
    """The way that ``ops`` documents."""
    B, V = 60000, 5
    p, q = torch.tensor(P, dtype=torch.float64), torch.tensor(Q, dtype=torch.float64)
    seeds = torch.arange(B) * 3 + 1
    draft = ops.sample(q.log().float().expand(B, V).contiguous().to(cuda), temperature=1.0, rng_seeds=seeds,
                       rng_offsets=torch.zeros(B, dtype=torch.int64)).sampled
    cu = torch.arange(B + 1, dtype=torch.int32)
    r = ops.verify_drafts(p.log().float().expand(2 * B, V).contiguous().to(cuda), draft, cu, 1,
                          draft_probs=q.float().expand(B, V).contiguous().to(cuda), temperature=1.0, rng_seeds=seeds,
                          rng_offsets=torch.ones(B, dtype=torch.int64))
    assert fits(frequencies(r.tokens[:, 0], V), p, B)


def test_a_seeded_request_without_drafts_is_the_samplers(cuda):
    g = torch.Generator().manual_seed(3)
    B, V = 12, 4000
    logits = (torch.randn((B, V), generator=g) * 2).to(cuda)
    md = example().sampling(B, 0.9, 0.95, cuda)
    md.generators = {i: KeyStream(50 + i) for i in range(B)}
    want = Sampler()(logits, md).sampled_token_ids
    md.generators = {i: KeyStream(50 + i) for i in range(B)}
    assert torch.equal(RejectionSampler()(SpecDecodeMetadata.make([[]] * B, cuda), None, logits, md).sampled_token_ids, want)
