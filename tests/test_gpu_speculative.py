"""The speculative-decoding front end and example on the GPU."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from vllm_webgpu_amd import ops
from vllm_webgpu_amd.v1.sample.rejection_sampler import RejectionSampler, SpecDecodeMetadata
from vllm_webgpu_amd.v1.sample.sampler import KeyStream, Sampler

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("speculative_decoding", os.path.join(ROOT, "examples", "speculative_decoding.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def batch(cuda, counts, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    drafts = [torch.randint(V, (n,), generator=g).tolist() for n in counts]
    return torch.randn((sum(counts) + len(counts), V), generator=g).mul_(4).to(cuda), SpecDecodeMetadata.make(drafts, cuda), drafts


def test_greedy_requests(cuda):
    logits, spec, drafts = batch(cuda, [3, 0, 2], 900)
    best = logits.argmax(1).tolist()
    spec.draft_token_ids[:2] = torch.tensor(best[:2], dtype=torch.int32)
    spec.draft_token_ids[3:] = torch.tensor(best[5:7], dtype=torch.int32)
    md = example().sampling(3, 1.0, 1.0, cuda)
    md.all_greedy, md.temperature = True, None
    out = RejectionSampler().forward(spec, None, logits, md).sampled_token_ids
    assert out.shape == (3, 4)
    assert RejectionSampler.parse_output(out, 900) == [best[0:3], [best[4]], best[5:8]]


def test_without_drafts_it_is_the_sampler(cuda):
    logits, spec, _ = batch(cuda, [0] * 9, 5000)
    md = example().sampling(9, 0.8, 0.9, cuda)
    torch.manual_seed(5)
    got = RejectionSampler()(spec, None, logits, md).sampled_token_ids
    torch.manual_seed(5)
    assert torch.equal(got, Sampler()(logits, md).sampled_token_ids)


def test_seeded_requests_repeat(cuda):
    logits, spec, _ = batch(cuda, [2, 4, 1, 3], 3000, seed=3)
    probs = torch.full((10, 3000), 1 / 3000.0, device=cuda)
    md = example().sampling(4, 1.0, 1.0, cuda)
    outs = []
    for _ in range(2):
        md.generators = {i: KeyStream(100 + i) for i in range(4)}
        outs.append(RejectionSampler()(spec, probs, logits, md).sampled_token_ids)
    assert torch.equal(outs[0], outs[1])


def test_refusals(cuda):
    logits, spec, _ = batch(cuda, [1], 100)
    for change in (dict(no_penalties=False), dict(max_num_logprobs=3), dict(bad_words_token_ids={0: [[1]]}),
                   dict(logit_bias=[{3: 1.0}]), dict(min_tokens={0: (2, {1})}),
                   dict(allowed_words=torch.zeros((1, 4), dtype=torch.int32))):
        md = example().sampling(1, 1.0, 1.0, cuda)
        for k, v in change.items():
            setattr(md, k, v)
        with pytest.raises(NotImplementedError):
            RejectionSampler()(spec, None, logits, md)


def test_the_example_learns_to_draft(cuda):
    rates = example().run(vocab=2000, rounds=3, batch=32, drafts=3, steps=4, train_steps=30)
    assert rates[0] < 0.5 and rates[-1] > rates[0] + 0.5, rates


def test_a_distilled_draft_is_accepted(cuda):
    """Gradient steps on the loss alone bring a draft's logits to the target's acceptance."""
    g = torch.Generator().manual_seed(1)
    V, N = 1500, 64
    target = (torch.randn((N, V), generator=g) * 2.5).to(cuda)
    lp = ops.sample(target, num_logprobs=64)
    student = torch.zeros((N, V), device=cuda, requires_grad=True)
    opt = torch.optim.Adam([student], lr=0.3)
    first = None
    for _ in range(60):
        loss = ops.distill_loss(student, lp.logprob_ids[:, 1:], lp.logprob_vals[:, 1:], tail="bucket").mean()
        first = float(loss.detach()) if first is None else first
        opt.zero_grad()
        loss.backward()
        opt.step()
    assert float(loss.detach()) < 0.05 * first
    q = torch.softmax(student.detach(), 1)
    overlap = torch.minimum(q, torch.softmax(target, 1)).sum(1).mean()
    rows = target.repeat_interleave(2, 0)
    accepted = torch.zeros((), device=cuda)
    for k in range(40):
        d = ops.sample(student.detach(), temperature=1.0, rng_key=1000 + k).sampled
        cu = torch.arange(N + 1, dtype=torch.int32, device=cuda)
        accepted += ops.verify_drafts(rows, d, cu, 1, draft_probs=q, temperature=1.0, rng_key=k).num_accepted.sum()
    rate, n = float(accepted) / (40 * N), 40 * N
    assert abs(rate - float(overlap)) < 5 * (0.25 / n) ** 0.5     # acceptance is the overlap of the two
