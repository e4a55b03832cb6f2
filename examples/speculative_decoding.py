"""Speculative decoding with a draft that learns from its target, on synthetic models.

    python examples/speculative_decoding.py [--vocab 4000] [--rounds 5] [--batch 64] [--drafts 4]

The target is a fixed random next-token model (an embedding of the last token, one hidden layer, an
output matrix); the draft a smaller one that starts with random weights.  Each round the requests
decode speculatively: the draft proposes ``--drafts`` tokens, the target's logits of all positions
are verified in one call (``RejectionSampler``).  The target's sampler then gives its top
log-probabilities at those positions, and the draft takes a few optimiser steps on the distillation
loss against them (``ops.distill_loss``).  The number of accepted drafts per step rises with the rounds,
while the emitted tokens stay distributed as the target's.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from vllm_webgpu_amd import ops  # noqa: E402
from vllm_webgpu_amd.v1.sample.metadata import SamplingMetadata  # noqa: E402
from vllm_webgpu_amd.v1.sample.rejection_sampler import RejectionSampler, SpecDecodeMetadata  # noqa: E402


class NextToken(torch.nn.Module):
    """Logits [n, V] of the tokens that follow ``tokens`` [n]."""

    def __init__(self, vocab: int, width: int, gain: float, generator: torch.Generator):
        super().__init__()
        def p(*shape, std):
            return torch.nn.Parameter(torch.randn(shape, generator=generator) * std)

        self.embed, self.mix = p(vocab, width, std=1.0), p(width, width, std=width ** -0.5)
        self.out = p(width, vocab, std=gain * width ** -0.5)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        h = self.embed[tokens.long()]
        return (h + torch.tanh(h @ self.mix)) @ self.out


def sampling(B: int, temperature: float, top_p: float, device) -> SamplingMetadata:
    return SamplingMetadata(temperature=torch.full((B,), temperature, device=device), all_greedy=False, all_random=True,
                            top_p=torch.full((B,), top_p, device=device) if top_p < 1 else None, top_k=None, generators={},
                            max_num_logprobs=None, no_penalties=True, prompt_token_ids=None, frequency_penalties=None,
                            presence_penalties=None, repetition_penalties=None, output_token_ids=[])


def draft_tokens(draft, last: torch.Tensor, count: int, temperature: float):
    """``count`` tokens [B, count] after each of ``last``, and the distributions they were drawn from."""
    tokens, probs = [], []
    for _ in range(count):
        logits = draft(last)
        probs.append(ops.softmax(logits, temperature)[0])
        key = int(torch.randint(2 ** 62, (1,)))
        last = ops.sample(logits, temperature=temperature, rng_key=key).sampled
        tokens.append(last)
    return torch.stack(tokens, 1), torch.stack(probs, 1)


def run(vocab=4000, rounds=5, batch=64, drafts=4, steps=8, temperature=0.8, top_p=0.95, top=32, train_steps=100, seed=0):
    """Accepted drafts per request and step, of each round."""
    dev = torch.device("cuda")
    torch.manual_seed(seed)
    g = torch.Generator().manual_seed(seed)
    target = NextToken(vocab, 64, 3.0, g).to(dev)
    draft = NextToken(vocab, 48, 0.1, g).to(dev)
    opt = torch.optim.Adam(draft.parameters(), lr=0.01)
    verifier, md = RejectionSampler(), sampling(batch, temperature, top_p, dev)
    spec = SpecDecodeMetadata.make([[0] * drafts] * batch, dev)
    last = torch.randint(64, (batch,), generator=g).int().to(dev)  # (few prompts, so that rounds meet the same tokens)
    first, rates = last.clone(), []
    for _ in range(rounds):
        seen, accepted = [], 0
        last = first.clone()
        for _ in range(steps):
            with torch.no_grad():
                tokens, probs = draft_tokens(draft, last, drafts, temperature)
                inputs = torch.cat([last.unsqueeze(1), tokens], 1)        # [B, drafts + 1]
                logits = target(inputs.reshape(-1))
                spec.draft_token_ids = tokens.reshape(-1)
                out = verifier(spec, probs.reshape(batch * drafts, vocab), logits, md).sampled_token_ids
                count = (out >= 0).sum(1)
                accepted += int((count - 1).sum())
                last = out.gather(1, (count - 1).unsqueeze(1)).squeeze(1)
                lp = ops.sample(logits, num_logprobs=top)                  # the target's top log-probabilities
                live = torch.arange(drafts + 1, device=dev) < count.unsqueeze(1)
                seen.append((inputs.reshape(-1), lp.logprob_ids[:, 1:], lp.logprob_vals[:, 1:], live.reshape(-1).float()))
        rates.append(accepted / (batch * steps))
        inputs, ids, values, weight = (torch.cat(t) for t in zip(*seen))
        for _ in range(train_steps):
            loss = ops.distill_loss(draft(inputs), ids, values, weight, tail="bucket").sum() / weight.sum()
            opt.zero_grad()
            loss.backward()
            opt.step()
    return rates


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("vocab", 4000), ("rounds", 5), ("batch", 64), ("drafts", 4)):
        ap.add_argument(f"--{name}", type=int, default=default)
    a = ap.parse_args()
    for i, rate in enumerate(run(a.vocab, a.rounds, a.batch, a.drafts)):
        print(f"round {i}: {rate:.2f} of {a.drafts} drafts accepted per request and step", flush=True)


if __name__ == "__main__":
    main()
