"""``RejectionSampler``: vLLM-v1's verification layer of speculative decoding as one call into the library.

The reference decodes one token per request and step (``vllm_webgpu/v1/model_runner.py:129-137``) and
has no drafts; this class keeps the shape of vLLM-v1's rejection sampler: ``forward(metadata,
draft_probs, logits, sampling_metadata) -> SamplerOutput`` with ``sampled_token_ids`` int32
``[B, max_spec_len + 1]`` (accepted drafts, one token drawn from the target, then ``PLACEHOLDER``),
and ``parse_output`` for the host's lists.  Unlike there, the logits are the target's rows of every
request together, the row after its last draft included (the bonus token is drawn in the same call):
``metadata.num_draft_tokens[i] + 1`` consecutive rows for request ``i``.

Temperature, top-k, top-p, min-p and seeded requests follow ``Sampler``; the logits are those after a
model's soft cap.  A seeded request with drafts is verified with keys of another domain than
``Sampler``'s: its drafts may have been sampled from a stream of the same seed, and a token raced with
the numbers that chose the refused draft would not be the target's.  Requests with penalties,
logits processors or raw logprobs change the distribution from one draft to the next and are refused:
sample them one by one.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ... import ops
from ..outputs import SamplerOutput
from .metadata import SamplingMetadata
from .sampler import _SEED_HI, _SEED_LO, SeedStaging, draw_seeds

PLACEHOLDER = -1
_DOMAIN = 0x6A09E667F3BCC908  # of requests with drafts (the fraction of sqrt(2): any constant will do)


@dataclass
class SpecDecodeMetadata:
    """A step's drafts, in vLLM-v1's names: ``draft_token_ids`` int32 ``[num_tokens]`` of all requests,
    ``num_draft_tokens`` per request, ``cu_num_draft_tokens`` int32 ``[B + 1]`` their running count from
    0 (vLLM-v1's starts with the first request's)."""

    draft_token_ids: torch.Tensor
    num_draft_tokens: list[int]
    cu_num_draft_tokens: torch.Tensor
    max_spec_len: int

    @classmethod
    def make(cls, draft_token_ids: list[list[int]], device: torch.device) -> "SpecDecodeMetadata":
        counts = [len(d) for d in draft_token_ids]
        cu = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32)
        flat = torch.tensor([t for d in draft_token_ids for t in d], dtype=torch.int32)
        return cls(flat.to(device), counts, cu.to(device), max(counts, default=0))


class RejectionSampler:
    def __init__(self) -> None:
        self._seeds = SeedStaging()

    def __call__(self, *args, **kwargs) -> SamplerOutput:
        return self.forward(*args, **kwargs)

    def forward(self, metadata: SpecDecodeMetadata, draft_probs: torch.Tensor | None, logits: torch.Tensor,
                sampling_metadata: SamplingMetadata) -> SamplerOutput:
        """``draft_probs`` ``[num_tokens, V]``: what the drafts were drawn from; None: looked-up or
        greedy drafts."""
        m = sampling_metadata
        if not m.no_penalties:
            raise NotImplementedError("drafts of requests with penalties are not verified")
        if (m.allowed_token_ids_mask is not None or m.allowed_words is not None or m.bad_words_token_ids or m.min_tokens
                or (m.logit_bias and any(m.logit_bias))):
            raise NotImplementedError("drafts of requests with logits processors are not verified")
        if m.max_num_logprobs is not None:
            raise NotImplementedError("raw logprobs are not computed for drafts")
        B = len(metadata.num_draft_tokens)
        temperature = None if m.all_greedy else m.temperature
        seeds = key = None
        if temperature is not None:
            if m.generators:
                domain = torch.tensor([_DOMAIN if n else 0 for n in metadata.num_draft_tokens], dtype=torch.int64)
                seeds = draw_seeds(B, m.generators, logits.device, self._seeds, domain)
            else:
                key = int(torch.randint(_SEED_LO, _SEED_HI, (1,), dtype=torch.int64))
        r = ops.verify_drafts(logits, metadata.draft_token_ids, metadata.cu_num_draft_tokens, metadata.max_spec_len,
                              draft_probs=draft_probs, temperature=temperature, top_k=m.top_k, top_p=m.top_p,
                              min_p=m.min_p, rng_seeds=seeds, rng_key=key)
        return SamplerOutput(sampled_token_ids=r.tokens, logprobs_tensors=None)

    @staticmethod
    def parse_output(output_token_ids: torch.Tensor, vocab_size: int) -> list[list[int]]:
        """Each request's emitted tokens, on the host."""
        return [[t for t in row if t != PLACEHOLDER and t < vocab_size] for row in output_token_ids.tolist()]
