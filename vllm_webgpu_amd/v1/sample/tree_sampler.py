"""``TreeSampler``: verification of drafted token trees, beside ``RejectionSampler`` for drafted chains.

The reference decodes one token per request and step (``vllm_webgpu/v1/model_runner.py:129-137``) and
has no drafts.  A request's tree has the last emitted token at its root (node 0) and drafted tokens below
it; the target's logits of every node come from one forward over all of them (``PagedKVCache.attend``).
A token is drawn from the target at every node, and the walk from the root follows the child that holds it: what
is emitted was drawn from the target, whatever was drafted.  Unlike a chain's rejection sampler the draft's
distribution is not needed, and siblings may be chosen in any way.

Temperature, top-k, top-p, min-p and seeded requests follow ``Sampler``: a seeded request's nodes draw
with one key of the step and their numbers as offsets, in the domain of ``RejectionSampler``'s keys.  Requests
with penalties or logits processors are refused, as there.  Raw logprobs are those of the emitted tokens.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ... import ops
from ..outputs import LogprobsTensors, SamplerOutput
from .metadata import SamplingMetadata
from .rejection_sampler import _DOMAIN, refuse_processors
from .sampler import _SEED_HI, _SEED_LO, SeedStaging, draw_seeds


@dataclass
class DraftTree:
    """A step's trees, all requests' nodes one after another: ``parents`` int32 [T] (numbers in the request, -1 for
    the root, node 0; each less than the node's own), ``cu_nodes`` int32 [B + 1] the running count of nodes,
    ``requests`` and ``numbers`` int64 [T] each node's request and number, ``depths`` int32 [T], ``visible`` int32
    [T, ceil(max_nodes / 32)] the bit words of each node's ancestors and itself (``ops.tree_attention``)."""

    parents: torch.Tensor
    cu_nodes: torch.Tensor
    requests: torch.Tensor
    numbers: torch.Tensor
    depths: torch.Tensor
    visible: torch.Tensor
    num_nodes: list[int]
    max_nodes: int
    max_depth: int

    @classmethod
    def make(cls, parents: list[list[int]], device: torch.device) -> "DraftTree":
        """From each request's parents, the root's -1 first."""
        counts = [len(p) for p in parents]
        most = max(counts, default=0)
        if not counts or min(counts) < 1 or most > ops._lib.MAX_TREE_NODES:
            raise ValueError(f"a tree has 1 to {ops._lib.MAX_TREE_NODES} nodes (got {counts})")
        words, depths, numbers = [], [], []
        for tree in parents:
            if tree[0] != -1 or any(not 0 <= p < i for i, p in enumerate(tree) if i):
                raise ValueError(f"a tree's root is its first node, and every parent comes before its node (got {tree})")
            seen, depth = [1], [0]
            for i, p in enumerate(tree[1:], 1):
                seen.append(seen[p] | 1 << i)
                depth.append(depth[p] + 1)
            for s in seen:
                row = [(s >> 32 * w) & 0xFFFFFFFF for w in range((most + 31) // 32)]
                words.append([w - 2 ** 32 if w >= 2 ** 31 else w for w in row])
            depths += depth
            numbers += range(len(tree))
        def put(x, dtype):
            return torch.tensor(x, dtype=dtype).to(device)

        cu = torch.tensor([0] + counts).cumsum(0)
        return cls(put([p for t in parents for p in t], torch.int32), cu.to(device=device, dtype=torch.int32),
                   torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts)).to(device),
                   put(numbers, torch.int64), put(depths, torch.int32), put(words, torch.int32), counts, most, max(depths))


@dataclass
class TreeSamplerOutput:
    sampler_output: SamplerOutput  # sampled_token_ids int32 [B, max_depth + 1]: the emitted tokens, then -1; with logprobs, those
                                   # of the positions [B * (max_depth + 1), L + 1] (past a request's last token ids are -1)
    path: torch.Tensor             # int32 [B, max_depth + 1]: the visited nodes, then -1 (``PagedKVCache.keep``)
    num_accepted: torch.Tensor     # int32 [B]: accepted drafted tokens (one token more is emitted)


class TreeSampler:
    def __init__(self) -> None:
        self._seeds = SeedStaging()

    def __call__(self, *args, **kwargs) -> TreeSamplerOutput:
        return self.forward(*args, **kwargs)

    def forward(self, tree: DraftTree, token_ids: torch.Tensor, logits: torch.Tensor,
                sampling_metadata: SamplingMetadata) -> TreeSamplerOutput:
        """``token_ids`` int32 [T]: the nodes' tokens; ``logits`` [T, V]: the target's at each node."""
        m, T, B = sampling_metadata, tree.parents.numel(), len(tree.num_nodes)
        refuse_processors(m)
        if logits.dim() != 2 or logits.shape[0] != T or token_ids.shape != (T,):
            raise ValueError(f"logits must be [{T}, V] and token_ids [{T}] (got {tuple(logits.shape)} and {tuple(token_ids.shape)})")

        def rows(name):
            t = getattr(m, name)
            if t is not None and t.shape != (B,):  # (a device would index past its end)
                raise ValueError(f"{name} must be [{B}], one for each tree (got {tuple(t.shape)})")
            return None if t is None else t[tree.requests]

        kw: dict = {}
        if not m.all_greedy and m.temperature is not None:
            kw = {name: rows(name) for name in ("temperature", "top_k", "top_p", "min_p")}
            if m.generators:
                domain = torch.full((B,), _DOMAIN, dtype=torch.int64)
                seeds = draw_seeds(B, m.generators, logits.device, self._seeds, domain)
                kw.update(rng_seeds=seeds[tree.requests], rng_offsets=tree.numbers)
            else:
                kw["rng_key"] = int(torch.randint(_SEED_LO, _SEED_HI, (1,), dtype=torch.int64))
        sampled = ops.sample(logits, **kw).sampled
        r = ops.accept_tree(sampled, token_ids, tree.parents, tree.cu_nodes, tree.max_depth + 1)
        lp = None
        if m.max_num_logprobs is not None:
            # only the visited nodes' rows are read
            live = r.path >= 0
            at = torch.where(live, tree.cu_nodes[:-1].unsqueeze(1) + r.path, T).long()
            ids = torch.full((T + 1,), -1, dtype=torch.int32, device=logits.device)
            ids[at.flatten()] = r.tokens.flatten()  # (the last entry takes what is past the walks)
            s = ops.token_logprobs(logits, ids[:T], m.max_num_logprobs)
            at = at.clamp(max=T - 1).flatten()
            off = ~live.flatten()
            lp = LogprobsTensors(s.logprob_ids[at].masked_fill_(off.unsqueeze(1), -1), s.logprob_vals[at].masked_fill_(off.unsqueeze(1), 0.0),
                                 s.logprob_ranks[at].masked_fill_(off, 0))
        return TreeSamplerOutput(SamplerOutput(sampled_token_ids=r.tokens, logprobs_tensors=lp), r.path, r.num_accepted)
