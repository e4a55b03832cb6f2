"""Decoding with drafted token trees over a paged cache, on a synthetic attention model.

    python examples/tree_decoding.py [--vocab 4000] [--batch 16] [--tokens 40] [--temperature 0]

The target is a small decoder with random weights (grouped heads, rotated positions).  A draft that knows the last
token only proposes, at every level of a tree, the most likely tokens after each node.  A step runs the target once over
all nodes of all requests: keys and values go into the paged cache with the rotation (``PagedKVCache.append``), every
node attends to its request's context and to its ancestors (``attend``), ``TreeSampler`` draws a token at each node and walks
down the tree, and the visited nodes' keys and values move up behind the context (``keep``).  Emitted tokens are
distributed as if the target had decoded one token at a time.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from vllm_webgpu_amd.v1.kv_cache import PagedKVCache  # noqa: E402
from vllm_webgpu_amd.v1.sample.metadata import SamplingMetadata  # noqa: E402
from vllm_webgpu_amd.v1.sample.tree_sampler import DraftTree, TreeSampler  # noqa: E402

BRANCHES = (3, 2, 1)  # drafted children of each node, level by level


class Target(torch.nn.Module):
    def __init__(self, vocab, width=256, layers=2, heads=4, kv_heads=2, dim=64, generator=None):
        super().__init__()
        def p(*shape, std):
            return torch.nn.Parameter(torch.randn(shape, generator=generator) * std, requires_grad=False)

        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.embed, self.out = p(vocab, width, std=1.0), p(width, vocab, std=3.0 * width ** -0.5)
        self.qkv = torch.nn.ParameterList(p(width, (heads + 2 * kv_heads) * dim, std=width ** -0.5) for _ in range(layers))
        self.mix = torch.nn.ParameterList(p(heads * dim, width, std=0.5 * (heads * dim) ** -0.5) for _ in range(layers))
        self.register_buffer("inv_freq", 10000.0 ** (-torch.arange(0, dim, 2).float() / dim))

    def forward(self, tokens, cache, table, context_lens, tree):
        """Logits [T, V] of every node."""
        x = self.embed[tokens.long()]
        positions, slots = (context_lens[tree.requests] + tree.depths).int(), cache.slots(table, context_lens, tree)
        for layer, (w, mix) in enumerate(zip(self.qkv, self.mix)):
            h = torch.nn.functional.layer_norm(x, x.shape[-1:])
            y = (h @ w).to(cache.k[0].dtype).unflatten(1, (-1, self.dim))
            q, k, v = y.split([self.heads, self.kv_heads, self.kv_heads], 1)
            q = cache.append(layer, k, v, slots, q=q, positions=positions, inv_freq=self.inv_freq)
            x = x + cache.attend(layer, q, table, context_lens, tree).flatten(1).float() @ mix
        return torch.nn.functional.layer_norm(x, x.shape[-1:]) @ self.out


def shape():
    """Parents of one request's tree, and the nodes of each level."""
    parents, levels = [-1], [[0]]
    for n in BRANCHES:
        level = []
        for p in levels[-1]:
            level += range(len(parents), len(parents) + n)
            parents += [p] * n
        levels.append(level)
    return parents, levels


def draft(target, last, levels):
    """Tokens [B, nodes]: the most likely ones after each node's token, as far as its embedding tells."""
    tokens = torch.zeros((last.shape[0], 1 + sum(len(v) for v in levels[1:])), dtype=torch.int32, device=last.device)
    tokens[:, 0] = last
    for n, above, level in zip(BRANCHES, levels, levels[1:]):
        e = torch.nn.functional.layer_norm(target.embed[tokens[:, above].long()], target.embed.shape[-1:])
        tokens[:, level] = (e @ target.out).topk(n, -1).indices.flatten(1).int()
    return tokens


def run(vocab=4000, batch=16, tokens=40, temperature=0.0, num_logprobs=None, seed=0, dtype=torch.float16):
    """(each request's prompt, its emitted tokens, their logprobs or None, accepted drafts per request and step, the target)."""
    dev = torch.device("cuda")
    g = torch.Generator().manual_seed(seed)
    torch.manual_seed(seed)
    target = Target(vocab, generator=g).to(dev)
    cache = PagedKVCache(len(target.qkv), 8 * batch + batch * (tokens // 16 + 4), target.kv_heads, target.dim, dtype=dtype, device=dev)
    names = [str(i) for i in range(batch)]
    prompts = [torch.randint(vocab, (int(n),), generator=g).tolist() for n in torch.randint(2, 100, (batch,), generator=g)]
    parents, levels = shape()
    for name, p in zip(names, prompts):
        cache.reserve(name, len(p) + tokens + 2 * len(parents))
    table = cache.block_table(names)
    md = SamplingMetadata(temperature=None if temperature == 0 else torch.full((batch,), temperature, device=dev),
                          all_greedy=temperature == 0, all_random=temperature > 0, top_p=None, top_k=None, generators={},
                          max_num_logprobs=num_logprobs, no_penalties=True, prompt_token_ids=None, frequency_penalties=None,
                          presence_penalties=None, repetition_penalties=None, output_token_ids=[])
    # the prompts but for their last tokens, as chains
    context = torch.zeros(batch, dtype=torch.int32, device=dev)
    chains = DraftTree.make([list(range(-1, len(p) - 2)) for p in prompts], dev)
    target(torch.tensor([t for p in prompts for t in p[:-1]], dtype=torch.int32, device=dev), cache, table, context, chains)
    context += torch.tensor([len(p) - 1 for p in prompts], dtype=torch.int32, device=dev)
    last = torch.tensor([p[-1] for p in prompts], dtype=torch.int32, device=dev)
    tree, sampler = DraftTree.make([parents] * batch, dev), TreeSampler()
    emitted, logprobs, accepted, steps = [[] for _ in names], [[] for _ in names], 0, 0
    while min(len(e) for e in emitted) < tokens:
        nodes = draft(target, last, levels).flatten()
        r = sampler(tree, nodes, target(nodes, cache, table, context, tree), md)
        cache.keep(table, context, r.path)
        count = r.num_accepted + 1
        # (requests that have their tokens stay where they are)
        more = torch.tensor([len(e) < tokens for e in emitted], device=dev)
        out = r.sampler_output.sampled_token_ids
        last = torch.where(more, out.gather(1, (count - 1).long().unsqueeze(1)).squeeze(1), last)
        context += torch.where(more, count, 0)
        lp = r.sampler_output.logprobs_tensors
        vals = None if lp is None else lp.logprobs.view(batch, out.shape[1], -1).tolist()
        for b, (row, n, m) in enumerate(zip(out.tolist(), count.tolist(), more.tolist())):
            if m:
                emitted[b] += row[:n]
                if vals is not None:
                    logprobs[b] += vals[b][:n]
        accepted += int(torch.where(more, r.num_accepted, 0).sum())
        steps += int(more.sum())
    return prompts, emitted, logprobs if num_logprobs is not None else None, accepted / steps, target


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, kind, default in (("vocab", int, 4000), ("batch", int, 16), ("tokens", int, 40), ("temperature", float, 0.0)):
        ap.add_argument(f"--{name}", type=kind, default=default)
    a = ap.parse_args()
    rate = run(a.vocab, a.batch, a.tokens, a.temperature)[3]
    print(f"{rate:.2f} of at most {len(BRANCHES)} drafted tokens accepted per request and step", flush=True)


if __name__ == "__main__":
    main()
