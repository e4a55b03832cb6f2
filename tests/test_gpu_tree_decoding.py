"""The operators around drafted trees as they are used together: a model that decodes through them, the front end, graphs,
streams."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from tests import tree_ref as R
from vllm_webgpu_amd import ops
from vllm_webgpu_amd.v1.kv_cache import PagedKVCache
from vllm_webgpu_amd.v1.sample.sampler import KeyStream, Sampler
from vllm_webgpu_amd.v1.sample.tree_sampler import DraftTree, TreeSampler

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example(name="tree_decoding"):
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, "examples", f"{name}.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def dense_logits(target, tokens):
    """Logits [n, V] of a whole sequence in 64 bits, without a cache."""
    norm = torch.nn.functional.layer_norm
    x = target.embed.double()[torch.tensor(tokens, device=target.embed.device)]
    n = len(tokens)
    for w, mix in zip(target.qkv, target.mix):
        y = (norm(x, x.shape[-1:]) @ w.double()).unflatten(1, (-1, target.dim))
        q, k, v = y.split([target.heads, target.kv_heads, target.kv_heads], 1)
        pos = torch.arange(n, device=x.device)
        q, k = R.rotate(q, pos, target.inv_freq)[0], R.rotate(k, pos, target.inv_freq)[0]
        k, v = (t.repeat_interleave(target.heads // target.kv_heads, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * target.dim ** -0.5
        s = s.masked_fill(torch.ones((n, n), dtype=torch.bool, device=x.device).triu(1), float("-inf"))
        x = x + torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v).flatten(1) @ mix.double()
    x = norm(x, x.shape[-1:])
    return x @ target.out.double(), x


def test_a_model_decodes_greedily_through_trees(cuda):
    """Every emitted token is the most likely one after what precedes it, by a dense forward in 64 bits."""
    prompts, emitted, lps, rate, target = example().run(vocab=2000, batch=6, tokens=25, num_logprobs=3)
    assert 0.3 < rate <= 3.0
    for p, e, lp in zip(prompts, emitted, lps):
        assert len(e) >= 25 and len(lp) == len(e)
        logits, x = dense_logits(target, p + e[:-1])
        logits, x = logits[len(p) - 1:], x[len(p) - 1:]
        # Queries, keys, values and outputs rounded to 2^-11, scores' errors of some 4 x 2^-11 times their size in the weights:
        # 16 x 2^-11 of a layer's mixed-in part, which is at most half of what it is added to, twice, through a norm
        off = 2 * 16 * 2.0 ** -11 * x.norm(dim=1) * target.out.double().norm(dim=0).max()
        mine = logits.gather(1, torch.tensor(e, device=cuda).unsqueeze(1)).squeeze(1)
        assert bool((mine >= logits.amax(1) - 2 * off).all())
        want = torch.log_softmax(logits, 1)
        got = torch.tensor(lp, device=cuda).double()
        assert bool(((got[:, 0] - want.gather(1, torch.tensor(e, device=cuda).unsqueeze(1)).squeeze(1)).abs() <= 2 * off).all())
        assert bool(((got[:, 1:] - want.topk(3, 1).values).abs() <= (2 * off).unsqueeze(1)).all())


def test_sampled_tokens_are_the_targets(cuda):
    """The first token after a root whose children are its likeliest tokens has the target's distribution, and so has the
    second one, given the first."""
    V, B = 40, 6000
    g = torch.Generator().manual_seed(2)
    first, second = (torch.randn(n, V, generator=g).mul_(1.5).to(cuda) for n in (1, V))
    kids = first[0].topk(3).indices.tolist()
    tree = DraftTree.make([[-1, 0, 0, 0]] * B, cuda)
    tokens = torch.tensor([0] + kids, dtype=torch.int32, device=cuda).repeat(B)
    logits = torch.stack([first[0]] + [second[k] for k in kids]).repeat(B, 1)
    md = example("speculative_decoding").sampling(B, 1.0, 1.0, cuda)
    torch.manual_seed(3)
    out = TreeSampler()(tree, tokens, logits, md)
    t = out.sampler_output.sampled_token_ids
    p = torch.softmax(first[0].double(), 0)
    share = torch.bincount(t[:, 0].long(), minlength=V).double() / B
    assert bool(((share - p).abs() <= 5 * (p * (1 - p) / B).sqrt() + 1e-9).all())
    for k in kids:
        rows = t[t[:, 0] == k]
        q = torch.softmax(second[k].double(), 0)
        got = torch.bincount(rows[:, 1].long(), minlength=V).double() / len(rows)
        assert bool(((got - q).abs() <= 5 * (q * (1 - q) / len(rows)).sqrt() + 5.0 / len(rows)).all())
    assert torch.equal(out.num_accepted, (t >= 0).sum(1).int() - 1)


def test_seeded_requests_repeat_and_logprobs(cuda):
    V, B = 3000, 4
    g = torch.Generator().manual_seed(4)
    tree = DraftTree.make([R.random_tree(n, g) for n in (1, 9, 40, 5)], cuda)
    T = tree.parents.numel()
    logits = torch.randn((T, V), generator=g).mul_(3).to(cuda)
    tokens = torch.randint(V, (T,), generator=g).int().to(cuda)
    md = example("speculative_decoding").sampling(B, 0.7, 0.9, cuda)
    md.max_num_logprobs = 4
    outs = []
    for _ in range(2):
        md.generators = {i: KeyStream(40 + i) for i in range(B)}
        outs.append(TreeSampler()(tree, tokens, logits, md))
    a, b = outs
    assert torch.equal(a.sampler_output.sampled_token_ids, b.sampler_output.sampled_token_ids) and torch.equal(a.path, b.path)
    lp = a.sampler_output.logprobs_tensors
    W = tree.max_depth + 1
    ids, vals = lp.logprob_token_ids.view(B, W, 5), lp.logprobs.view(B, W, 5)
    want = torch.log_softmax(logits.double(), 1)
    for i in range(B):
        for j, node in enumerate(a.path[i].tolist()):
            if node < 0:
                assert ids[i, j].tolist() == [-1] * 5 and not bool(vals[i, j].any())
                continue
            row = want[int(tree.cu_nodes[i]) + node]
            assert int(ids[i, j, 0]) == int(a.sampler_output.sampled_token_ids[i, j])
            assert ids[i, j, 1:].tolist() == row.topk(4).indices.tolist()
            assert bool(((vals[i, j].double() - row[ids[i, j].long()]).abs() < 1e-5).all())


def test_the_front_end_refuses_what_it_cannot_verify(cuda):
    tree = DraftTree.make([[-1, 0]], cuda)
    logits, tokens = torch.zeros((2, 50), device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    for change in (dict(no_penalties=False), dict(bad_words_token_ids={0: [[1]]}), dict(logit_bias=[{3: 1.0}])):
        md = example("speculative_decoding").sampling(1, 1.0, 1.0, cuda)
        for k, v in change.items():
            setattr(md, k, v)
        with pytest.raises(NotImplementedError):
            TreeSampler()(tree, tokens, logits, md)
    with pytest.raises(ValueError):
        TreeSampler()(tree, tokens, logits[:1], example("speculative_decoding").sampling(1, 1.0, 1.0, cuda))


def test_prompt_logprobs(cuda):
    g = torch.Generator().manual_seed(5)
    logits, ids = torch.randn((30, 700), generator=g).to(cuda), torch.randint(700, (30,), generator=g).to(cuda)
    lp = Sampler().gather_logprobs(logits, 6, ids)
    w = R.logprobs(logits, ids, 1.0, 6)
    assert torch.equal(lp.logprob_token_ids.long(), w["ids"]) and torch.equal(lp.selected_token_ranks.long(), w["ranks"])
    assert bool(((lp.logprobs.double() - w["vals"]).abs() <= w["vals_off"]).all())


def step_inputs(dev, seed, contexts=(300, 17, 900), nodes=(12, 5, 30)):
    g = torch.Generator().manual_seed(seed)
    tree = DraftTree.make([R.random_tree(n, g) for n in nodes], dev)
    T = tree.parents.numel()
    cache = PagedKVCache(1, 120, 2, 128, device=dev)
    cache.k[0].copy_(torch.randn(cache.k[0].shape, generator=g))
    cache.v[0].copy_(torch.randn(cache.v[0].shape, generator=g))
    for i, (c, n) in enumerate(zip(contexts, nodes)):
        cache.reserve(str(i), c + n)
    table = cache.block_table([str(i) for i in range(len(nodes))])
    context = torch.tensor(contexts, dtype=torch.int32).to(dev)
    x = torch.randn((T, 12 * 128), generator=g).bfloat16().to(dev).unflatten(1, (12, 128))
    logits = torch.randn((T, 5003), generator=g).mul_(2).to(dev)
    tokens = torch.randint(5003, (T,), generator=g).int().to(dev)
    return dict(tree=tree, cache=cache, table=table, context=context, x=x, logits=logits, tokens=tokens,
                inv_freq=10000.0 ** (-torch.arange(64, device=dev).float() / 64))


def one_step(s):
    """Every operator in the order of a decoding step; the cache is left as it was."""
    q, k, v = s["x"].split([8, 2, 2], 1)
    tree, cache = s["tree"], s["cache"]
    saved = cache.k[0].clone(), cache.v[0].clone()
    slots = cache.slots(s["table"], s["context"], tree)
    q = cache.append(0, k, v, slots, q=q, positions=s["context"][tree.requests] + tree.depths, inv_freq=s["inv_freq"])
    out = cache.attend(0, q, s["table"], s["context"], tree)
    best = ops.argmax(s["logits"])
    r = ops.accept_tree(best, torch.where(tree.numbers % 2 == 0, best[tree.cu_nodes[:-1].long()[tree.requests] + tree.parents.clamp(min=0)],
                                          s["tokens"]), tree.parents, tree.cu_nodes, tree.max_depth + 1)
    cache.keep(s["table"], s["context"], r.path)
    after = cache.k[0].clone(), cache.v[0].clone()
    cache.k[0].copy_(saved[0])
    cache.v[0].copy_(saved[1])
    lp = ops.token_logprobs(s["logits"], best, 5, True)
    return [q, out, r.tokens, r.path, r.num_accepted, *after, lp.logprobs, lp.entropy, lp.logprob_ids, lp.logprob_vals, lp.logprob_ranks]


def test_a_step_in_a_graph(cuda):
    """Captured once, replayed with other inputs in the same memory, with eager steps between the replays; two graphs."""
    s, other = step_inputs(cuda, 1), step_inputs(cuda, 2, contexts=(20, 1000, 450), nodes=(30, 12, 5))
    for t in (s, other):
        one_step(t)
    torch.cuda.synchronize()
    graphs = []
    for t in (s, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = one_step(t)
        graphs.append((g, outs, t))
    gen = torch.Generator(device=cuda).manual_seed(7)
    for i in range(4):
        for g, outs, t in graphs:
            t["x"].copy_(torch.randn(t["x"].shape, generator=gen, device=cuda))
            t["logits"].copy_(torch.randn(t["logits"].shape, generator=gen, device=cuda))
            want = one_step(t)
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
    # both at once, beside eager steps
    streams = [torch.cuda.Stream() for _ in graphs]
    want = [one_step(t) for _, _, t in graphs]
    torch.cuda.synchronize()
    for (g, _, _), st in zip(graphs, streams):
        with torch.cuda.stream(st):
            g.replay()
    third = step_inputs(cuda, 9)
    eager = one_step(third)
    torch.cuda.synchronize()
    for (_, outs, _), w in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(outs, w))
    assert all(torch.equal(a, b) for a, b in zip(eager, one_step(third)))


def test_steps_on_several_streams(cuda):
    """Steps that overlap on streams of their own, and on one stream in turn, give what one alone gives."""
    inputs = [step_inputs(cuda, i) for i in range(4)]
    want = [one_step(s) for s in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = []
    for _ in range(3):
        got = []
        for s, st in zip(inputs, streams):
            with torch.cuda.stream(st):
                got.append(one_step(s))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_training_in_a_graph_beside_an_eager_one(cuda):
    """A forward and backward captured while an eager graph of another leaf lives; replays against eager gradients."""
    g = torch.Generator(device=cuda).manual_seed(8)
    x = torch.randn((40, 7001), generator=g, device=cuda).bfloat16().requires_grad_()
    ids = torch.randint(-1, 7001, (40,), generator=g, device=cuda).int()
    gl, gh = torch.randn(40, generator=g, device=cuda), torch.randn(40, generator=g, device=cuda)

    def grads(leaf):
        r = ops.token_logprobs(leaf, ids, entropy=True, temperature=0.9)
        return [r.logprobs.detach(), torch.autograd.grad([r.logprobs, r.entropy], [leaf], [gl, gh])[0]]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        grads(x)
    torch.cuda.current_stream().wait_stream(s)
    other = x.detach().clone().requires_grad_()
    alive = ops.token_logprobs(other, ids, entropy=True)     # an eager graph that outlives the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = grads(x)
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g, device=cuda))
        want = grads(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    assert torch.autograd.grad(alive.logprobs.sum(), other)[0].shape == x.shape
