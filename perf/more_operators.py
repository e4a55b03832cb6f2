"""The work that the operators around a verified tree of drafts are measured on: the paged cache that
the target's attention reads, that attention, the walk down the tree, and the log-probabilities of the
tokens that come out (or that a prompt or a rollout holds), with their gradient.

A case is one call on device-resident tensors, as a serving or training loop makes it:

* ``op="append"``: ``ops.append_kv``, a layer's keys and values into the cache, keys and queries rotated;
* ``op="tree"``: ``ops.tree_attention``, every request's drafted tree over its cached context;
* ``op="accept"``: ``ops.accept_tree``, the sampled tokens walked down each request's tree;
* ``op="compact"``: ``ops.compact_kv``, a layer's accepted keys and values moved up behind the context;
* ``op="score"``: ``ops.token_logprobs`` with entropy, ranks and top alternatives;
* ``op="train"``: its log-probabilities and entropies, and through autograd the logits' gradient.

With ``own`` false the same results come from elementary torch operations in 32 bits (angles in 64).

The cache has ``pages`` of ``page`` tokens: keys [pages, kv_heads, page, dim], values
[pages, kv_heads, dim, page]; a request's pages are scattered over it.  Queries, keys and values are
N(0, 1).  A tree is a root (the last sampled token) and drafted nodes, each after its parent, of
whom a node sees its ancestors and itself: ``visible``, bit words.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

_APPEND = {"op": "append", "tokens": 1, "runs": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "page": 16,
           "dtype": "bf16", "interleaved": False, "far": 8192, "skipped": 0.0, "cached": 65536}
_TREE = {"op": "tree", "batch": 1, "context": 2048, "ragged": False, "nodes": 16, "shape": "tree", "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16"}
_ACCEPT = {"op": "accept", "batch": 1, "nodes": 16, "ragged": False, "hit": 0.7}
_COMPACT = {"op": "compact", "batch": 1, "context": 1024, "nodes": 16, "accepted": 5, "kv_heads": 8, "dim": 128,
            "page": 16, "dtype": "bf16"}
_SCORE = {"op": "score", "rows": 1, "vocab": 32000, "dtype": "bf16", "top": 20, "temperature": 1.0, "masked": 0.0}


def _case(base, name=None, **kw):
    c = dict(base, **kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # a step's trees of 48 requests, one layer: few tokens, each in a page of its own request
        _case(_APPEND, "append_trees", tokens=701, runs=48, far=32768),
        # prompts of five requests, one layer: whole pages but for the ends; half of each head rotated
        _case(_APPEND, "append_prompts", tokens=16384, runs=5, kv_heads=4, rotary=64, interleaved=True, dtype="f16", page=64),
        # one chat request's tree of twelve nodes: latency
        _case(_TREE, "tree_one", nodes=12, context=1900),
        # a batch of chats, contexts and trees of many lengths
        _case(_TREE, "tree_64", batch=64, context=8192, ragged=True, nodes=32, page=32),
        # long documents; few requests, all of the chip for each
        _case(_TREE, "tree_long", batch=3, context=131000, nodes=8, heads=64, dtype="f16"),
        # one request's tree, and a full batch of the largest trees
        _case(_ACCEPT, "accept_one", nodes=12),
        _case(_ACCEPT, "accept_256", batch=256, nodes=64, ragged=True),
        # the same two, one layer's cache
        _case(_COMPACT, "compact_one", nodes=12, accepted=3),
        _case(_COMPACT, "compact_200", batch=200, nodes=64, accepted=7, kv_heads=4, page=64),
        # the tokens of one verified request, on a vocabulary whose rows start unaligned: latency
        _case(_SCORE, "score_7_odd", rows=7, vocab=50257, dtype="f32", top=5),
        # a prompt's log-probabilities with twenty alternatives each
        _case(_SCORE, "score_1999", rows=1999, vocab=151936),
        # a policy's rollouts, prompt positions masked out: log-probabilities, entropy, gradient
        _case(_SCORE, "train_4096", op="train", rows=4096, vocab=128256, masked=0.2, temperature=0.9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "tree", "tree", "accept", "compact", "score", "train"])
    kv_heads, group = rng.choice([(8, 4), (8, 8), (4, 7), (2, 8), (1, 16), (16, 1), (5, 3)])
    dim = rng.choice([64, 128, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    heads = dict(heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if op == "append":
        tokens = max(1, min(_log_int(rng, 1, 16384), (1 << 26) // (dim * (kv_heads * group + kv_heads))))
        return _case(_APPEND, tokens=tokens, runs=rng.randint(1, min(64, tokens)), rotary=rng.choice([dim, dim, dim // 2]),
                     interleaved=rng.random() < 0.3, far=_log_int(rng, 100, 1 << 20), skipped=rng.choice([0.0, 0.0, 0.1]), **heads)
    if op == "tree":
        nodes = rng.choice([1, rng.randint(2, 16), _log_int(rng, 2, 64)])
        context = rng.choice([rng.randint(0, 300), _log_int(rng, 100, 131000)])
        most = min((3 * 131000) // (context + nodes), (3 * 131000 * 8 * 64) // ((context + nodes) * nodes * kv_heads * group),
                   (3 * 131000 * 1024) // ((context + nodes) * kv_heads * dim))
        return _case(_TREE, batch=max(1, min(_log_int(rng, 1, 128), most)), context=context, ragged=rng.random() < 0.6,
                     nodes=nodes, shape=rng.choice(["tree", "tree", "chain"]), **heads)
    if op == "accept":
        return _case(_ACCEPT, batch=_log_int(rng, 1, 256), nodes=rng.randint(1, 64), ragged=rng.random() < 0.5,
                     hit=round(rng.uniform(0.2, 0.95), 2))
    if op == "compact":
        del heads["heads"]
        nodes = rng.randint(4, 64)
        return _case(_COMPACT, batch=_log_int(rng, 1, 200), context=rng.randint(0, 1024), nodes=nodes,
                     accepted=rng.randint(0, min(12, nodes // 2 - 1)), **heads)
    vocab = rng.choice([32000, 128256, 151936, 262144, _log_int(rng, 1000, 262144) | 1])
    rows = max(1, min(_log_int(rng, 1, 4096), (1 << 28) // vocab))
    return _case(_SCORE, op=op, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "bf16", "bf16", "f16"]),
                 top=rng.choice([0, 5, 20, rng.randint(1, 64)]), temperature=rng.choice([1.0, round(rng.uniform(0.5, 2.0), 2)]),
                 masked=rng.choice([0.0, 0.0, 0.3]))


# ---- inputs ---------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 6151 + 47)


def _running(counts):
    return torch.tensor([0] + list(counts), device="cuda").cumsum(0)


def _cache(g, pages, kv_heads, dim, page, dtype):
    """(keys, values): N(0, 1)."""
    out = []
    for shape in ((pages, kv_heads, page, dim), (pages, kv_heads, dim, page)):
        t = torch.empty(shape, dtype=_DTYPES[dtype], device="cuda")
        for i in range(0, pages, 4096):
            t[i:i + 4096] = torch.randn(t[i:i + 4096].shape, generator=g, device="cuda")
        out.append(t)
    return out


def _append_inputs(case, seed):
    g, dev, T, page = _generator(seed), "cuda", case["tokens"], case["page"]
    H, Hk, D, R = case["heads"], case["kv_heads"], case["dim"], case["rotary"]
    qkv = torch.randn((T, (H + 2 * Hk) * D), generator=g, device=dev).to(_DTYPES[case["dtype"]])  # one projection's output
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([H * D, Hk * D, Hk * D], 1))
    # the tokens in `runs` runs, each from some position on, in pages of its own
    n = T // case["runs"]
    lengths = [n] * (case["runs"] - 1) + [T - n * (case["runs"] - 1)]
    starts = torch.randint(case["far"], (len(lengths),), generator=g, device=dev)
    need = [(n + page - 1) // page + 1 for n in lengths]
    pages = max(case["cached"] // page, sum(need))
    order, first = torch.randperm(pages, generator=g, device=dev), _running(need)
    run = torch.repeat_interleave(torch.arange(len(lengths), device=dev), torch.tensor(lengths, device=dev))
    at = torch.arange(T, device=dev) - _running(lengths)[run]
    inside = (starts % page)[run] + at
    slots = order[first[run] + inside // page] * page + inside % page
    if case["skipped"]:
        slots = torch.where(torch.rand(T, generator=g, device=dev) < case["skipped"], -1, slots)
    k_cache, v_cache = _cache(g, pages, Hk, D, page, case["dtype"])
    inv_freq = 10000.0 ** (-torch.arange(0, R, 2, device=dev).float() / R)
    return {"q": q, "k": k, "v": v, "k_cache": k_cache, "v_cache": v_cache, "slots": slots.int(),
            "positions": (starts[run] + at).int(), "inv_freq": inv_freq, "interleaved": case["interleaved"]}


def _counts(case):
    """Nodes of each request, on the host: the same for every seed."""
    B, n = case["batch"], case["nodes"]
    return [n - (b * 37) % n for b in range(B)] if case["ragged"] else [n] * B


def _parents(B, n, g, chain=False):
    """[B, n]: each node's parent, an earlier one; -1 for the root."""
    i = torch.arange(n, device="cuda").expand(B, n)
    if chain:
        return i - 1
    lo = (i - 6).clamp(min=0)
    p = lo + (torch.rand((B, n), generator=g, device="cuda") * (i - lo)).long()
    return torch.where(i == 0, -1, torch.minimum(p, (i - 1).clamp(min=0)))


def _closure(parents):
    """[B, n, n] bool: whether node i sees node j."""
    B, n = parents.shape
    see = torch.eye(n, dtype=torch.bool, device="cuda").repeat(B, 1, 1)
    rows = torch.arange(B, device="cuda")
    for i in range(1, n):
        see[:, i] |= see[rows, parents[:, i]]
    return see


def _words(bits):
    """[..., n] bool -> [..., ceil(n / 32)] int32."""
    n = bits.shape[-1]
    b = torch.nn.functional.pad(bits.long(), (0, -n % 32)).unflatten(-1, (-1, 32))
    return (b << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)


def _table(g, lengths, page, pages=0):
    """(block table [B, most pages], number of pages): scattered pages; -1 behind a request's last."""
    need = [(n + page - 1) // page for n in lengths]
    pages = pages or sum(need) + 3
    table = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int64, device="cuda")
    order, at = torch.randperm(pages, generator=g, device="cuda"), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table.int(), pages


def _tree_inputs(case, seed):
    g, dev = _generator(seed), "cuda"
    counts, B = _counts(case), case["batch"]
    context = torch.full((B,), case["context"], device=dev)
    if case["ragged"] and case["context"]:
        context = torch.randint(case["context"] // 8, case["context"] + 1, (B,), generator=g, device=dev)
        context[0] = case["context"]
    cu, chain = _running(counts), case["shape"] == "chain"
    table, pages = _table(g, [c + n for c, n in zip(context.tolist(), counts)], case["page"])
    q = torch.randn((sum(counts), case["heads"], case["dim"]), generator=g, device=dev).to(_DTYPES[case["dtype"]])
    k_cache, v_cache = _cache(g, pages, case["kv_heads"], case["dim"], case["page"], case["dtype"])
    visible = None
    if not chain:
        see = _closure(_parents(B, case["nodes"], g))
        live = torch.arange(case["nodes"], device=dev) < torch.tensor(counts, device=dev).unsqueeze(1)
        visible = _words(see)[live]
    return {"q": q, "k_cache": k_cache, "v_cache": v_cache, "block_table": table, "context_lens": context.int(),
            "cu_nodes": cu.int(), "max_nodes": case["nodes"], "visible": visible}


def _accept_inputs(case, seed):
    g, dev = _generator(seed), "cuda"
    counts, B, n = _counts(case), case["batch"], case["nodes"]
    parents = _parents(B, n, g)
    see = _closure(parents)
    tokens = torch.randint(500, (B, n), generator=g, device=dev)  # (few tokens: siblings share some)
    sampled = torch.randint(500, (B, n), generator=g, device=dev)
    # most nodes' sampled token is one of their children's
    child = torch.arange(n, device=dev).expand(B, n)
    hit = torch.rand((B, n), generator=g, device=dev) < case["hit"]
    last = torch.zeros((B, n), dtype=torch.int64, device=dev).scatter_reduce(1, parents.clamp(min=0), child, "amax")
    sampled = torch.where(hit & (last > 0), tokens.gather(1, last), sampled)
    live = child < torch.tensor(counts, device=dev).unsqueeze(1)
    return {"sampled": sampled[live].int(), "tokens": tokens[live].int(), "parents": parents[live].int(),
            "cu_nodes": _running(counts).int(), "max_path": n, "see": see}


def _compact_inputs(case, seed):
    g, dev = _generator(seed), "cuda"
    B, n, most, page = case["batch"], case["nodes"], case["accepted"], case["page"]
    context = torch.randint(case["context"] // 2, case["context"] + 1, (B,), generator=g, device=dev)
    accepted = torch.randint(0, most + 1, (B,), generator=g, device=dev)
    accepted[0] = most
    table, pages = _table(g, (context + n).tolist(), page, B * ((case["context"] + n + page - 1) // page))
    # each request's accepted nodes, in order, from behind where they go
    pick = torch.rand((B, n - most - 1), generator=g, device=dev).argsort(1)[:, :most].sort(1).values + most + 1
    col = torch.arange(most + 1, device=dev)
    path = torch.cat([torch.zeros((B, 1), dtype=torch.int64, device=dev), pick], 1)
    path = torch.where(col <= accepted.unsqueeze(1), path, -1)
    k_cache, v_cache = _cache(g, pages, case["kv_heads"], case["dim"], page, case["dtype"])
    return {"k_cache": k_cache, "v_cache": v_cache, "block_table": table, "context_lens": context.int(), "path": path.int()}


def _score_inputs(case, seed):
    g, dev = _generator(seed), "cuda"
    N, V = case["rows"], case["vocab"]
    logits = torch.empty((N, V), dtype=_DTYPES[case["dtype"]], device=dev)
    ids = torch.empty(N, dtype=torch.int32, device=dev)
    for i in range(0, N, 512):
        x = torch.randn((min(512, N - i), V), generator=g, device=dev).mul_(2.0)
        at = torch.randint(V, (x.shape[0], 12), generator=g, device=dev)
        x.scatter_(1, at, x.gather(1, at) + 8.0)
        logits[i:i + 512] = x
        e = -torch.log(torch.rand(x.shape, generator=g, device=dev).clamp_(2.0 ** -24, 1.0 - 2.0 ** -24))
        ids[i:i + 512] = (x - torch.log(e)).argmax(1).int()  # the tokens are drawn from the model's softmax
    if case["masked"]:
        ids = torch.where(torch.rand(N, generator=g, device=dev) < case["masked"], -1, ids)
    t = {"logits": logits, "token_ids": ids, "temperature": case["temperature"]}
    if case["op"] == "score":
        return {**t, "num_logprobs": case["top"]}
    # a mean over the rows of advantage times log-probability, and a bonus for entropy
    g_logprob = torch.randn(N, generator=g, device=dev) / N
    return {**t, "g_logprob": g_logprob, "g_entropy": torch.full((N,), -0.01 / N, device=dev)}


_INPUTS = {"append": _append_inputs, "tree": _tree_inputs, "accept": _accept_inputs, "compact": _compact_inputs,
           "score": _score_inputs, "train": _score_inputs}


def prepare(case, seed):
    t = _INPUTS[case["op"]](case, seed)
    if case["op"] == "train":
        t["logits"].requires_grad_()
    return {"op": case["op"], **t}


# ---- one pass ---------------------------------------------------------------------------------


def run(state):
    t = {k: v for k, v in state.items() if k != "op"}
    if own:
        return _run_own(state["op"], t)
    with torch.no_grad():
        return _PLAIN[state["op"]](**t)


def _run_own(op, t):
    from vllm_webgpu_amd import ops

    if op == "append":
        q = ops.append_kv(t.pop("k"), t.pop("v"), t["k_cache"], t["v_cache"], t["slots"], q=t["q"],
                          positions=t["positions"], inv_freq=t["inv_freq"], interleaved=t["interleaved"])
        return {"q": q, "k_cache": t["k_cache"], "v_cache": t["v_cache"]}
    if op == "tree":
        return {"out": ops.tree_attention(**t)}
    if op == "accept":
        r = ops.accept_tree(t["sampled"], t["tokens"], t["parents"], t["cu_nodes"], t["max_path"])
        return {"tokens": r.tokens, "path": r.path, "num_accepted": r.num_accepted}
    if op == "compact":
        ops.compact_kv(**t)
        return {"k_cache": t["k_cache"], "v_cache": t["v_cache"]}
    if op == "score":
        r = ops.token_logprobs(entropy=True, **t)
        return {"entropy": r.entropy, "ids": r.logprob_ids, "logprobs": r.logprob_vals, "ranks": r.logprob_ranks}
    g = [t.pop("g_logprob"), t.pop("g_entropy")]
    r = ops.token_logprobs(entropy=True, **t)
    grad, = torch.autograd.grad([r.logprobs, r.entropy], [t["logits"]], g)
    return {"logprobs": r.logprobs.detach(), "entropy": r.entropy.detach(), "grad": grad}


def _rotate(x, cos, sin, interleaved):
    """x [T, H, D] in 32 bits; cos and sin [T, R / 2] in 32 bits."""
    R = 2 * cos.shape[1]
    c, s = cos.unsqueeze(1), sin.unsqueeze(1)
    head = x[..., :R]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else head.chunk(2, -1)
    a, b = a * c - b * s, b * c + a * s
    head = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([head, x[..., R:]], -1)


def _plain_append(q, k, v, k_cache, v_cache, slots, positions, inv_freq, interleaved):
    angle = positions.double().unsqueeze(1) * inv_freq.double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    page = k_cache.shape[2]
    kept = slots >= 0
    at = slots[kept].long()
    k_cache[at // page, :, at % page] = _rotate(k.float(), cos, sin, interleaved)[kept].to(k.dtype)
    v_cache[at // page, :, :, at % page] = v[kept]
    return {"q": _rotate(q.float(), cos, sin, interleaved).to(q.dtype), "k_cache": k_cache, "v_cache": v_cache}


def _plain_tree(q, k_cache, v_cache, block_table, context_lens, cu_nodes, max_nodes, visible):
    dev, (T, H, D), B = q.device, q.shape, block_table.shape[0]
    Hk, page, n = k_cache.shape[1], k_cache.shape[2], max_nodes
    table = block_table.long().clamp(min=0)
    k = k_cache[table].permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D).float()
    v = v_cache[table].permute(0, 2, 1, 4, 3).reshape(B, Hk, -1, D).float()
    req = torch.searchsorted(cu_nodes.long(), torch.arange(T, device=dev), right=True) - 1
    at = torch.arange(T, device=dev) - cu_nodes.long()[req]
    qp = torch.zeros((B, n, H, D), device=dev)
    qp[req, at] = q.float()
    qp = qp.view(B, n, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    # which keys a node sees: the context, and what its words say of the tree
    key = torch.arange(k.shape[2], device=dev)
    rel = key - context_lens.long().unsqueeze(1)  # [B, S]
    if visible is None:
        see = torch.ones((n, n), dtype=torch.bool, device=dev).tril().expand(B, n, n)
    else:
        bits = (visible.unsqueeze(2) >> torch.arange(32, device=dev)).bitwise_and(1).bool().flatten(1)[:, :n]
        see = torch.zeros((B, n, n), dtype=torch.bool, device=dev)
        see[req, at] = bits
    count = (cu_nodes[1:] - cu_nodes[:-1]).long().unsqueeze(1)
    inside = (rel >= 0) & (rel < count)
    see = see.gather(2, rel.clamp(0, n - 1).unsqueeze(1).expand(B, n, -1)) & inside.unsqueeze(1)
    see = (see | (rel < 0).unsqueeze(1)).unsqueeze(1).unsqueeze(1)  # [B, 1, 1, n, S]
    s = torch.matmul(qp, k.transpose(2, 3)).mul_(D ** -0.5).view(B, Hk, H // Hk, n, -1)
    s = torch.where(see, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, 0.0)
    out = torch.matmul(p.view(B, Hk, -1, p.shape[-1]), v).view(B, H, n, D)
    return {"out": out.transpose(1, 2)[req, at].to(q.dtype)}


def _plain_accept(sampled, tokens, parents, cu_nodes, max_path, see):
    dev, T, (B, n, _) = sampled.device, sampled.shape[0], see.shape
    cu = cu_nodes.long()
    req = torch.searchsorted(cu, torch.arange(T, device=dev), right=True) - 1
    at = torch.arange(T, device=dev) - cu[req]
    pad = lambda x, v: torch.full((B, n), v, dtype=torch.int64, device=dev).index_put_((req, at), x.long())  # noqa: E731
    smp, tok, par = pad(sampled, -1), pad(tokens, -2), pad(parents, -3)
    # a node continues its parent if it holds the parent's sampled token, the first of its siblings
    fits = (tok == smp.gather(1, par.clamp(min=0))) & (par >= 0)
    twin = (par.unsqueeze(2) == par.unsqueeze(1)) & fits.unsqueeze(1)
    fits &= ~(twin & torch.ones((n, n), dtype=torch.bool, device=dev).tril(-1)).any(2)
    fits[:, 0] = True
    visited = (~see | fits.unsqueeze(1)).all(2)
    # the visited nodes in order, then -1
    node = torch.arange(n, device=dev)
    path = torch.where(visited, node, n).sort(1).values
    live = path < n
    out = smp.gather(1, path.clamp(max=n - 1))
    fill = lambda x: torch.where(live, x, -1).int()[:, :max_path]  # noqa: E731
    return {"tokens": fill(out), "path": fill(path), "num_accepted": (visited.sum(1) - 1).int()}


def _plain_compact(k_cache, v_cache, block_table, context_lens, path):
    page, table = k_cache.shape[2], block_table.long()
    b, j = torch.nonzero(path > 0, as_tuple=True)
    src, dst = context_lens.long()[b] + path.long()[b, j], context_lens.long()[b] + j
    k = k_cache[table[b, src // page], :, src % page]
    v = v_cache[table[b, src // page], :, :, src % page]
    k_cache[table[b, dst // page], :, dst % page] = k
    v_cache[table[b, dst // page], :, :, dst % page] = v
    return {"k_cache": k_cache, "v_cache": v_cache}


def _plain_logprobs(logits, token_ids, temperature):
    """(live rows, the tokens' places, log-probabilities [N, V], the tokens', entropies)."""
    live = (token_ids >= 0) & (token_ids < logits.shape[1])
    at = torch.where(live, token_ids, 0).long().unsqueeze(1)
    z = logits.float() / temperature
    z = z - z.amax(1, keepdim=True)
    z = z - torch.log(torch.exp(z).sum(1, keepdim=True))
    p = torch.exp(z)
    entropy = -torch.where(p > 0, p * z, 0.0).sum(1)
    return live, at, z, torch.where(live, z.gather(1, at).squeeze(1), 0.0), torch.where(live, entropy, 0.0)


def _plain_score(logits, token_ids, temperature, num_logprobs):
    V = logits.shape[1]
    live, at, logp, mine, entropy = _plain_logprobs(logits, token_ids, temperature)
    x = logits.float() + 0.0
    rank = torch.where(live, (x >= x.gather(1, at)).sum(1), 0)
    # value, then the lower index: both in one integer
    bits = x.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2 ** 20 + (2 ** 20 - 1 - torch.arange(V, device=x.device))
    top = 2 ** 20 - 1 - (torch.topk(key, num_logprobs, 1).values & (2 ** 20 - 1))
    ids = torch.cat([at, top], 1)
    row = live.unsqueeze(1)
    return {"entropy": entropy, "ids": torch.where(row, ids, -1).int(),
            "logprobs": torch.where(row, logp.gather(1, ids), 0.0), "ranks": rank.int()}


def _plain_train(logits, token_ids, temperature, g_logprob, g_entropy):
    live, at, logp, mine, entropy = _plain_logprobs(logits, token_ids, temperature)
    gl, ge = (torch.where(live, g, 0.0).unsqueeze(1) for g in (g_logprob, g_entropy))
    p = torch.exp(logp)
    grad = -p * (gl + ge * torch.where(p > 0, logp + entropy.unsqueeze(1), 0.0))
    grad = grad.scatter_add_(1, at, gl) / temperature
    return {"logprobs": mine, "entropy": entropy, "grad": grad.to(logits.dtype)}


_PLAIN = {"append": _plain_append, "tree": _plain_tree, "accept": _plain_accept, "compact": _plain_compact,
          "score": _plain_score, "train": _plain_train}


def work(case):
    """Bytes: inputs read once and outputs written once; of the cache what the call writes (append), moves
    (compact) or reads (tree).  Flops: two products and an exponential per key and query head; a
    rotation's six per pair; an exponential, three products and three sums per logit."""
    op, size = case["op"], 2 if case.get("dtype") != "f32" else 4
    if op == "append":
        T, H, Hk, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": 2 * T * (H + 2 * Hk) * D * size + 8 * T, "flops": 3 * T * (H + Hk) * case["rotary"]}
    if op == "tree":
        B, n, H, Hk, D = case["batch"], case["nodes"], case["heads"], case["kv_heads"], case["dim"]
        if case["ragged"]:
            n, S = (n + 1) / 2, case["context"] * 9 / 16
        else:
            S = case["context"]
        return {"bytes": int(B * (2 * (S + n) * Hk * D * size + 2 * n * H * D * size)),
                "flops": int(B * n * H * (S + n / 2) * (4 * D + 4))}
    if op == "accept":
        nodes = case["batch"] * (case["nodes"] + 1 if case["ragged"] else 2 * case["nodes"]) // 2
        return {"bytes": 12 * nodes + case["batch"] * (8 * case["nodes"] + 8), "flops": 4 * nodes}
    if op == "compact":
        moved = case["batch"] * case["accepted"] / 2 + 1
        return {"bytes": int(4 * moved * case["kv_heads"] * case["dim"] * size + case["batch"] * 4 * (case["accepted"] + 2)),
                "flops": int(moved)}
    live, V = case["rows"] * (1.0 - case["masked"]), case["vocab"]
    total = live * V * size + 12 * case["rows"]
    if op == "train":
        total += case["rows"] * V * size + 8 * case["rows"]
    else:
        total += case["rows"] * 8 * (case["top"] + 1)
    return {"bytes": int(total), "flops": int(7 * live * V * (2 if op == "train" else 1))}


# ---- the same in 64 bits ----------------------------------------------------------------------


def _exact_append(case, t):
    page, R, D = case["page"], case["rotary"], case["dim"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(t["positions"].double(), t["inv_freq"].double()))

    def turned(x):
        y = x.double().clone()
        first, second = (slice(0, R, 2), slice(1, R, 2)) if case["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn.unsqueeze(1)
        y[..., first], y[..., second] = z.real, z.imag
        return y

    kc, vc = t["k_cache"].double(), t["v_cache"].double()
    tokens = torch.nonzero(t["slots"] >= 0).squeeze(1)
    s = t["slots"][tokens].long()
    p, o = torch.div(s, page, rounding_mode="floor"), torch.remainder(s, page)
    head = torch.arange(case["kv_heads"], device="cuda")
    kc[p.unsqueeze(1), head, o.unsqueeze(1)] = turned(t["k"])[tokens]
    vc.permute(0, 1, 3, 2)[p.unsqueeze(1), head, o.unsqueeze(1)] = t["v"].double()[tokens]
    return {"q": turned(t["q"]), "k_cache": kc, "v_cache": vc}


def _exact_tree(case, t):
    page, H, Hk, D = case["page"], case["heads"], case["kv_heads"], case["dim"]
    cu, context = t["cu_nodes"].tolist(), t["context_lens"].tolist()
    out = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda")
    for b, c in enumerate(context):
        q, n = t["q"][cu[b]:cu[b + 1]], cu[b + 1] - cu[b]
        pages = t["block_table"][b, :(c + n + page - 1) // page].long()
        hidden = torch.zeros((n, c + n), dtype=torch.bool, device="cuda")
        i = torch.arange(n, device="cuda")
        if t["visible"] is None:
            hidden[:, c:] = i.unsqueeze(0) > i.unsqueeze(1)
        else:
            words = t["visible"][cu[b]:cu[b + 1]].long()
            hidden[:, c:] = (words[:, i // 32] >> (i % 32)) & 1 == 0
        for h in range(Hk):
            k = t["k_cache"][pages, h].reshape(-1, D)[:c + n].double()
            v = t["v_cache"][pages, h].transpose(1, 2).reshape(-1, D)[:c + n].double()
            mine = slice(h * (H // Hk), (h + 1) * (H // Hk))
            s = (q[:, mine].double().reshape(-1, D) @ k.T).view(n, -1, c + n) / math.sqrt(D)
            w = torch.softmax(s.masked_fill(hidden.unsqueeze(1), -math.inf), -1)
            out[cu[b]:cu[b + 1], mine] = (w.view(-1, c + n) @ v).view(n, -1, D)
    return {"out": out}


def _exact_compact(case, t):
    page = case["page"]
    kc, vc = t["k_cache"].double(), t["v_cache"].double()
    table, context = t["block_table"].tolist(), t["context_lens"].tolist()
    for b, path in enumerate(t["path"].tolist()):
        for j, node in enumerate(path):
            if node > 0:
                (p, i), (r, k) = divmod(context[b] + node, page), divmod(context[b] + j, page)
                kc[table[b][r], :, k] = t["k_cache"][table[b][p], :, i].double()
                vc[table[b][r], :, :, k] = t["v_cache"][table[b][p], :, :, i].double()
    return {"k_cache": kc, "v_cache": vc}


def exact(case, seed):
    op = case["op"]
    if op == "accept":
        return None  # whole numbers
    t = _INPUTS[op](case, seed)
    if op in ("append", "tree", "compact"):
        return {"append": _exact_append, "tree": _exact_tree, "compact": _exact_compact}[op](case, t)
    parts = {"entropy": [], "logprobs": [], "grad": []}
    for i in range(0, case["rows"], 128):
        x, ids = t["logits"][i:i + 128], t["token_ids"][i:i + 128].long()
        logp = torch.log_softmax(x.double() / case["temperature"], 1)
        dist, row = logp.exp(), (ids >= 0).unsqueeze(1)
        entropy = torch.special.entr(dist).sum(1, keepdim=True)
        parts["entropy"].append((entropy * row).squeeze(1))
        if op == "score":
            best = logp.sort(1, descending=True).values[:, :case["top"]]
            parts["logprobs"].append(torch.cat([logp.gather(1, ids.clamp(min=0).unsqueeze(1)), best], 1) * row)
            continue
        parts["logprobs"].append((logp.gather(1, ids.clamp(min=0).unsqueeze(1)) * row).squeeze(1))
        one = torch.zeros_like(dist).scatter_(1, ids.clamp(min=0).unsqueeze(1), 1.0)
        gl, ge = t["g_logprob"][i:i + 128].double().unsqueeze(1), t["g_entropy"][i:i + 128].double().unsqueeze(1)
        d = gl * (one - dist) + ge * (torch.special.entr(dist) - dist * entropy)
        parts["grad"].append(d * row / case["temperature"])
    out = {k: torch.cat(v) for k, v in parts.items() if v}
    if op == "score":
        out.update(ids=None, ranks=None)
    return out
