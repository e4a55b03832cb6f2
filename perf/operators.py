"""The work that the speculative-decoding operators' speed is measured on: verification of drafted
tokens against the target model, and the distillation loss that keeps a draft model close to it.

A case is one call on device-resident logits, as a serving or training loop makes it:

* ``op="verify"``: ``ops.verify_drafts`` on the target's logits of a batch of requests, each with
  some drafted tokens and one row more than it has drafts;
* ``op="eval"``: the forward of ``ops.distill_loss`` (a held-out batch's loss);
* ``op="train"``: its forward and, through autograd, its backward;
* ``op="step"``: ``ops.distill_loss_and_grad``, loss and gradient in one call.

With ``own`` false the same results come from elementary torch operations in 32 bits.

Vocabularies are those of the models the package's workloads are shaped after (32 000, 128 256,
151 936, 262 144), 50 257 (rows that start unaligned) and anything between.  The target's rows are
N(0, spread) plus ``spikes`` tokens lifted by ``lift``; the draft's logits are the target's plus
N(0, 0.7) noise, and drafts are drawn from its softmax, so that most are accepted, as with a useful
draft.  Teacher rows lift the K tokens that the teacher returns by a power law; the student's
logits are the teacher's plus N(0, 1) noise.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_GREEDY_T = 1e-5          # temperatures below it mean greedy
_ACCEPT_BASE = 1 << 19    # generated acceptance uniforms: token places past the largest vocabulary

_VERIFY = {"op": "verify", "batch": 1, "drafts": 4, "ragged": False, "vocab": 32000, "dtype": "bf16",
           "probs": "none", "spread": 2.0, "spikes": 12, "lift": 9.0, "temperature": 1.0, "top_k": 0,
           "top_p": 1.0, "min_p": 0.0, "mixed": False, "uniforms": "generated"}
_DISTILL = {"op": "train", "rows": 1, "vocab": 32000, "dtype": "bf16", "k": 20, "tail": "renormalize",
            "temperature": 1.0, "masked": 0.0}


def _case(base, name=None, **kw):
    c = dict(base, **kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one greedy request with three looked-up drafts on a small vocabulary: latency
        _case(_VERIFY, "verify_one_greedy", drafts=3, vocab=32000, dtype="f32", temperature=0.0),
        # one chat request at a chat model's usual settings, drafts of a draft model
        _case(_VERIFY, "verify_one_chat", drafts=5, vocab=128256, probs="bf16", temperature=0.6, top_p=0.9),
        # a batch with looked-up drafts, some requests with none, top-k
        _case(_VERIFY, "verify_48_ngram", batch=48, drafts=4, ragged=True, vocab=151936, temperature=0.8, top_k=50),
        # rollouts at temperature 1 with nothing cut, up to seven drafts, everything in fp32
        _case(_VERIFY, "verify_64_rollout", batch=64, drafts=7, ragged=True, vocab=128256, dtype="f32", probs="f32",
              uniforms="given"),
        # odd vocabulary: rows start unaligned; top-p and min-p
        _case(_VERIFY, "verify_20_odd", batch=20, drafts=3, ragged=True, vocab=50257, dtype="f32", probs="f32",
              temperature=0.9, top_p=0.95, min_p=0.02, uniforms="given"),
        # a full batch of heterogeneous requests on the largest vocabulary
        _case(_VERIFY, "verify_256_mixed", batch=256, drafts=4, ragged=True, vocab=262144, probs="bf16", mixed=True),
        # a handful of positions: the smallest training call, latency
        _case(_DISTILL, "train_4", rows=4, vocab=32000, dtype="f32", k=20),
        # held-out loss of a batch against the teacher's top 64
        _case(_DISTILL, "eval_512", op="eval", rows=512, vocab=151936, k=64, tail="bucket"),
        # a training batch with prompt positions masked out, softened targets
        _case(_DISTILL, "train_2048_masked", rows=2048, vocab=128256, k=20, temperature=2.0, masked=0.3),
        # odd vocabulary and row count in fp32, the rest of the vocabulary as one event
        _case(_DISTILL, "train_301_odd", rows=301, vocab=50257, dtype="f32", k=50, tail="bucket"),
        # few positions of the largest vocabulary, many teacher logits, half precision
        _case(_DISTILL, "step_48_f16", op="step", rows=48, vocab=262144, dtype="f16", k=256, tail="bucket"),
        # a large training step
        _case(_DISTILL, "step_4096", op="step", rows=4096, vocab=128256, k=64, tail="bucket"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    vocab = rng.choice([32000, 128256, 151936, 262144, _log_int(rng, 32000, 262144),
                        _log_int(rng, 32000, 262144) | 1])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if rng.random() < 0.5:
        drafts = rng.randint(1, 8)
        most = (1 << 27) // (vocab * (drafts + 1))
        kind = rng.choice(["greedy", "plain", "topk", "topp", "minp", "mixed"])
        some_t = round(rng.uniform(0.4, 1.2), 3)
        kw = {"greedy": {"temperature": 0.0}, "plain": {"temperature": rng.choice([1.0, some_t])},
              "topk": {"temperature": some_t, "top_k": rng.randint(5, 100), "top_p": rng.choice([1.0, 0.9])},
              "topp": {"temperature": some_t, "top_p": round(rng.uniform(0.7, 0.98), 3)},
              "minp": {"temperature": some_t, "min_p": round(rng.uniform(0.01, 0.1), 3)},
              "mixed": {"mixed": True}}[kind]
        return _case(_VERIFY, batch=max(1, min(_log_int(rng, 1, 256), most)), drafts=drafts,
                     ragged=rng.random() < 0.7, vocab=vocab, dtype=dtype, probs=rng.choice(["none", "f32", "bf16"]),
                     spikes=rng.randint(5, 40), lift=round(rng.uniform(6.0, 10.0), 2),
                     uniforms=rng.choice(["given", "generated"]), **kw)
    most = (1 << 28) // vocab
    tail = rng.choice(["renormalize", "bucket"])
    return _case(_DISTILL, op=rng.choice(["eval", "train", "step"]), rows=max(1, min(_log_int(rng, 1, 4096), most)),
                 vocab=vocab, dtype=dtype, k=_log_int(rng, 1, 256), tail=tail,
                 temperature=1.0 if tail == "bucket" else rng.choice([1.0, round(rng.uniform(0.8, 4.0), 2)]),
                 masked=rng.choice([0.0, 0.0, 0.3]))


# ---- inputs ---------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)


def _counts(case, g):
    """Drafts of each request, on the host."""
    B, n = case["batch"], case["drafts"]
    if not case["ragged"]:
        return [n] * B
    c = torch.randint(n + 1, (B,), generator=g, device="cuda").tolist()
    c[0] = n
    return c


def _verify_inputs(case, seed):
    g, dev = _generator(seed), "cuda"
    B, V, n_max = case["batch"], case["vocab"], case["drafts"]
    counts = _counts(case, g)
    D, R = sum(counts), sum(counts) + B
    rand = lambda *s: torch.rand(s, generator=g, device=dev)  # noqa: E731
    x = torch.randn((R, V), generator=g, device=dev).mul_(case["spread"])
    at = torch.randint(V, (R, case["spikes"]), generator=g, device=dev)
    x.scatter_(1, at, x.gather(1, at) + case["lift"])
    t = {"logits": x.to(_DTYPES[case["dtype"]])}
    full = lambda v, d=torch.float32: torch.full((B,), v, dtype=d, device=dev)  # noqa: E731
    if case["mixed"]:
        temp = 0.3 + rand(B)
        temp[torch.randperm(B, generator=g, device=dev)[: B // 8]] = 0.0
        ks = torch.tensor([0, 20, 50], dtype=torch.int32, device=dev)
        t["temperature"], t["top_k"] = temp, ks[torch.randint(3, (B,), generator=g, device=dev)]
        t["top_p"] = torch.where(rand(B) < 0.4, 1.0, 0.7 + 0.3 * rand(B)).float()
        t["min_p"] = torch.where(rand(B) < 0.7, 0.0, 0.05).float()
    else:
        t["temperature"] = full(case["temperature"])
        t["top_k"] = full(case["top_k"], torch.int32) if case["top_k"] else None
        t["top_p"] = full(case["top_p"]) if case["top_p"] < 1.0 else None
        t["min_p"] = full(case["min_p"]) if case["min_p"] else None
    cu = torch.tensor([0] + counts, device=dev).cumsum(0)
    of_draft = torch.repeat_interleave(torch.arange(B, device=dev), torch.tensor(counts, device=dev))
    draft_rows = torch.arange(D, device=dev) + of_draft
    # the draft model: the target's logits with noise, at the request's temperature
    temp = t["temperature"].clamp(min=0.05)[of_draft].unsqueeze(1)
    tokens, probs = torch.empty(D, dtype=torch.int32, device=dev), None
    if case["probs"] != "none":
        probs = torch.empty((D, V), dtype=_DTYPES[case["probs"]], device=dev)
    for i in range(0, D, 128):
        y = (x[draft_rows[i:i + 128]] + 0.7 * torch.randn((min(128, D - i), V), generator=g, device=dev)) / temp[i:i + 128]
        q = torch.softmax(y, 1)
        if probs is not None:
            probs[i:i + 128] = q
            q = probs[i:i + 128].float()
        e = -torch.log(torch.rand(q.shape, generator=g, device=dev).clamp_(2.0 ** -24, 1.0 - 2.0 ** -24))
        tokens[i:i + 128] = (q / e).argmax(1).int()
    del x
    t.update(draft_tokens=tokens, cu_drafts=cu.int(), max_drafts=n_max, draft_probs=probs)
    if case["uniforms"] == "given":
        # multiples of 2^-24 in (0, 1), as the generated ones are
        t["accept_uniforms"] = rand(D).clamp_(2.0 ** -24, 1.0 - 2.0 ** -24)
        t["uniforms"] = rand(B, V).clamp_(2.0 ** -24, 1.0 - 2.0 ** -24)
    else:
        t["rng_seeds"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (B,), generator=g, device=dev)
    return t


def _distill_inputs(case, seed):
    g, dev = _generator(seed), "cuda"
    N, V, K, T = case["rows"], case["vocab"], case["k"], case["temperature"]
    ids = torch.randperm(V, generator=g, device=dev)[:K].unsqueeze(0)
    ids = (ids + torch.randint(V, (N, 1), generator=g, device=dev)) % V
    lift = 12.0 - 1.5 * torch.arange(1, K + 1, device=dev).float().log()
    logits = torch.empty((N, V), dtype=_DTYPES[case["dtype"]], device=dev)
    lp = torch.empty((N, K), device=dev)
    for i in range(0, N, 512):
        x = torch.randn((min(512, N - i), V), generator=g, device=dev)
        at = ids[i:i + 512]
        x.scatter_(1, at, x.gather(1, at) + lift)
        lp[i:i + 512] = x.gather(1, at) - torch.logsumexp(x, 1, keepdim=True)
        logits[i:i + 512] = x.add_(torch.randn(x.shape, generator=g, device=dev))
    weight = None
    if case["masked"]:
        weight = (torch.rand(N, generator=g, device=dev) >= case["masked"]).float()
    valid = float(N) if weight is None else weight.sum().clamp(min=1.0)
    grad_out = torch.ones(N, device=dev) / valid  # a mean over the rows that count
    return {"logits": logits, "teacher_ids": ids.int().contiguous(), "teacher_logprobs": lp, "row_weight": weight,
            "temperature": T, "tail": case["tail"], "grad_output": grad_out}


def prepare(case, seed):
    if case["op"] == "verify":
        return {"op": "verify", **_verify_inputs(case, seed)}
    t = _distill_inputs(case, seed)
    t["logits"].requires_grad_(case["op"] == "train")
    return {"op": case["op"], **t}


# ---- one pass ---------------------------------------------------------------------------------


def run(state):
    t = {k: v for k, v in state.items() if k != "op"}
    if own:
        return _run_own(state["op"], t)
    if state["op"] == "verify":
        return _plain_verify(**t)
    with torch.no_grad():
        return _plain_distill(state["op"], **t)


def _run_own(op, t):
    from vllm_webgpu_amd import ops

    if op == "verify":
        r = ops.verify_drafts(t.pop("logits"), t.pop("draft_tokens"), t.pop("cu_drafts"), t.pop("max_drafts"), **t)
        return {"tokens": r.tokens, "num_accepted": r.num_accepted, "logprobs": r.logprobs}
    g = t.pop("grad_output")
    args = t.pop("logits"), t.pop("teacher_ids"), t.pop("teacher_logprobs")
    if op == "eval":
        return {"loss": ops.distill_loss(*args, **t)}
    if op == "step":
        loss, grad = ops.distill_loss_and_grad(*args, grad_output=g, **t)
        return {"loss": loss, "grad": grad}
    loss = ops.distill_loss(*args, **t)
    return {"loss": loss.detach(), "grad": torch.autograd.grad(loss, args[0], g)[0]}


def _philox_uniforms(seeds, tokens):
    """[B, n] uniforms of the tokens [n] (or [B, n]) under the 64-bit keys [B]: word t % 4 of
    Philox-4x32-10 at counter (t / 4, 0, 0, 0), as (2 floor(w / 2^9) + 1) 2^-24."""
    mask = 0xFFFFFFFF
    k0, k1 = (seeds & mask).unsqueeze(1), ((seeds >> 32) & mask).unsqueeze(1)
    c0 = (tokens >> 2) + torch.zeros_like(k0)
    c1, c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0), torch.zeros_like(c0)
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & mask) ^ c1 ^ k0, p1 & mask, ((p0 >> 32) & mask) ^ c3 ^ k1, p0 & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    j = tokens & 3
    w = torch.where(j == 0, c0, torch.where(j == 1, c1, torch.where(j == 2, c2, c3)))
    return (2 * (w >> 9) + 1).float() * 2.0 ** -24


def _plain_verify(logits, draft_tokens, cu_drafts, max_drafts, draft_probs=None, temperature=None, top_k=None,
                  top_p=None, min_p=None, accept_uniforms=None, uniforms=None, rng_seeds=None):
    dev, (R, V) = logits.device, logits.shape
    B, D = cu_drafts.numel() - 1, draft_tokens.numel()
    cu, drafts = cu_drafts.long(), draft_tokens.long()
    count = cu[1:] - cu[:-1]
    req = torch.searchsorted(cu + torch.arange(B + 1, device=dev), torch.arange(R, device=dev), right=True) - 1
    req_d = torch.searchsorted(cu, torch.arange(D, device=dev), right=True) - 1
    pos_d = torch.arange(D, device=dev) - cu[req_d]
    rows_d = torch.arange(D, device=dev) + req_d
    # the target's distribution, row by row
    greedy = temperature < _GREEDY_T
    y = logits.float() / torch.where(greedy, 1.0, temperature)[req].unsqueeze(1)
    m, top = y.max(1, keepdim=True)
    e = torch.exp(y - m)
    if min_p is not None:
        e = torch.where(y - m >= torch.log(min_p)[req].unsqueeze(1), e, 0.0)
    if top_k is not None or top_p is not None:
        ys, order = y.sort(dim=1, stable=True)  # ascending, the lower index first
        if top_k is not None:
            k = torch.where((top_k <= 0) | (top_k >= V), V, top_k)[req].long()
            e = torch.where(y >= ys.gather(1, (V - k).unsqueeze(1)), e, 0.0)
        if top_p is not None:
            c = e.gather(1, order).cumsum(1)
            gone = c <= (1.0 - top_p)[req].unsqueeze(1) * c[:, -1:]
            gone &= (top_p < 1.0)[req].unsqueeze(1)
            gone[:, -1] = False
            e = torch.where(torch.zeros_like(gone).scatter_(1, order, gone), 0.0, e)
        del ys, order
    p = e / e.sum(1, keepdim=True)
    # acceptance, in order, up to the first refusal
    if accept_uniforms is None:
        places = _ACCEPT_BASE + torch.arange(max_drafts, device=dev)
        accept_uniforms = _philox_uniforms(rng_seeds, places)[req_d, pos_d]
    p_d = p[rows_d, drafts]
    q_d = 1.0 if draft_probs is None else draft_probs[torch.arange(D, device=dev), drafts].float()
    ok = (accept_uniforms * q_d < p_d) & (torch.as_tensor(q_d, device=dev) > 0)
    ok = torch.where(greedy[req_d], drafts == top[rows_d, 0], ok)
    run_of = torch.zeros((B, max_drafts + 1), dtype=torch.int32, device=dev)
    run_of[req_d, pos_d] = ok.int()
    accepted = run_of.cumprod(1).sum(1)
    # one more token: of the residual after a refusal, of the target's row after the last draft
    row = cu[:-1] + torch.arange(B, device=dev) + accepted
    w = p[row]
    refused = (accepted < count).unsqueeze(1)
    if D:
        at = (cu[:-1] + accepted).clamp(max=D - 1)
        if draft_probs is None:
            w = torch.where(refused, w.scatter(1, drafts[at].unsqueeze(1), 0.0), w)
        else:
            w = torch.where(refused, (w - draft_probs[at].float()).clamp(min=0.0), w)
    u = uniforms if uniforms is not None else _philox_uniforms(rng_seeds, torch.arange(V, device=dev))
    key, token = (w / -torch.log(u)).max(1)
    token = torch.where(greedy | ~(key > 0), top[row, 0], token)
    # outputs
    pad = torch.full((B, max_drafts + 1), -1, dtype=torch.int64, device=dev)
    tokens = pad.clone()
    keep_d = pos_d < accepted[req_d]
    tokens[req_d, pos_d] = torch.where(keep_d, drafts, -1)
    tokens.scatter_(1, accepted.unsqueeze(1), token.unsqueeze(1))
    col = torch.arange(max_drafts + 1, device=dev)
    rows = (cu[:-1] + torch.arange(B, device=dev)).unsqueeze(1) + torch.minimum(col, count.unsqueeze(1))
    lp = torch.log(p[rows, tokens.clamp(min=0)])
    lp = torch.where((tokens < 0) | greedy.unsqueeze(1), 0.0, lp)
    return {"tokens": tokens.int(), "num_accepted": accepted.int(), "logprobs": lp}


def _plain_distill(op, logits, teacher_ids, teacher_logprobs, row_weight, temperature, tail, grad_output):
    ids = teacher_ids.long()
    z = logits.float() / temperature
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    logq = z.gather(1, ids) - m - torch.log(total)
    w = torch.ones_like(total) if row_weight is None else row_weight.unsqueeze(1)
    if tail == "renormalize":
        lp = teacher_logprobs / temperature
        lp = lp - lp.amax(1, keepdim=True)
        lp = lp - torch.log(torch.exp(lp).sum(1, keepdim=True))
        loss = (torch.exp(lp) * (lp - logq)).sum(1, keepdim=True)
    else:
        lp = teacher_logprobs
        r = (1.0 - torch.exp(lp).sum(1, keepdim=True)).clamp(min=0.0)
        s = e.scatter(1, ids, 0.0).sum(1, keepdim=True) / total
        loss = (torch.exp(lp) * (lp - logq)).sum(1, keepdim=True) + torch.where(r > 0, r * torch.log(r / s), 0.0)
    out = {"loss": (w * loss).squeeze(1)}
    if op == "eval":
        return out
    scale = w * grad_output.unsqueeze(1) / temperature
    q = e / total
    if tail == "renormalize":
        g = q.scatter_add(1, ids, -torch.exp(lp))
    else:
        g = (q * (1.0 - r / s)).scatter(1, ids, q.gather(1, ids) - torch.exp(lp))
    out["grad"] = (g * scale).to(logits.dtype)
    return out


def work(case):
    """Bytes: every target row, student row and teacher entry read once, outputs and gradients
    written once; of the draft's distribution and of given uniforms one row a request (where
    nothing is cut: only kept tokens need them), of the rest of the draft's rows one value each.
    Flops: an exponential, a product and two sums per logit."""
    V, size = case["vocab"], 4 if case["dtype"] == "f32" else 2
    if case["op"] != "verify":
        N, K = case["rows"], case["k"]
        live = N * (1.0 - case["masked"])
        total = live * V * size + 8 * N * K + 8 * N
        if case["op"] != "eval":
            total += N * V * size  # the gradient, masked rows' zeros among it
        return {"bytes": int(total), "flops": int(4 * live * V)}
    B, n = case["batch"], case["drafts"]
    D = B * n if not case["ragged"] else n + (B - 1) * n // 2
    total = (D + B) * V * size + 8 * D + 16 * B + B * (n + 1) * 8
    if case["temperature"] >= _GREEDY_T and not (case["top_k"] or case["top_p"] < 1.0 or case["min_p"] or case["mixed"]):
        total += 4 * B * V if case["uniforms"] == "given" else 0
        total += 0 if case["probs"] == "none" else B * V * (4 if case["probs"] == "f32" else 2)
    return {"bytes": int(total), "flops": int(4 * (D + B) * V)}


# ---- the same in 64 bits ----------------------------------------------------------------------


def _race_uniforms(seed, first, count, dev):
    """As float64: the generated uniforms of `count` tokens from `first` (a multiple of 4)."""
    lo, hi = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    block = torch.arange((count + 3) // 4, device=dev, dtype=torch.int64) + first // 4
    zero = torch.zeros_like(block)
    x = [block, zero, zero, zero]
    for r in range(10):
        a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        ka, kb = (lo + r * 0x9E3779B9) & 0xFFFFFFFF, (hi + r * 0xBB67AE85) & 0xFFFFFFFF
        x = [((b >> 32) & 0xFFFFFFFF) ^ x[1] ^ ka, b & 0xFFFFFFFF, ((a >> 32) & 0xFFFFFFFF) ^ x[3] ^ kb, a & 0xFFFFFFFF]
    words = torch.stack(x, 1).reshape(-1)[:count]
    return ((words // 512) * 2 + 1).double() / 2 ** 24


def _exact_row(x, T, k, p, min_p):
    """The kept tokens' probabilities of one row, in float64 ([V])."""
    y = x.double() / T
    V = y.numel()
    prob = torch.softmax(y, 0)
    if min_p > 0:
        prob = prob * (y >= y.max() + math.log(min_p))
    if 0 < k < V:
        prob = prob * (y >= torch.topk(y, k).values[-1])
    prob = prob / prob.sum()
    if p < 1.0:
        down = torch.flip(torch.sort(y, stable=True).indices, [0])  # most probable first, the higher index first
        above = torch.cumsum(prob[down], 0) - prob[down]            # mass before each
        stay = above < p
        stay[0] = True
        prob = prob * torch.zeros(V, dtype=torch.bool, device=y.device).scatter_(0, down, stay)
        prob = prob / prob.sum()
    return prob


def _exact_verify(case, t):
    B, V = case["batch"], case["vocab"]
    dev = t["logits"].device
    host = {k: (v.tolist() if v is not None else None)
            for k, v in ((k, t.get(k)) for k in ("temperature", "top_k", "top_p", "min_p", "draft_tokens",
                                                 "cu_drafts", "accept_uniforms", "rng_seeds"))}
    one = lambda name, b, off: off if host[name] is None else host[name][b]  # noqa: E731
    logp = torch.zeros((B, case["drafts"] + 1), dtype=torch.float64)
    for b in range(B):
        T = host["temperature"][b]
        if T < _GREEDY_T:
            continue  # a sure token: log 1
        first, n = host["cu_drafts"][b], host["cu_drafts"][b + 1] - host["cu_drafts"][b]
        for i in range(n + 1):
            prob = _exact_row(t["logits"][first + b + i], T, one("top_k", b, 0), one("top_p", b, 1.0),
                              one("min_p", b, 0.0))
            weight = prob
            if i < n:
                d = host["draft_tokens"][first + i]
                u = (host["accept_uniforms"][first + i] if host["accept_uniforms"] is not None else
                     float(_race_uniforms(host["rng_seeds"][b], _ACCEPT_BASE, i + 1, dev)[i]))
                q = None if t["draft_probs"] is None else t["draft_probs"][first + i].double()
                q_d = 1.0 if q is None else float(q[d])
                if q_d > 0 and u * q_d < float(prob[d]):
                    logp[b, i] = math.log(float(prob[d]))
                    continue
                if q is None:
                    weight = prob.clone()
                    weight[d] = 0.0
                else:
                    weight = (prob - q).clamp(min=0.0)
            u = t["uniforms"][b].double() if t.get("uniforms") is not None else _race_uniforms(host["rng_seeds"][b], 0, V, dev)
            logp[b, i] = torch.log(prob[(weight / -torch.log(u)).argmax()]).cpu()
            break
    return {"tokens": None, "num_accepted": None, "logprobs": logp}


def exact(case, seed):
    if case["op"] == "verify":
        return _exact_verify(case, _verify_inputs(case, seed))
    t = _distill_inputs(case, seed)
    T, bucket = case["temperature"], case["tail"] == "bucket"
    losses, grads = [], []
    for i in range(0, case["rows"], 128):
        part = slice(i, i + 128)
        ids = t["teacher_ids"][part].long()
        logq = torch.log_softmax(t["logits"][part].double() / T, 1)
        lp = t["teacher_logprobs"][part].double()
        if not bucket:
            lp = torch.log_softmax(lp / T, 1)
        tp = lp.exp()
        loss = (tp * (lp - logq.gather(1, ids))).sum(1)
        g = logq.exp()
        if bucket:
            mine = g.gather(1, ids)
            rest, s = 1.0 - tp.sum(1), g.scatter(1, ids, 0.0).sum(1)
            loss = loss + torch.where(rest > 0, rest * torch.log(rest.clamp(min=1e-300) / s), 0.0)
            g = (g * (1.0 - rest.clamp(min=0.0) / s).unsqueeze(1)).scatter(1, ids, mine - tp)
        else:
            g.scatter_add_(1, ids, -tp)
        w = 1.0 if t["row_weight"] is None else t["row_weight"][part].double()
        losses.append(w * loss)
        if case["op"] != "eval":
            grads.append(g * (w * t["grad_output"][part].double() / T).unsqueeze(1))
    out = {"loss": torch.cat(losses)}
    if grads:
        out["grad"] = torch.cat(grads)
    return out
