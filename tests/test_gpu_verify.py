"""Draft verification (``ops.verify_drafts``) on the GPU against a plain 64-bit reference, against the
sampler itself, and by the distribution of what it emits.

Tokens and counts must match wherever the reference can tell: a request is left out when one of its
decisions lies within the arithmetic's error (32-bit exponentials, sums and logarithms, each within
a few 2^-24: acceptance within 1e-5 of equality, two race keys within 1e-5 and what a cancelled
residual loses).  Log probabilities: y - m rounds to
2^-24 |y - m| (|y - m| <= 40 here, 2.4e-6), the logarithm of the sum to 2^-24 of 13, the sum itself to
2e-6: 1e-5 in all."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import speculative_ref as R
from vllm_webgpu_amd import _lib, ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LP_TOL = 1e-5


def make(cuda, counts, V, dtype="f32", probs=None, seed=0, spread=2.5, noise=0.7, T=1.0, spikes=4):
    """Logits, drafts drawn from a noisy copy's softmax, and uniforms, as device tensors."""
    g = torch.Generator().manual_seed(seed)
    B, D = len(counts), sum(counts)
    x = torch.randn((D + B, V), generator=g) * spread
    x[torch.arange(D + B).unsqueeze(1), torch.randint(V, (D + B, spikes), generator=g)] += 6.0
    x = x.to(DT[dtype])
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    rows = torch.tensor([cu[b] + b + i for b in range(B) for i in range(counts[b])], dtype=torch.long)
    t = torch.as_tensor(T, dtype=torch.float32).expand(B)
    per = torch.tensor([float(t[b]) for b in range(B) for _ in range(counts[b])]).clamp(min=0.05).reshape(-1, 1)
    q = torch.softmax((x[rows].float() + noise * torch.randn((D, V), generator=g)) / per, 1) if D else torch.zeros((0, V))
    if probs:
        q = q.to(DT[probs])
    drafts = (q.float() / -torch.log(torch.rand((D, V), generator=g).clamp(1e-7, 1 - 1e-7))).argmax(1).int() if D else torch.zeros(0, dtype=torch.int32)
    au = torch.rand(D, generator=g).clamp(2.0 ** -24, 1 - 2.0 ** -24)
    u = torch.rand((B, V), generator=g).clamp(2.0 ** -24, 1 - 2.0 ** -24)
    return dict(logits=x.to(cuda), draft_tokens=drafts.to(cuda), cu_drafts=torch.from_numpy(cu).to(cuda),
                draft_probs=q.to(cuda) if probs else None, accept_uniforms=au.to(cuda), uniforms=u.to(cuda))


def full(v, B, dt):
    return np.full(B, v, dt) if np.isscalar(v) else np.asarray(v, dt)


def check(t, K, T=1.0, k=0, p=1.0, min_p=0.0, max_near=0.1):
    B = t["cu_drafts"].numel() - 1
    T, k, p, min_p = full(T, B, np.float32), full(k, B, np.int32), full(p, B, np.float32), full(min_p, B, np.float32)
    r = ops.verify_drafts(max_drafts=K, temperature=torch.from_numpy(T),
                          top_k=torch.from_numpy(k) if k.any() else None,
                          top_p=torch.from_numpy(p) if (p < 1).any() else None,
                          min_p=torch.from_numpy(min_p) if min_p.any() else None, **t)
    torch.cuda.synchronize()
    h = {a: (None if v is None else v.float().cpu().numpy() if v.is_floating_point() else v.cpu().numpy()) for a, v in t.items()}
    tok, acc, lp, near = R.verify(h["logits"], h["draft_tokens"], h["cu_drafts"], K, h["draft_probs"], T, k, p, min_p,
                                  h["accept_uniforms"], h["uniforms"])
    ok = ~near
    assert near.mean() <= max_near, f"{near.sum()} of {B} requests too close to call"
    np.testing.assert_array_equal(r.num_accepted.cpu().numpy()[ok], acc[ok])
    np.testing.assert_array_equal(r.tokens.cpu().numpy()[ok], tok[ok])
    np.testing.assert_allclose(r.logprobs.cpu().numpy()[ok], lp[ok], rtol=0, atol=LP_TOL)
    return r, acc[ok]


RAGGED = [3, 0, 1, 5, 2, 0, 4, 5, 1, 3, 2, 5]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("probs", [None, "f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [997, 32000, 50257])
def test_types_and_vocabularies(cuda, dtype, probs, V):
    _, acc = check(make(cuda, RAGGED, V, dtype, probs, seed=V + 1, T=0.9), 5, T=0.9)
    assert acc.min() == 0 and (probs is None or acc.max() >= 1)  # (looked-up drafts are mostly refused here)


@pytest.mark.parametrize("V", [1, 2, 3, 4, 7, 8, 9, 63, 65, 255, 257, 1023, 4095, 4096, 4097, 8191, 16385])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_odd_vocabularies(cuda, V, dtype):
    check(make(cuda, [2, 0, 3, 1], V, dtype, "f32", seed=V, spikes=1), 3, max_near=0.5 if V < 4 else 0.25)


@pytest.mark.parametrize("cut", [dict(k=1), dict(k=50), dict(k=700), dict(p=0.9), dict(p=0.3), dict(p=0.0), dict(p=0.999),
                                 dict(min_p=0.05), dict(min_p=1.0), dict(k=20, p=0.8), dict(k=40, p=0.95, min_p=0.02),
                                 dict(k=5000, p=0.97)])
@pytest.mark.parametrize("dtype,probs", [("f32", "f32"), ("bf16", "bf16"), ("bf16", None)])
def test_cuts(cuda, cut, dtype, probs):
    check(make(cuda, RAGGED, 12345, dtype, probs, seed=11, T=0.8, spread=2.0), 5, T=0.8, max_near=0.5, **cut)


def test_mixed_requests(cuda):
    rng = np.random.default_rng(5)
    B = 24
    T = np.where(rng.random(B) < 0.2, 0.0, rng.uniform(0.4, 1.3, B)).astype(np.float32)
    k = rng.choice([0, 0, 20, 100], B).astype(np.int32)
    p = np.where(rng.random(B) < 0.4, 1.0, rng.uniform(0.6, 0.99, B)).astype(np.float32)
    mp = np.where(rng.random(B) < 0.6, 0.0, 0.05).astype(np.float32)
    t = make(cuda, list(rng.integers(0, 6, B)), 20011, "bf16", "f32", seed=6, T=T)
    check(t, 5, T=T, k=k, p=p, min_p=mp, max_near=0.3)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_greedy(cuda, dtype):
    """Accepted while the draft is the row's argmax, the lowest index among equal logits."""
    t = make(cuda, [4, 4, 0, 2], 5003, dtype, seed=3)
    x = t["logits"]
    x[0, 4000] = x[0, 17] = x[0].max() + 1          # a tie: 17 is the argmax
    x[5, 4000] = x[5, 17] = x[5].max() + 1
    best = x.float().argmax(1).int()
    d = t["draft_tokens"]
    d[:4] = torch.stack([torch.tensor(17, device=cuda, dtype=torch.int32), best[1], best[2], best[3]])
    d[4:8] = torch.stack([torch.tensor(4000, device=cuda, dtype=torch.int32), best[6], best[7], best[8]])
    r, acc = check(t, 4, T=0.0)
    assert list(acc[:2]) == [4, 0] and int(r.tokens[1, 0]) == 17
    none = ops.verify_drafts(x, d, t["cu_drafts"], 4)  # no temperature: greedy, no random numbers needed
    assert torch.equal(none.tokens, r.tokens) and torch.equal(none.num_accepted, r.num_accepted)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_without_a_finite_maximum_and_nan(cuda, dtype):
    inf = float("inf")
    t = make(cuda, [1, 1, 1, 1, 2, 1], 3001, dtype, seed=9)
    x, d, lo = t["logits"], t["draft_tokens"], torch.finfo(DT[dtype]).min
    x[0] = -inf                      # nothing left: the first index
    d[0] = 0
    x[1] = float("nan")
    x[2, 100] = x[2, 900] = inf      # a sure token
    d[1] = 100
    x[4, ::2] = float("nan")         # NaN never wins and has no mass
    x[6] = lo                        # masks of the type's lowest value
    x[6, 7] = 1.0
    d[3] = 7
    x[8, 5:] = -inf
    x[9, 1:] = lo
    x[9, 2000] = -inf
    check(t, 2, T=1.0, max_near=0.5)
    check(t, 2, T=1.0, p=0.9, k=5, max_near=0.5)
    check(t, 2, T=0.0)


def test_all_logits_equal(cuda):
    """Every mass equal: the cut is decided by the index alone."""
    t = make(cuda, [2, 1, 0], 9001, "bf16", "f32", seed=4)
    t["logits"][:] = 1.5
    check(t, 2, T=1.0, p=0.75, max_near=0.7)
    check(t, 2, T=1.0, k=3)
    check(t, 2, T=1.0, p=0.0)
    check(t, 2)


def test_drafts_outside_the_vocabulary_are_refused(cuda):
    t = make(cuda, [2, 2, 2], 4001, "f32", "f32", seed=5)
    t["draft_tokens"][:] = torch.tensor([-1, 5, 4001, 5, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    r, acc = check(t, 2, T=1.0)
    t["draft_probs"] = None
    check(t, 2, T=1.0)
    assert int(acc.max()) == 0


def test_a_draft_its_distribution_gives_no_mass_is_refused(cuda):
    t = make(cuda, [1] * 8, 501, "f32", "f32", seed=6)
    t["draft_probs"][torch.arange(8), t["draft_tokens"].long()] = 0.0
    r, acc = check(t, 1, T=1.0)
    assert int(acc.max()) == 0


def test_an_empty_residual_gives_the_most_probable_token(cuda):
    t = make(cuda, [1] * 6, 700, "f32", "f32", seed=7)
    t["draft_probs"][:] = 1.0
    t["accept_uniforms"][:] = 1.0 - 2.0 ** -24
    r, _ = check(t, 1, T=1.0)
    bad = (r.num_accepted == 0).cpu()
    assert bad.any()
    assert torch.equal(r.tokens[:, 0].cpu()[bad], t["logits"].cpu()[::2].argmax(1).int()[bad])


def test_a_perfect_draft_is_always_accepted(cuda):
    t = make(cuda, [5] * 10, 3000, "f32", "f32", seed=8, noise=0.0)
    t["draft_probs"] *= 1.0 - 1e-5
    r, _ = check(t, 5, T=1.0)
    assert int(r.num_accepted.min()) == 5


@pytest.mark.parametrize("dtype,V", [("f32", 32000), ("bf16", 50257), ("f16", 4099)])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.92), dict(min_p=0.05), dict(top_p=0.8, min_p=0.01)])
@pytest.mark.parametrize("rng", ["uniforms", "seeds", "key"])
def test_without_drafts_it_is_the_sampler(cuda, dtype, V, kw, rng):
    """One row per request and no draft: the same token as ``ops.sample``, bit for bit."""
    B = 37
    t = make(cuda, [0] * B, V, dtype, seed=12)
    T = torch.linspace(0.0, 1.4, B)
    r = {"uniforms": dict(uniforms=t["uniforms"]), "seeds": dict(rng_seeds=torch.arange(B) * 977 - 5, rng_offsets=torch.arange(B) * 3),
         "key": dict(rng_key=0x1234567890ABCDEF)}[rng]
    want = ops.sample(t["logits"], temperature=T, **kw, **r)
    more = dict(accept_uniforms=t["accept_uniforms"]) if rng == "uniforms" else {}
    got = ops.verify_drafts(t["logits"], t["draft_tokens"], t["cu_drafts"], 0, temperature=T, **kw, **r, **more)
    assert torch.equal(got.tokens[:, 0], want.sampled)
    assert int(got.num_accepted.abs().max()) == 0


def test_the_kept_set_is_the_samplers(cuda):
    """The kept sum, read off the logprobs, against the sampler's count of kept tokens on rows whose
    kept tokens are equally probable: log p = -log(count)."""
    V, B = 6007, 16
    g = torch.Generator().manual_seed(1)
    x = torch.full((B, V), -30.0)
    for b in range(B):
        x[b, torch.randperm(V, generator=g)[:200 + 13 * b]] = 2.0
    x = x.to(torch.bfloat16).to(cuda)
    u = torch.rand((B, V), generator=g).clamp(1e-6, 1 - 1e-6).to(cuda)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=cuda)
    for kw in (dict(top_p=0.9), dict(top_p=0.35), dict(top_k=7, top_p=0.5), dict(top_k=7)):
        want = ops.sample(x, temperature=0.7, uniforms=u, **kw)
        got = ops.verify_drafts(x, torch.zeros(0, dtype=torch.int32), cu, 0, temperature=0.7, uniforms=u,
                                accept_uniforms=torch.zeros(0), **kw)
        assert torch.equal(got.tokens[:, 0], want.sampled)
        n = torch.exp(-got.logprobs[:, 0].double())
        assert torch.allclose(n, want.num_kept.double(), rtol=1e-5, atol=0), kw


def test_generated_numbers_are_the_uniforms_of_the_same_key(cuda):
    """Seeds against the same numbers passed as uniforms."""
    from oracle import sampler as O

    counts, V = [3, 0, 2, 4], 2003
    t = make(cuda, counts, V, "f32", "f32", seed=13)
    seeds = np.array([3, 2 ** 63 + 9, 12345678901234567, 0], np.uint64)
    u = O.philox_uniforms(seeds, V).astype(np.float32)
    at = np.arange(8, dtype=np.int64) + 2 ** 19
    au = []
    for b, n in enumerate(counts):
        wide = _philox(int(seeds[b]), at)
        au += list(wide[:n])
    t["uniforms"], t["accept_uniforms"] = torch.from_numpy(u).to(cuda), torch.tensor(au, dtype=torch.float32, device=cuda)
    want, _ = check(t, 4)
    del t["uniforms"], t["accept_uniforms"]
    got = ops.verify_drafts(max_drafts=4, temperature=1.0, rng_seeds=torch.from_numpy(seeds.view(np.int64)), **t)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.logprobs, want.logprobs)


def _philox(seed, tokens):
    out = []
    for t in tokens:
        c, k0, k1 = [int(t) >> 2, 0, 0, 0], seed & 0xFFFFFFFF, seed >> 32
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k0, b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k1, a & 0xFFFFFFFF]
            k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
        out.append((2 * (c[int(t) & 3] >> 9) + 1) * 2.0 ** -24)
    return out


@pytest.mark.parametrize("with_probs", [False, True])
def test_emitted_tokens_are_distributed_as_the_targets(cuda, with_probs):
    """The first emitted token of many requests with one set of logits: frequencies within five
    standard deviations of p, whatever the drafts' distribution."""
    B, V = 60000, 12
    g = torch.Generator().manual_seed(21)
    x = torch.randn((1, V), generator=g) * 1.5
    p = torch.softmax(x[0].double(), 0)
    q = torch.softmax(torch.randn(V, generator=g) * 1.5, 0)
    drafts = torch.multinomial(q, B, replacement=True, generator=g).int().to(cuda)
    cu = torch.arange(B + 1, dtype=torch.int32, device=cuda)
    r = ops.verify_drafts(x.expand(2 * B, V).contiguous().to(cuda), drafts, cu, 1,
                          draft_probs=q.expand(B, V).contiguous().to(cuda) if with_probs else None, temperature=1.0, rng_key=77)
    f = torch.bincount(r.tokens[:, 0].cpu().long(), minlength=V).double() / B
    assert ((f - p).abs() <= 5 * torch.sqrt(p * (1 - p) / B) + 1e-9).all(), (f, p)
    both = r.tokens[r.num_accepted.bool()][:, 1].cpu().long()  # the bonus token, after an acceptance
    f = torch.bincount(both, minlength=V).double() / both.numel()
    assert ((f - p).abs() <= 5 * torch.sqrt(p * (1 - p) / both.numel()) + 1e-9).all()


def test_many_drafts(cuda):
    t = make(cuda, [64, 0, 33], 1009, "bf16", "bf16", seed=14, noise=0.05)
    r, acc = check(t, 64, max_near=0.7)
    assert r.tokens.shape == (3, 65)


def test_strides_and_alignment(cuda):
    t = make(cuda, RAGGED, 4111, "bf16", "bf16", seed=15)
    want = ops.verify_drafts(max_drafts=5, temperature=0.9, top_p=0.9, **t)
    plain = ops.verify_drafts(max_drafts=5, temperature=0.9, **t)
    for off in (1, 3, 8):
        s = dict(t)
        for name in ("logits", "draft_probs", "uniforms"):
            wide = torch.full((t[name].shape[0], 4111 + 19), float("nan"), dtype=t[name].dtype, device=cuda)
            wide[:, off:off + 4111] = t[name]
            s[name] = wide[:, off:off + 4111]
        for kw, ref in ((dict(top_p=0.9), want), ({}, plain)):
            r = ops.verify_drafts(max_drafts=5, temperature=0.9, **kw, **s)
            assert torch.equal(r.tokens, ref.tokens) and torch.equal(r.num_accepted, ref.num_accepted)
            assert torch.allclose(r.logprobs, ref.logprobs, rtol=0, atol=LP_TOL)
    s = dict(t, logits=t["logits"].t().contiguous().t(), draft_tokens=t["draft_tokens"].long(), cu_drafts=t["cu_drafts"].cpu())
    r = ops.verify_drafts(max_drafts=5, temperature=0.9, **s)
    assert torch.equal(r.tokens, plain.tokens)


def test_largest_vocabulary_and_rows_past_32_bits(cuda):
    V, D = 1 << 19, 4200           # 4201 rows x 2^19: element offsets past 2^31
    x = torch.full((D + 1, V), -9.0, dtype=torch.bfloat16, device=cuda)
    want = (torch.arange(D + 1, device=cuda) * 7919 + V - 40000) % V
    x[torch.arange(D + 1, device=cuda), want] = 5.0
    drafts = want[:D].int()
    cu = torch.tensor([0] + list(range(60, D + 1, 60)), dtype=torch.int32, device=cuda)
    B = cu.numel() - 1
    rows = torch.cat([want, want[-1:].expand(B - 1)])
    del x
    x = torch.full((D + B, V), -9.0, dtype=torch.bfloat16, device=cuda)
    req = torch.arange(D, device=cuda) // 60
    x[torch.arange(D, device=cuda) + req, drafts.long()] = 5.0
    x[cu[1:].long() + torch.arange(B, device=cuda), 3] = 5.0
    r = ops.verify_drafts(x, drafts, cu, 60)
    assert bool((r.num_accepted == 60).all())
    assert torch.equal(r.tokens[:, :60].reshape(-1), drafts) and bool((r.tokens[:, 60] == 3).all())
    assert rows.numel() == D + B


def test_bounds_that_do_not_fit_give_no_token(cuda):
    t = make(cuda, [2, 2, 2], 800, "f32", "f32", seed=16)
    good = ops.verify_drafts(max_drafts=2, temperature=1.0, **t)
    for cu in ([0, 2, 1, 6], [0, 4, 4, 6], [0, 2, 4, 99], [-3, 2, 4, 6], [0, 2 ** 31 - 1, 4, 6], [9, 9, 9, 9],
               [0, -2 ** 31, 4, 6]):
        r = ops.verify_drafts(max_drafts=2, temperature=1.0, **dict(t, cu_drafts=torch.tensor(cu, dtype=torch.int32)))
        torch.cuda.synchronize()
        acc = r.num_accepted.cpu()
        assert bool((acc >= -1).all()) and bool((acc == -1).any())
        assert bool((r.tokens.cpu()[acc == -1] == -1).all())
    again = ops.verify_drafts(max_drafts=2, temperature=1.0, **t)
    assert torch.equal(again.tokens, good.tokens)


def test_no_requests(cuda):
    r = ops.verify_drafts(torch.empty((0, 100), device=cuda), torch.empty(0, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 3)
    assert r.tokens.shape == (0, 4) and r.num_accepted.shape == (0,)


def test_same_answer_each_time_and_on_another_stream(cuda):
    t = make(cuda, RAGGED * 3, 40009, "bf16", "f32", seed=17)
    want = ops.verify_drafts(max_drafts=5, temperature=0.8, top_p=0.95, **t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            got.append(ops.verify_drafts(max_drafts=5, temperature=0.8, top_p=0.95, **t))
    torch.cuda.synchronize()
    for r in got:
        assert torch.equal(r.tokens, want.tokens) and torch.equal(r.logprobs, want.logprobs)


def test_in_a_graph(cuda):
    t = make(cuda, [3, 1, 0, 4], 30011, "bf16", "bf16", seed=18)
    other = make(cuda, [3, 1, 0, 4], 30011, "bf16", "bf16", seed=19)
    T, P = torch.full((4,), 0.9, device=cuda), torch.full((4,), 0.9, device=cuda)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.verify_drafts(max_drafts=4, temperature=T, top_p=P, **t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = ops.verify_drafts(max_drafts=4, temperature=T, top_p=P, **t)
    first = {k: (v.clone() if v is not None else None) for k, v in t.items()}
    for source in (first, other, first, other):
        for k in ("logits", "draft_tokens", "draft_probs", "accept_uniforms", "uniforms"):
            t[k].copy_(source[k])
        want = ops.verify_drafts(max_drafts=4, temperature=T, top_p=P, **{**source, "cu_drafts": t["cu_drafts"]})
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(r.tokens, want.tokens) and torch.equal(r.logprobs, want.logprobs)


def test_refusals(cuda):
    t = make(cuda, [2, 1], 300, "f32", "f32", seed=20)
    call = lambda **kw: ops.verify_drafts(**{**dict(max_drafts=2, temperature=1.0), **t, **kw})  # noqa: E731
    for bad in (dict(max_drafts=-1), dict(max_drafts=65), dict(uniforms=None, accept_uniforms=None),
                dict(accept_uniforms=None), dict(accept_uniforms=torch.rand(2)), dict(logits=t["logits"][:-1]),
                dict(logits=t["logits"].cpu()), dict(draft_probs=t["draft_probs"][:, :-1]), dict(uniforms=t["uniforms"][:1]),
                dict(logits=t["logits"][0]), dict(draft_tokens=t["draft_tokens"].reshape(1, -1)),
                dict(temperature=torch.ones(3)), dict(top_k=torch.ones(5, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(TypeError):
        call(logits=t["logits"].double())
    with pytest.raises(TypeError):
        call(draft_probs=t["draft_probs"].double())
    with pytest.raises(_lib.VwsError) as e:
        big = torch.zeros((5, (1 << 19) + 8), device=cuda)
        ops.verify_drafts(big, t["draft_tokens"], t["cu_drafts"], 2)
    assert e.value.status == _lib.ERR_LIMIT


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("requests", [1, 12, 70, 110])
def test_flat_rows(cuda, dtype, requests):
    """Rows whose nucleus is most of the vocabulary, few and more than the launch sets aside."""
    t = make(cuda, [2] * requests, 9001 if requests > 12 else 33001, dtype, "f32", seed=requests, spread=0.5, spikes=1)
    check(t, 2, T=1.3, p=0.9, max_near=0.5)
    check(t, 2, T=0.9, p=0.5, max_near=0.5)
