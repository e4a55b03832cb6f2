"""Draft verification on rows with large finite logits: tokens masked by a large negative value, rows
masked whole by one, rows far from zero.  Against the plain 64-bit reference, which takes y = fl32(x / T)
and fl32(y - max) as the sampler does, and against the sampler itself.

Tolerance: log p = (y - m) - log(sum).  The first term is the reference's own; the sum is good to
2e-6 near zero and wherever |max log2(e) / T| exceeds 2^14, from where it is over the same rounded
y; below that it is over x log2(e) / T, and y and m round to 2^-24 of |m| each, its constant likewise."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import speculative_ref as R
from tests.test_gpu_verify import DT, LP_TOL, full, make
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def check(t, K, T=1.0, k=0, p=1.0, min_p=0.0, max_near=0.1, size=0.0):
    """As test_gpu_verify's, with a tolerance for rows whose |max / T| is ``size``."""
    B = t["cu_drafts"].numel() - 1
    T, k, p, min_p = full(T, B, np.float32), full(k, B, np.int32), full(p, B, np.float32), full(min_p, B, np.float32)
    r = ops.verify_drafts(max_drafts=K, temperature=torch.from_numpy(T), top_k=torch.from_numpy(k) if k.any() else None,
                          top_p=torch.from_numpy(p) if (p < 1).any() else None,
                          min_p=torch.from_numpy(min_p) if min_p.any() else None, **t)
    torch.cuda.synchronize()
    h = {a: (None if v is None else v.float().cpu().numpy() if v.is_floating_point() else v.cpu().numpy()) for a, v in t.items()}
    tok, acc, lp, near = R.verify(h["logits"], h["draft_tokens"], h["cu_drafts"], K, h["draft_probs"], T, k, p, min_p,
                                  h["accept_uniforms"], h["uniforms"])
    ok = ~near
    assert near.mean() <= max_near, f"{near.sum()} of {B} requests too close to call"
    if size:  # a decision within the larger tolerance may fall either way: a few in a thousand
        same = (r.tokens.cpu().numpy() == tok).all(1)
        assert same[ok].mean() >= 0.6
        ok &= same
    np.testing.assert_allclose(r.logprobs.cpu().numpy()[ok], lp[ok], rtol=0, atol=LP_TOL + 4 * 2.0 ** -24 * size)
    np.testing.assert_array_equal(r.num_accepted.cpu().numpy()[ok], acc[ok])
    np.testing.assert_array_equal(r.tokens.cpu().numpy()[ok], tok[ok])
    return acc[ok]


def masks(dtype):
    lo = float(torch.finfo(DT[dtype]).min)
    return [v for v in (-1e4, -3e4, -1e9, -1e10, -3.3e10, -1e20, -1e30, lo / 2) if v > lo] + [lo]


CUTS = [dict(), dict(p=0.9), dict(k=20), dict(min_p=0.02), dict(k=40, p=0.8, min_p=0.01)]


@pytest.mark.parametrize("T", [0.7, 1.0, 1.2, 3.0])
@pytest.mark.parametrize("dtype,probs", [("f32", "f32"), ("bf16", None), ("bf16", "bf16"), ("f16", "f32")])
def test_tokens_masked_by_a_large_value(cuda, dtype, probs, T):
    """All but a few tokens, long runs, or every other one."""
    values = masks(dtype)
    B, V = len(values), 33001
    t = make(cuda, [2] * B, V, dtype, probs, seed=3, T=T)
    x = t["logits"]
    for b, v in enumerate(values):
        x[3 * b, :30000] = v
        x[3 * b + 1, 40:] = v
        x[3 * b + 2, ::2] = v
    for cut in CUTS:
        check(t, 2, T=T, max_near=0.4, **cut)


@pytest.mark.parametrize("T", [0.7, 1.0, 1.2])
@pytest.mark.parametrize("probs", [None, "f32"])
@pytest.mark.parametrize("dtype,value", [("f32", -1e9), ("f32", -1e10), ("f32", -1e20), ("f32", -1e30), ("f32", 1e10), ("f32", 1e30),
                                         ("f32", -2.0e38), ("bf16", -1e10), ("bf16", -1e30), ("bf16", 3e9), ("f16", -65504.0),
                                         ("f16", 60000.0), ("f32", -20000.5)])
def test_rows_of_one_large_value(cuda, dtype, value, probs, T):
    """A row that is masked whole is uniform over its tokens, as its logits are equal."""
    t = make(cuda, [1, 2, 0, 1, 1, 1], 9001, dtype, probs, seed=5, T=T)
    if probs:
        t["draft_probs"][:3] = 1.0 / 9001
    t["logits"][:] = value
    acc = check(t, 2, T=T, max_near=0.5)
    assert probs is None or len(acc)
    for p in (0.9, 0.5):
        check(t, 2, T=T, p=p, max_near=0.8)
    check(t, 2, T=T, k=3, max_near=0.5)
    check(t, 2, T=T, min_p=0.5, max_near=0.5)


@pytest.mark.parametrize("T", [0.7, 1.0, 1.2])
@pytest.mark.parametrize("V", [11, 5000, 33000])
def test_without_drafts_it_is_the_sampler(cuda, V, T):
    """The type's lowest value among the fills: at T < 1 the scaled logits are infinite."""
    g = torch.Generator().manual_seed(V)
    for dtype in ("f32", "bf16", "f16"):
        values = masks(dtype) + [-min(masks(dtype)), 1e4]
        B = 2 * len(values)
        x = torch.randn((B, V), generator=g).to(DT[dtype])
        for i, v in enumerate(values):
            x[2 * i] = v
            x[2 * i + 1, V // 3] = v
        x = x.to(cuda)
        u = torch.rand((B, V), generator=g).clamp(2.0 ** -24, 1 - 2.0 ** -24).to(cuda)
        cu = torch.zeros(B + 1, dtype=torch.int32, device=cuda)
        for kw in (dict(), dict(top_p=0.9), dict(top_k=5), dict(min_p=0.1)):
            want = ops.sample(x, temperature=T, uniforms=u, **kw)
            got = ops.verify_drafts(x, torch.zeros(0, dtype=torch.int32), cu, 0, temperature=T, uniforms=u,
                                    accept_uniforms=torch.zeros(0), **kw)
            assert torch.equal(got.tokens[:, 0], want.sampled), (dtype, kw)
            assert torch.isfinite(got.logprobs).all() and not (got.logprobs > LP_TOL).any()


@pytest.mark.parametrize("T", [0.7, 1.0, 1.2])
@pytest.mark.parametrize("probs", [None, "f32"])
def test_one_token_near_the_largest_value(cuda, probs, T):
    """It is certain, by its logit or (T < 1) as the row's only infinite one: its draft is accepted."""
    t = make(cuda, [1, 1, 1, 1], 4001, "f32", probs, seed=7)
    t["logits"][:] = 0.0
    t["logits"][::2, 77] = 3.38e38
    t["draft_tokens"][:] = torch.tensor([77, 5, 77, 4000], dtype=torch.int32)
    r = ops.verify_drafts(max_drafts=1, temperature=T, **t)
    assert r.num_accepted.tolist() == [1, 0, 1, 0]
    assert r.tokens[:, 0].tolist() == [77] * 4
    assert float(r.logprobs[:, 0].abs().max()) <= LP_TOL
    assert torch.allclose(r.logprobs[::2, 1], torch.full((2,), -np.log(4001.0), device=cuda, dtype=torch.float32), atol=LP_TOL)


@pytest.mark.parametrize("offset", [100.0, -1000.0, 1.2e4, -1.0e5, 1.0e6, 1.0e7, -1.6e7])
@pytest.mark.parametrize("T", [0.7, 1.0, 2.5])
@pytest.mark.parametrize("probs", [None, "f32"])
def test_rows_far_from_zero(cuda, offset, T, probs):
    t = make(cuda, [2, 0, 3, 1, 2, 2], 20011, "f32", probs, seed=9, T=T)
    t["logits"] += offset
    size = abs(offset) / T
    size = size if size * 1.4427 < 2.0 ** 14 else 0.0
    for cut in CUTS:
        check(t, 3, T=T, max_near=0.9, size=size, **cut)


@pytest.mark.parametrize("T", [0.7, 1.0])
def test_rows_on_both_sides_of_the_bound(cuda, T):
    """|max log2(e) / T| around 2^14, with parts of one row on either side of it."""
    edge = 2.0 ** 14 / 1.4426950 * T
    V = 40000
    t = make(cuda, [1] * 6, V, "f32", "f32", seed=11, T=T)
    x = t["logits"]
    for r, at in enumerate((edge - 40, edge - 1, edge + 1, edge + 40, -edge - 1, -edge + 1, edge * 1.0001)):
        x[r] = at + x[r] * 0.5
        x[r, :V // 2] += 2.0 if r % 2 else -2.0
        x[r, V - 5000:] = 0.0
    x[8, :V // 2] = -2.0 ** 21
    x[9, V // 2:] = 2.0 ** 18
    check(t, 1, T=T, max_near=0.9, size=2.0 ** 14 / 1.4427)
    check(t, 1, T=T, p=0.9, max_near=0.9, size=2.0 ** 14 / 1.4427)
