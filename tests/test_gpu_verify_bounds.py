"""Draft verification with bounds that decrease: a row that two requests claim is one request's, the
other gets no token, whatever each cuts, and what the workspace held before is never read."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_verify import LP_TOL, make
from vllm_webgpu_amd import _lib, ops

pytestmark = pytest.mark.gpu

DIRT = (0x00, 0x7F, 0xFF, 0x11)  # of counts and indices read by mistake: 0, huge, -1, 286331153


def dirty(cuda, byte):
    """Fills the stream's workspace past the fixed region, which may hold anything."""
    _ = ops.workspace(1 << 24, cuda)
    ws = ops.workspace(1, cuda)
    ws[_lib.lib().vws_sample_workspace_size(1, 1, 0):].fill_(byte)


def fits(cu, D, K):
    """Per request: its bounds fit and each of its rows is its own (the last that starts before it)."""
    B = len(cu) - 1
    owner = [max((b for b in range(B) if cu[b] + b <= r), default=0) for r in range(D + B)]
    return [0 <= cu[b] <= cu[b + 1] <= D and cu[b + 1] - cu[b] <= K
            and all(owner[cu[b] + b + i] == b for i in range(cu[b + 1] - cu[b] + 1)) for b in range(B)]


PARAMS = {  # per request, in turn: cut ones beside uncut and greedy ones
    "topk_and_plain": dict(temperature=[0.9, 0.8, 1.1, 0.7], top_k=[5, 0, 7, 0]),
    "plain_and_topk": dict(temperature=[0.9, 0.8, 1.1, 0.7], top_k=[0, 5, 0, 7]),
    "topp_and_greedy": dict(temperature=[0.9, 0.0, 1.3, 0.0], top_p=[0.8, 1.0, 0.95, 0.5]),
    "flat_topp_and_minp": dict(temperature=[3.0, 0.9, 3.0, 0.0], top_p=[0.9, 1.0, 0.9, 1.0], min_p=[0.0, 0.05, 0.0, 0.1]),
}


@pytest.mark.parametrize("params", list(PARAMS))
@pytest.mark.parametrize("cu,K", [([0, 3, 1, 4], 3), ([0, 5, 2, 4], 5), ([0, 2, 4, 6], 2), ([0, 2, 1, 6], 5), ([0, 2, 99, 4, 6], 2),
                                  ([0, 4, 4, 0, 4], 4), ([3, 0, 3, 0, 3], 3), ([0, 1, 2, 2, 1, 3, 3], 2), ([0, -2 ** 31, 4], 4),
                                  ([0, 2 ** 31 - 1, 1, 2], 2), ([2 ** 31 - 1, -2 ** 31, 1, 2], 2)])
def test_a_row_is_one_requests(cuda, cu, K, params):
    B, V = len(cu) - 1, 40011
    D = max(c for c in cu if c < 90)
    t = make(cuda, [D] + [0] * (B - 1), V, "bf16", "f32", seed=D + B)     # rows and drafts; the bounds are `cu`
    kw = {k: [v[b % 4] for b in range(B)] for k, v in PARAMS[params].items()}
    dt = {k: torch.int32 if k == "top_k" else torch.float32 for k in kw}
    t["cu_drafts"] = torch.tensor(cu, dtype=torch.int32)
    ok = fits(cu, D, K)
    for byte in DIRT:
        dirty(cuda, byte)
        r = ops.verify_drafts(max_drafts=K, **{k: torch.tensor(v, dtype=dt[k]) for k, v in kw.items()}, **t)
        acc = r.num_accepted.cpu()
        assert [int(a) >= 0 for a in acc] == ok
        bad = torch.tensor([not o for o in ok])
        assert bool((r.tokens.cpu()[bad] == -1).all()) and not r.logprobs.cpu()[bad].any()
        for b in (b for b in range(B) if ok[b]):           # what it gives alone
            lo, hi = cu[b], cu[b + 1]
            one = ops.verify_drafts(t["logits"][lo + b:hi + b + 1], t["draft_tokens"][lo:hi], torch.tensor([0, hi - lo]), K,
                                    draft_probs=t["draft_probs"][lo:hi], accept_uniforms=t["accept_uniforms"][lo:hi],
                                    uniforms=t["uniforms"][b:b + 1], **{k: torch.tensor(v[b:b + 1], dtype=dt[k]) for k, v in kw.items()})
            assert int(one.num_accepted[0]) == int(acc[b]) and torch.equal(one.tokens[0], r.tokens[b])
            assert torch.allclose(one.logprobs[0], r.logprobs[b], rtol=0, atol=2 * LP_TOL)


@pytest.mark.parametrize("B", [65, 1000, 5000])
def test_many_requests_around_a_decreasing_bound(cuda, B):
    """Past the 64 bounds that a step of the search compares: every request has a token or none, and the
    first ones, far from the fault, have what they have without it."""
    V = 513
    counts = [b % 3 for b in range(B)]
    t = make(cuda, counts, V, "f32", None, seed=B)
    kw = dict(temperature=torch.tensor([0.0, 0.9, 1.1, 0.8] * B)[:B], top_k=torch.tensor([0, 4, 0, 0] * B, dtype=torch.int32)[:B],
              top_p=torch.tensor([1.0, 1.0, 0.9] * B)[:B])
    good = ops.verify_drafts(max_drafts=2, **kw, **t)
    cu = t["cu_drafts"].clone()
    cu[B - 3] = cu[B - 9]
    for byte in DIRT:
        dirty(cuda, byte)
        r = ops.verify_drafts(max_drafts=2, **kw, **dict(t, cu_drafts=cu))
        acc = r.num_accepted.cpu()
        assert bool((acc >= -1).all()) and bool((acc == -1).any())
        assert bool((r.tokens.cpu()[acc == -1] == -1).all())
        n = B // 2
        assert torch.equal(r.tokens[:n], good.tokens[:n]) and torch.equal(r.num_accepted[:n], good.num_accepted[:n])
    dirty(cuda, 0x7F)
    again = ops.verify_drafts(max_drafts=2, **kw, **t)
    assert torch.equal(again.tokens, good.tokens) and torch.equal(again.logprobs, good.logprobs)
