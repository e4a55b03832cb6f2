"""Draft verification of more rows than one launch of a workgroup each takes."""
from __future__ import annotations

import pytest
import torch

from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(top_k=2), dict(top_p=0.6), dict()])
def test_more_rows_than_a_launch_takes(cuda, kw):
    """Four million requests of one row each, but for a few with a draft at either end and in the middle:
    what each gives in a call of a few."""
    V, B = 6, (1 << 22) + 11
    g = torch.Generator().manual_seed(2)
    picks = [0, 1, (1 << 21) - 1, 1 << 21, (1 << 21) + 1, 1 << 22, B - 2, B - 1]
    counts = torch.zeros(B, dtype=torch.int64)
    counts[picks[::2]] = 1
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = counts.cumsum(0)
    D = int(cu[-1])
    x = torch.randn((4096, V), generator=g).to(cuda).repeat(-(-(B + D) // 4096), 1)[:B + D]
    drafts = torch.randint(V, (D,), generator=g).int()
    seeds = torch.arange(B) * 7 + 3
    try:
        r = ops.verify_drafts(x, drafts, cu, 1, temperature=0.9, rng_seeds=seeds, **kw)
        rows = torch.cat([torch.arange(int(cu[b]) + b, int(cu[b + 1]) + b + 1) for b in picks]).to(cuda)
        few = torch.cat([torch.zeros(1, dtype=torch.int64), counts[picks].cumsum(0)])
        one = ops.verify_drafts(x[rows], drafts, few, 1, temperature=0.9, rng_seeds=seeds[picks], **kw)
        at = torch.tensor(picks, device=cuda)
        assert torch.equal(r.tokens[at], one.tokens) and torch.equal(r.num_accepted[at], one.num_accepted)
        assert torch.allclose(r.logprobs[at], one.logprobs, rtol=0, atol=1e-5)
        assert bool((r.num_accepted >= 0).all()) and bool((r.tokens[:, 0] >= 0).all()) and bool((r.tokens[:, 0] < V).all())
        share = torch.bincount(r.tokens[:, 0].long(), minlength=V).double()
        if not kw:
            want = torch.softmax(x[:4096].double() / 0.9, 1).mean(0)
            assert (share / B - want).abs().max() < 5 * (0.25 / B) ** 0.5 + 1e-5
    finally:  # (its 13 GB of workspace are nobody else's need)
        del x
        ops._ws_cache.clear()
        torch.cuda.empty_cache()
