"""The paged cache's appends on tensors that lie in each other's gaps: the same as on tensors of their own, or refused."""
from __future__ import annotations

import pytest
import torch

from tests import tree_ref as R
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def test_inputs_in_the_cache_are_refused(cuda):
    """Tokens copied from one place of a cache to another: through memory of their own."""
    kc, vc = R.make_cache(cuda, 4, 2, 16, 64, "bf16")
    slots = torch.arange(16, device=cuda).int() + 32
    k, v = kc[0].transpose(0, 1), vc[0].permute(2, 0, 1)
    for keys, values in ((k, v.contiguous()), (k.contiguous(), vc.view(-1, 2, 64)[:16]), (k, v)):
        with pytest.raises(ops._lib.VwsError):
            ops.append_kv(keys, values, kc, vc, slots)
    with pytest.raises(ops._lib.VwsError):
        ops.append_kv(k.contiguous(), v.contiguous(), kc, vc, slots, q=kc[1].transpose(0, 1))
    ops.append_kv(k.contiguous(), v.contiguous(), kc, vc, slots)
    assert torch.equal(kc[2], kc[0]) and torch.equal(vc[2], vc[0])
