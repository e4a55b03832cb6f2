"""The paged cache's appends on tensors that lie in each other's gaps: the same as on tensors of their own, or refused."""
from __future__ import annotations

import pytest
import torch

from tests import tree_ref as R
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def views(dev, layout, T, H, dim):
    """q, k and v in one buffer of random numbers."""
    x = torch.randn((T * 3 * H * dim,), device=dev, generator=torch.Generator(device=dev).manual_seed(T)).bfloat16()
    if layout == "rows":
        return x, [t.unflatten(1, (H, dim)) for t in x.view(T, -1).chunk(3, 1)]
    if layout == "heads in turn":
        return x, list(x.view(T, H, 3, dim).unbind(2))
    return x, [t.transpose(0, 1) for t in x.view(3, H, T, dim)]  # (heads outermost)


@pytest.mark.parametrize("layout", ["rows", "heads in turn", "heads outermost"])
@pytest.mark.parametrize("T", [1, 5, 2100])
def test_queries_turned_in_place_beside_their_keys(cuda, layout, T):
    H, dim = 3, 64
    x, (q, k, v) = views(cuda, layout, T, H, dim)
    slots, pos, f = torch.arange(T, device=cuda).int() + 2, torch.arange(T, device=cuda).int() * 3, torch.linspace(0.01, 1, dim // 2, device=cuda)
    args = dict(slots=slots, positions=pos, inv_freq=f)
    (ka, va), (kb, vb) = (R.make_cache(cuda, T // 16 + 2, H, 16, dim, "bf16") for _ in range(2))
    want = ops.append_kv(k.contiguous(), v.contiguous(), ka, va, q=q.contiguous(), **args)
    keep = k.clone(), v.clone()
    assert ops.append_kv(k, v, kb, vb, q=q, out=q, **args) is q
    assert torch.equal(q, want) and torch.equal(k, keep[0]) and torch.equal(v, keep[1])
    assert torch.equal(ka, kb) and torch.equal(va, vb)
    if T > 1 and layout == "rows":
        assert torch.equal(x.view(T, 3, H, dim)[:, 0], want)


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
