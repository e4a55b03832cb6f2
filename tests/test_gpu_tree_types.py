"""Integer arguments of the paged cache's and drafted trees' operators: any integer type, and no other."""
from __future__ import annotations

import pytest
import torch

from tests import tree_ref as R
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def calls(dev):
    """(operator, arguments, the integer ones' names) of a step of one request."""
    kc, vc = R.make_cache(dev, 2, 2, 16, 64, "bf16")
    q, k, v = (torch.randn((3, h, 64), device=dev).bfloat16() for h in (4, 2, 2))
    at = lambda *x: torch.tensor(x, device=dev).int()  # noqa: E731
    page = dict(k_cache=kc, v_cache=vc)
    table = dict(block_table=at(0, 1).view(1, 2), context_lens=at(5))
    return [
        (ops.append_kv, dict(k=k, v=v, **page, slots=at(5, 6, 7), q=q, positions=at(5, 6, 7), inv_freq=torch.ones(32, device=dev)),
         ("slots", "positions")),
        (ops.tree_attention, dict(q=q, **page, **table, cu_nodes=at(0, 3), max_nodes=3), ("block_table", "context_lens", "cu_nodes")),
        (ops.accept_tree, dict(sampled=at(1, 2, 3), tokens=at(0, 1, 2), parents=at(-1, 0, 1), cu_nodes=at(0, 3), max_path=3), ("cu_nodes",)),
        (ops.compact_kv, dict(**page, **table, path=at(0, 2).view(1, 2)), ("block_table", "context_lens", "path")),
    ]


@pytest.mark.parametrize("which", range(4))
def test_whole_numbers_only(cuda, which):
    """Positions of 5.5, or slots that went through floating point, are not cut to whole numbers without a word."""
    call, args, names = calls(cuda)[which]
    for name in names:
        for dtype in (torch.float32, torch.float64, torch.bfloat16, torch.bool):
            with pytest.raises(ValueError, match=name):
                call(**{**args, name: args[name].to(dtype)})


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("dtype", [torch.int64, torch.int16, torch.int8])
def test_any_integer_type(cuda, which, dtype):
    call, args, names = calls(cuda)[which]
    first = lambda r: r if torch.is_tensor(r) else r.tokens  # noqa: E731
    want = first(call(**args))
    assert torch.equal(first(call(**{**args, **{n: args[n].to(dtype) for n in names}})), want)
