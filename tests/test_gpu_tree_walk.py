"""The walk down a drafted tree where parents and bounds are odd: every output against the plain walk."""
from __future__ import annotations

import pytest
import torch

from tests import tree_ref as R
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("parents,cu,counts", [
    ([-1, 0, 1, 0, 1], [0, 3, 2, 5], [2, -1, 2]), ([-1, 0, 1, 0, 1], [0, 6, 5, 5], [-1, -1, -1]),
    ([-1, 0, 1, 0, 1], [-1, 2, 5, 2 ** 31 - 1], [-1, 2, -1]), ([-1, 0, 1, 2, 3], [0, 5, 5, 2], [4, -1, -1]),
    ([-1, 0, 1, 2, 3], [0, 4, 5, 5], [3, 0, -1]), ([-1, 0, 5, 1, 3], [0, 5, 5], [3, -1]),
])
@pytest.mark.parametrize("width", [1, 3, 70])
def test_walks_of_odd_trees(cuda, parents, cu, counts, width):
    """Every node holds the token that is sampled at every node, so that a walk goes as far as the tree does."""
    dev = lambda x: torch.tensor(x, device=cuda).int()  # noqa: E731
    r = ops.accept_tree(dev([7] * 5), dev([7] * 5), dev(parents), dev(cu), width)
    assert r.num_accepted.tolist() == [min(c, width - 1) for c in counts]
    for b, count in enumerate(counts):
        lo, hi = (cu[b], cu[b + 1]) if count >= 0 else (0, 0)
        out, path, _ = R.walk([7] * (hi - lo), [7] * (hi - lo), parents[lo:hi], [0, hi - lo], width)
        assert r.tokens[b].tolist() == out[0] and r.path[b].tolist() == path[0]
