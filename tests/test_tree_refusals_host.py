"""Calls of the drafted trees' and paged cache's C ABI that are refused before anything is launched."""
from __future__ import annotations

import ctypes

import pytest

from tests.test_tree_host import append_args, cache, tree_args
from vllm_webgpu_amd import _lib


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_scales_whose_powers_of_two_overflow(scale):
    """Finite, but times log2 e no 32-bit number: a score of 0 would be none either."""
    L = _lib.lib()
    a = tree_args(L, cache(k=1 << 30, v=1 << 31), scale=scale)
    assert L.vws_tree_attention(ctypes.byref(a)) == _lib.ERR_INVALID_ARGUMENT and b"scale" in L.vws_last_error()
