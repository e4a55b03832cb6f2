"""Calls of the drafted trees' and paged cache's C ABI that are refused before anything is launched."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests.test_tree_host import append_args, cache, tree_args
from vllm_webgpu_amd import _lib, ops


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_scales_whose_powers_of_two_overflow(scale):
    """Finite, but times log2 e no 32-bit number: a score of 0 would be none either."""
    L = _lib.lib()
    a = tree_args(L, cache(k=1 << 30, v=1 << 31), scale=scale)
    assert L.vws_tree_attention(ctypes.byref(a)) == _lib.ERR_INVALID_ARGUMENT and b"scale" in L.vws_last_error()


@pytest.mark.parametrize("name", ["k", "v", "q", "slots", "positions", "inv_freq"])
@pytest.mark.parametrize("at", ["k", "v", "last of k", "first of v from before"])
def test_inputs_in_the_cache_are_refused(name, at):
    """What a call reads it must not overwrite on the way: five tokens' keys, values, queries, slots, positions or frequencies in the
    cache's own memory."""
    L = _lib.lib()
    page = 2 * 16 * 64
    c = cache(k=1 << 30, v=1 << 31)
    where = {"k": 1 << 30, "v": 1 << 31, "last of k": (1 << 30) + 2 * (10 * page) - 2, "first of v from before": (1 << 31) - 2}[at]
    fine = dict(k=1 << 32, v=1 << 33, q=1 << 34, q_out=1 << 34, slots=1 << 35, positions=1 << 36, inv_freq=1 << 37)
    a = append_args(c, **{**fine, name: where, **({"q_out": 1 << 38} if name == "q" else {})})
    if at == "first of v from before" and name in ("slots", "positions", "inv_freq"):
        setattr(a, name, (1 << 31) - 4)
    assert L.vws_append_kv(ctypes.byref(a)) == _lib.ERR_INVALID_ARGUMENT and b"overlap" in L.vws_last_error()


@pytest.mark.parametrize("name", ["k", "v", "slots", "positions", "inv_freq"])
def test_queries_are_not_written_over_inputs(name):
    L = _lib.lib()
    fine = dict(k=1 << 32, v=1 << 33, q=1 << 34, q_out=1 << 38, slots=1 << 35, positions=1 << 36, inv_freq=1 << 37)
    a = append_args(cache(k=1 << 30, v=1 << 31), **{**fine, name: (1 << 38) + 2 * 5 * 256 - 4})
    assert L.vws_append_kv(ctypes.byref(a)) == _lib.ERR_INVALID_ARGUMENT and b"overlap" in L.vws_last_error()


def test_what_overlaps():
    """Rows of one projection side by side, heads of one projection in turn, heads outermost; and each one element too near."""
    x = torch.zeros(7 * 6 * 3 * 64)
    base, turn = x[:7 * 18 * 64].view(7, 18, 64), x.view(7, 6, 3, 64)
    q, k, v = base.split([10, 4, 4], 1)
    for a, b, meet in ((q, k, False), (k, v, False), (q, q, True), (q, base[:, 9:11], True), (turn[:, :, 0], turn[:, :, 1], False),
                       (turn[:, :, 0], turn[:, :, 2], False), (turn[:, :, 2], turn[:, :, 2], True), (turn[:, :2, 0], turn[:, 3:, 0], False),
                       (turn[:, :, 0], x[63:63 + 7 * 18 * 64 - 128].as_strided((6, 6, 64), (18 * 64, 192, 1)), True),
                       (q[3:], q[:3], False), (q[2:], k[:4], False), (base.view(-1)[:4 * 7 * 64].view(4, 7, 64).transpose(0, 1), base[4:, :4], False),
                       (base.view(-1)[:4 * 7 * 64].view(4, 7, 64).transpose(0, 1), base[1:, :4], True), (q[:1], k[:1], False), (q[:0], q, False)):
        assert ops._meet(a, b) == meet and ops._meet(b, a) == meet


@pytest.mark.parametrize("place,strides", [(0, (18 * 64, 64)), (10 * 64 - 1, (18 * 64, 64)), (17 * 64 - 1, (18 * 64, 64)), (64, (18 * 64, 192)),
                                           (10 * 64, (-18 * 64, 64)), (18 * 64 * 3 + 64, (18 * 64, -64))])
def test_queries_turned_in_place_on_keys(place, strides):
    """Queries of 10 heads in rows of 18 heads' elements, and keys of 2 heads one element too near (those that lie beside the queries
    are stored: a test on the device)."""
    L = _lib.lib()
    at = 1 << 34
    a = append_args(cache(k=1 << 30, v=1 << 31), heads=10, q=at, q_out=at, q_token_stride=18 * 64, q_head_stride=64, q_out_token_stride=18 * 64,
                    q_out_head_stride=64, k=at + 2 * place, k_token_stride=strides[0], k_head_stride=strides[1], v=1 << 33, slots=1 << 35,
                    positions=1 << 36, inv_freq=1 << 37)
    assert L.vws_append_kv(ctypes.byref(a)) == _lib.ERR_INVALID_ARGUMENT and b"overlap" in L.vws_last_error()
