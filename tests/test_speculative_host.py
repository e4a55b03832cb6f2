"""The speculative-decoding entry points on the CPU: sizes, argument checks and the status codes that
the header documents.  Every call here returns before a launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

from vllm_webgpu_amd import _lib, ops

FAKE = 0x10000000


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def verify_args(L, **over):
    a = _lib.VerifyArgs()
    a.struct_size = ctypes.sizeof(_lib.VerifyArgs)
    a.batch, a.vocab, a.dtype, a.num_drafts, a.max_drafts = 4, 1000, _lib.DTYPE_F32, 8, 3
    a.logits, a.logits_row_stride, a.draft_tokens, a.cu_drafts = FAKE, 1000, FAKE, FAKE
    a.temperature, a.rng_key_set = FAKE, 1
    a.tokens, a.num_accepted, a.logprobs = FAKE, FAKE, FAKE
    a.workspace, a.workspace_bytes = FAKE, L.vws_verify_workspace_size(4, 8, 1000)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(struct_size=8), 1), (dict(logits=None), 1), (dict(batch=0), 1), (dict(vocab=0), 5), (dict(vocab=(1 << 19) + 1), 5),
    (dict(dtype=3), 2), (dict(logits_row_stride=999), 1), (dict(num_drafts=-1), 1), (dict(max_drafts=65), 5),
    (dict(max_drafts=-1), 5), (dict(num_drafts=(1 << 24)), 5), (dict(cu_drafts=None), 1), (dict(draft_tokens=None), 1),
    (dict(draft_probs=FAKE, draft_probs_dtype=7, draft_probs_row_stride=1000), 2),
    (dict(draft_probs=FAKE, draft_probs_row_stride=999), 1), (dict(rng_key_set=0), 1),
    (dict(uniforms=FAKE, uniforms_row_stride=999, accept_uniforms=FAKE), 1),
    (dict(uniforms=FAKE, uniforms_row_stride=1000), 1), (dict(tokens=None), 1), (dict(num_accepted=None), 1),
    (dict(logprobs=None), 1), (dict(workspace=None), 3), (dict(workspace_bytes=1000), 3), (dict(workspace=FAKE + 16), 1),
])
def test_verify_refusals(L, over, status):
    a = verify_args(L, **over)
    assert L.vws_verify_drafts(ctypes.byref(a)) == status
    assert L.vws_last_error()


def distill_args(L, **over):
    a = _lib.DistillArgs()
    a.struct_size = ctypes.sizeof(_lib.DistillArgs)
    a.rows, a.vocab, a.dtype, a.teacher_k, a.tail, a.temperature = 4, 1000, _lib.DTYPE_BF16, 20, 1, 1.0
    a.logits, a.logits_row_stride = FAKE, 1000
    a.teacher_ids, a.teacher_ids_row_stride, a.teacher_logprobs, a.teacher_logprobs_row_stride = FAKE, 20, FAKE, 20
    a.loss, a.saved, a.saved_bytes = FAKE, FAKE, L.vws_distill_saved_size(4, 20)
    a.grad, a.grad_row_stride = FAKE + 0x100000, 1000
    a.workspace, a.workspace_bytes = FAKE, L.vws_distill_workspace_size(4, 1000)
    for k, v in over.items():
        setattr(a, k, v)
    return a


BOTH = ("vws_distill_forward", "vws_distill_backward", "vws_distill_step")
FWD, BWD = ("vws_distill_forward", "vws_distill_step"), ("vws_distill_backward", "vws_distill_step")


@pytest.mark.parametrize("names,over,status", [
    (BOTH, dict(struct_size=8), 1), (BOTH, dict(logits=None), 1), (BOTH, dict(rows=0), 1), (BOTH, dict(rows=(1 << 24) + 1), 5),
    (BOTH, dict(vocab=(1 << 19) + 1), 5), (BOTH, dict(dtype=9), 2), (BOTH, dict(logits_row_stride=999), 1),
    (BOTH, dict(teacher_k=0), 5), (BOTH, dict(teacher_k=257), 5), (BOTH, dict(tail=2), 1), (BOTH, dict(temperature=0.0), 1),
    (BOTH, dict(temperature=float("nan")), 1), (BOTH, dict(temperature=float("inf")), 1), (BOTH, dict(teacher_ids=None), 1),
    (BOTH, dict(teacher_logprobs=None), 1), (BOTH, dict(teacher_ids_row_stride=19), 1),
    (BOTH, dict(teacher_logprobs_row_stride=19), 1), (BOTH, dict(saved=None), 3), (BOTH, dict(saved_bytes=100), 3),
    (BOTH, dict(saved=FAKE + 4), 1), (FWD, dict(loss=None), 1), (FWD, dict(workspace=None), 3),
    (FWD, dict(workspace_bytes=10), 3), (FWD, dict(workspace=FAKE + 8), 1), (BWD, dict(grad=None), 1),
    (BWD, dict(grad_row_stride=999), 1), (BWD, dict(grad=FAKE + 2), 1), (BWD, dict(grad=FAKE, grad_row_stride=1001), 1),
    (BWD, dict(grad=FAKE + 7999 - 2000), 1),
])
def test_distill_refusals(L, names, over, status):
    for name in names:
        a = distill_args(L, **over)
        assert getattr(L, name)(ctypes.byref(a)) == status, name
        assert L.vws_last_error()


def test_null_arguments(L):
    for f in (L.vws_verify_drafts, L.vws_distill_forward, L.vws_distill_backward, L.vws_distill_step):
        assert f(None) == _lib.ERR_INVALID_ARGUMENT


def test_sizes(L):
    fixed = L.vws_sample_workspace_size(1, 1, 0)
    for B in (1, 7, 256, 5000, 1 << 23):
        for D in (0, 1, 900, 1 << 22):
            for V in (1, 64, 32000, 1 << 19):
                n = L.vws_verify_workspace_size(B, D, V)
                assert n >= fixed + 24 * (B + D) + 12 * B and n % 256 == 0
    for bad in ((0, 1, 10), (1, -1, 10), (1, 1, 0), (1, 1, (1 << 19) + 1), (1 << 24, 1, 10), ((1 << 24) + 1, 0, 10)):
        assert L.vws_verify_workspace_size(*bad) == 0
    for N in (1, 100, 8192, 8193, 20000):
        for V in (1, 32000, 1 << 19):
            assert L.vws_distill_workspace_size(N, V) >= fixed
        assert L.vws_distill_saved_size(N, 20) == 4 * N * 28
    assert L.vws_distill_workspace_size(0, 10) == 0 and L.vws_distill_workspace_size(1, (1 << 19) + 1) == 0
    assert L.vws_distill_saved_size(0, 4) == 0 and L.vws_distill_saved_size(4, 0) == 0


def test_no_fallback_on_host_tensors():
    with pytest.raises(ValueError):
        ops.verify_drafts(torch.zeros(2, 10), torch.zeros(1, dtype=torch.int32), torch.tensor([0, 1]), 1)
    with pytest.raises(ValueError):
        ops.distill_loss(torch.zeros(2, 10), torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1)))
