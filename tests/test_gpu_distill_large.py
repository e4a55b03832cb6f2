"""The distillation loss and its gradient on student rows with large finite logits: masked spans, rows
masked whole, rows far from zero.  Against the 64-bit reference; tolerances as in test_gpu_distill, by
differences of logits (x - max) / T, which round to 2^-24 of themselves however large x is."""
from __future__ import annotations

import pytest
import torch

from tests import speculative_ref as R
from tests.test_gpu_distill import DT, ROUND, TOL, close, make
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu

TAILS = ["renormalize", "bucket"]


def fills(dtype):
    lo = float(torch.finfo(DT[dtype]).min)
    return [v for v in (-3e4, -1e9, -1e10, -3.3e10, -1e20, -1e30, lo / 2) if v > lo] + [lo]


def reference(x, ids, lp, T, tail, g):
    """Of the rows less their maxima, which changes neither loss nor gradient: differences of two logits are exact in
    64 bits where they matter, log(sum) beside a maximum of 1e30 is not."""
    z = x.double()
    leaf = (z - z.amax(1, keepdim=True)).requires_grad_(True)
    loss = R.distill(leaf, ids, lp, None, T, tail)
    (grad,) = torch.autograd.grad(loss, leaf, g.double())
    return loss.detach(), grad


def run(x, ids, lp, T, tail, g):
    """(loss, gradient) through autograd, by the one call, and in place."""
    leaf = x.detach().clone().requires_grad_(True)
    loss = ops.distill_loss(leaf, ids, lp, None, T, tail)
    (grad,) = torch.autograd.grad(loss, leaf, g)
    yield loss.detach(), grad
    one = ops.distill_loss_and_grad(x, ids, lp, None, T, tail, grad_output=g)
    yield one
    inplace = x.detach().clone()
    two = ops.distill_loss_and_grad(inplace, ids, lp, None, T, tail, grad_output=g, out=inplace)
    assert torch.equal(two[0], one[0]) and torch.equal(inplace, one[1])


# rows that the two kernels take, and (enough of them) those that one workgroup holds, of each size
SHAPES = [(1, 33001, "f32"), (1, 33001, "bf16"), (1, 33001, "f16"), (1, 1000, "f32"),
          (1600, 128256, "bf16"), (1310, 155000, "f16"), (1600, 65533, "f32"), (2400, 57347, "bf16"), (2350, 29001, "f32")]


@pytest.mark.parametrize("tail", TAILS)
@pytest.mark.parametrize("T", [1.0, 2.0, 0.7])
@pytest.mark.parametrize("rows,V,dtype", SHAPES)
def test_masked_spans(cuda, rows, V, dtype, T, tail):
    """The entries' logits stay; most of the rest is masked, in long runs or every other token."""
    values = fills(dtype)
    n = 3 * len(values)
    x, ids, lp = make(cuda, n, V, 40, dtype, seed=V)
    lp = lp - 0.7                 # (below 1 at any T)
    entry = torch.zeros((n, V), dtype=torch.bool, device=cuda).scatter_(1, ids.long(), True)
    for i, v in enumerate(values):
        span = torch.zeros((3, V), dtype=torch.bool, device=cuda)
        span[0, :V - V // 8], span[1, 100:], span[2, ::2] = True, True, True
        part = x[3 * i:3 * i + 3]
        part[span & ~entry[3 * i:3 * i + 3]] = v
    g = torch.linspace(0.5, 1.5, n, device=cuda)
    want, want_grad = reference(x, ids, lp, T, tail, g)
    rep = -(-rows // n)
    for loss, grad in run(x.repeat(rep, 1), ids.repeat(rep, 1), lp.repeat(rep, 1), T, tail, g.repeat(rep)):
        for part in (slice(0, n), slice((rep - 1) * n, rep * n)):
            close(loss[part], grad[part], want, want_grad, None, g, T, x.dtype)


@pytest.mark.parametrize("tail", TAILS)
@pytest.mark.parametrize("T", [1.0, 2.0])
@pytest.mark.parametrize("rows,V,dtype", SHAPES)
def test_rows_far_from_zero_and_masked_whole(cuda, rows, V, dtype, T, tail):
    """Rows of one large value are uniform; rows of five large values, far apart, over those of the largest."""
    lo = float(torch.finfo(DT[dtype]).max)
    values = [v for v in (6e4, -6e4, 1e6, 3.3e6, -1e10, 1e10, -1e30, 2e38) if abs(v) < lo] + [-lo, lo]
    n = 2 * len(values)
    x, ids, lp = make(cuda, n, V, 40, dtype, seed=V + 1)
    lp = lp - 0.7
    for i, v in enumerate(values):
        x[2 * i] = v                                                          # one value
        step = abs(torch.tensor(v, dtype=DT[dtype]).double()) * 2.0 ** -6     # a few of the type's steps apart
        x[2 * i + 1] = (v * (1 - 2.0 ** -7) - torch.sign(torch.tensor(v)) * step *
                        torch.arange(V, device=cuda).remainder(5)).to(x.dtype)
    g = torch.linspace(0.5, 1.5, n, device=cuda)
    want, want_grad = reference(x, ids, lp, T, tail, g)
    ok = want.abs() < 3e38
    rep = -(-rows // n)
    for loss, grad in run(x.repeat(rep, 1), ids.repeat(rep, 1), lp.repeat(rep, 1), T, tail, g.repeat(rep)):
        for part in (slice(0, n), slice((rep - 1) * n, rep * n)):
            assert torch.isfinite(grad[part]).all()
            close(loss[part][ok], grad[part][ok], want[ok], want_grad[ok], None, g[ok], T, x.dtype)


@pytest.mark.parametrize("rows,V,dtype", SHAPES)
@pytest.mark.parametrize("value", [-1e10, -6e4])
def test_a_rest_masked_whole(cuda, rows, V, dtype, value):
    """Bucket: every token outside the entries at one large negative value.  log(s) is as large as the gap, the loss
    r times that, and the rest's gradient spreads over its tokens: each to 2e-5 of itself (r, a sum of 32 bits, and
    its tokens' sum)."""
    if value < torch.finfo(DT[dtype]).min:
        return
    n = 6
    x, ids, lp = make(cuda, n, V, 40, dtype, seed=V + 2)
    lp = lp - 0.7
    entry = torch.zeros((n, V), dtype=torch.bool, device=cuda).scatter_(1, ids.long(), True)
    x[~entry] = value
    g = torch.linspace(0.5, 1.5, n, device=cuda)
    want, want_grad = reference(x, ids, lp, 1.0, "bucket", g)
    rep = -(-rows // n)
    for loss, grad in run(x.repeat(rep, 1), ids.repeat(rep, 1), lp.repeat(rep, 1), 1.0, "bucket", g.repeat(rep)):
        for part in (slice(0, n), slice((rep - 1) * n, rep * n)):
            assert ((loss[part].double() - want).abs() <= TOL * want.abs()).all()
            rel, sub = ROUND[x.dtype]
            off = (grad[part].double() - want_grad).abs()
            near = torch.where(entry, TOL * g.double().unsqueeze(1), 2 * TOL * want_grad.abs())
            assert (off <= near + rel * want_grad.abs() + sub).all()


@pytest.mark.parametrize("tail", TAILS)
@pytest.mark.parametrize("T", [1e-5, 1e-3, 1e4, 1e30, 3e38])
def test_extreme_temperatures(cuda, T, tail):
    """A token counts while it lies within 20 T of the maximum, and that difference over T is good to 2^-22 of 20."""
    x, ids, lp = make(cuda, 5, 5003, 20, "f32", seed=4)
    lp = lp - 0.7
    x[1, :4000] = -1e10
    x[2] = -1e10
    x[3] = x[3].sign() * 4096.0
    g = torch.ones(5, device=cuda)
    lp = lp if tail == "bucket" else lp * min(T, 1.0)
    want, want_grad = reference(x, ids, lp, T, tail, g)
    for loss, grad in run(x, ids, lp, T, tail, g):
        close(loss, grad, want, want_grad, None, g, T, x.dtype)
