"""The distillation loss and its gradient (``ops.distill_loss``, ``ops.distill_loss_and_grad``) on the GPU
against a plain 64-bit reference, whose gradient is autograd's, and against differences.

Tolerances.  In powers of two, a logit enters as fma(x, log2(e) / T, -max): the constant's rounding
costs 2^-24 |x - max| / T, the fma's 2^-24 of the result, each below 3e-6 for rows that span 40; sums
and logarithms add a few 2^-24 of at most 20.  Log probabilities are good to 1e-5, so is a loss of unit
weight (convex sums of them), and a probability to 1e-5 of itself.  A gradient is weight * upstream / T
times differences of such probabilities, rounded to its type: half an ulp, 2^-9 (bf16) or 2^-12 (f16, and
2^-25 of its subnormals) of itself."""
from __future__ import annotations

import pytest
import torch

from tests import speculative_ref as R
from vllm_webgpu_amd import _lib, ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TOL = 1e-5
ROUND = {torch.float32: (0.0, 0.0), torch.bfloat16: (2.0 ** -8, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -24)}


def make(cuda, N, V, K, dtype="f32", seed=0, lift=9.0, noise=1.0):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn((N, V), generator=g)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)]) if V < 5000 else (
        torch.randperm(V, generator=g)[:K].unsqueeze(0) + torch.randint(V, (N, 1), generator=g)) % V
    t.scatter_add_(1, ids, (lift - 1.2 * torch.arange(K).float().log1p()).expand(N, K).contiguous())
    lp = torch.log_softmax(t.double(), 1).gather(1, ids).float()
    x = (t + noise * torch.randn((N, V), generator=g)).to(DT[dtype])
    return x.to(cuda), ids.int().to(cuda), lp.to(cuda)


def reference(x, ids, lp, w, T, tail, g):
    leaf = x.detach().double().requires_grad_(True)
    loss = R.distill(leaf, ids, lp, w, T, tail)
    (grad,) = torch.autograd.grad(loss, leaf, g.double())
    return loss.detach(), grad


def close(loss, grad, want, want_grad, w, g, T, dtype):
    w = torch.ones_like(want) if w is None else w.double().abs()
    assert ((loss.double() - want).abs() <= TOL * (w + want.abs()) + 1e-12).all(), (loss.double() - want).abs().max()
    rel, sub = ROUND[dtype]
    scale = (w * g.double().abs() / T).unsqueeze(1)
    bound = TOL * scale + rel * want_grad.abs() + sub
    off = (grad.double() - want_grad).abs()
    assert (off <= bound).all(), f"{(off / bound.clamp(min=1e-300)).max():.3g} times the bound"


def check(x, ids, lp, w=None, T=1.0, tail="renormalize"):
    """Forward and backward through autograd, the one call, and the one call in place."""
    N = x.shape[0]
    g = torch.linspace(0.5, 1.5, N, device=x.device)
    want, want_grad = reference(x, ids, lp, w, T, tail, g)
    leaf = x.detach().clone().requires_grad_(True)
    loss = ops.distill_loss(leaf, ids, lp, w, T, tail)
    (grad,) = torch.autograd.grad(loss, leaf, g)
    assert grad.dtype == x.dtype and loss.dtype == torch.float32
    close(loss.detach(), grad, want, want_grad, w, g, T, x.dtype)
    one, one_grad = ops.distill_loss_and_grad(x, ids, lp, w, T, tail, grad_output=g)
    close(one, one_grad, want, want_grad, w, g, T, x.dtype)
    inplace = x.detach().clone()
    two, two_grad = ops.distill_loss_and_grad(inplace, ids, lp, w, T, tail, grad_output=g, out=inplace)
    assert two_grad is inplace and torch.equal(two, one) and torch.equal(inplace, one_grad)
    return loss.detach(), grad


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,V,K", [(1, 32000, 20), (7, 50257, 64), (33, 4099, 5), (300, 1024, 256), (3, 262144, 128), (2, 524288, 9)])
def test_shapes_and_types(cuda, tail, dtype, N, V, K):
    check(*make(cuda, N, V, K, dtype, seed=N + V), tail=tail)


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("V", [1, 2, 3, 5, 7, 8, 9, 31, 33, 64, 255, 256, 257, 1025, 4095, 4097, 8193, 12289])
def test_odd_vocabularies(cuda, tail, V):
    for dtype in ("f32", "bf16"):
        check(*make(cuda, 5, V, min(V, 3), dtype, seed=V), tail=tail)


@pytest.mark.parametrize("V,dtype", [(31999, "f32"), (65537, "bf16"), (128256, "bf16"), (128256, "f32"), (131072, "f16"),
                                     (131073, "bf16"), (151936, "bf16"), (163841, "f16"), (65536, "f32"), (81921, "f32")])
@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_long_rows_with_many_of_them(cuda, V, dtype, tail):
    """Enough rows that a row is one workgroup's."""
    x, ids, lp = make(cuda, 1, V, 40, dtype, seed=V)
    N = 530
    x = (x.float() + 0.1 * torch.randn((N, 1), generator=torch.Generator().manual_seed(1)).to(cuda)).to(x.dtype)
    x[:, ::3] += torch.linspace(-1, 1, N, device=cuda).to(x.dtype).unsqueeze(1)
    ids, lp = ids.expand(N, -1), lp.expand(N, -1)
    g = torch.linspace(0.5, 1.5, N, device=cuda)
    loss, grad = ops.distill_loss_and_grad(x, ids, lp, tail=tail, grad_output=g)
    for part in (slice(0, 40), slice(N - 40, N)):
        want, want_grad = reference(x[part], ids[part], lp[part], None, 1.0, tail, g[part])
        close(loss[part], grad[part], want, want_grad, None, g[part], 1.0, x.dtype)
    leaf = x.requires_grad_(True)
    two = ops.distill_loss(leaf, ids, lp, tail=tail)
    (two_grad,) = torch.autograd.grad(two, leaf, g)
    assert torch.allclose(two, loss, rtol=TOL, atol=TOL)
    rel, sub = ROUND[x.dtype]
    off, top = (two_grad.float() - grad.float()).abs(), two_grad.float().abs()
    assert (off <= 2 * TOL * g.unsqueeze(1) + 2 * rel * top + 2 * sub).all()
    del x.grad
    inplace = x.detach()
    one, _ = ops.distill_loss_and_grad(inplace, ids, lp, tail=tail, grad_output=g, out=inplace)
    assert torch.equal(one, loss) and torch.equal(inplace, grad)


@pytest.mark.parametrize("V,dtype,N", [(49160, "bf16", 4200), (65529, "f16", 3100), (128257, "bf16", 1600), (25001, "f32", 4100),
                                       (65533, "f32", 1600), (155000, "f16", 1310), (77000, "f32", 1400), (57347, "bf16", 2400),
                                       (29001, "f32", 2350)])
@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_large_steps(cuda, V, dtype, N, tail):
    """Calls beyond the last-level cache, whose rows one workgroup holds: against the two kernels (forward
    and backward by autograd) on some rows, rows that do not count among them, and in place."""
    x, ids, lp = make(cuda, 1, V, 40, dtype, seed=V)
    w = (torch.arange(N, device=cuda) % 5 != 2).float() * 1.5
    x = x.expand(N, -1).contiguous()
    x[:, ::7] += torch.linspace(-2, 2, N, device=cuda).to(x.dtype).unsqueeze(1)
    x[2] = float("nan")          # (weight 0: not read)
    ids, lp = ids.expand(N, -1).contiguous(), lp.expand(N, -1).contiguous()
    ids[4, 3], ids[5, 1], ids[N - 1, 6:] = -1, ids[5, 0], V + 3
    g = torch.linspace(0.5, 1.5, N, device=cuda)
    loss, grad = ops.distill_loss_and_grad(x, ids, lp, w, 1.0, tail, grad_output=g)
    for part in (slice(0, 24), slice(N - 24, N)):
        live = [i for i in range(*part.indices(N)) if w[i] != 0]
        want, want_grad = reference(x[live], ids[live], lp[live], w[live], 1.0, tail, g[live])
        close(loss[live], grad[live], want, want_grad, w[live], g[live], 1.0, x.dtype)
    assert not loss[2::5].any() and not grad[2::5].any()
    again = ops.distill_loss_and_grad(x, ids, lp, w, 1.0, tail, grad_output=g, out=x)
    assert torch.equal(again[0], loss) and torch.equal(x, grad)


@pytest.mark.parametrize("T", [0.5, 1.0, 2.0, 3.7])
@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_temperature_and_weights(cuda, T, tail):
    x, ids, lp = make(cuda, 24, 9001, 16, "f32", seed=2)
    if tail == "bucket":  # the teacher's log probabilities are those at T
        lp = lp - 1.0
    w = torch.rand(24, generator=torch.Generator().manual_seed(3)).to(cuda) * 3
    w[5] = w[11] = 0.0
    loss, grad = check(x, ids, lp, w, T, tail)
    assert loss[5] == 0 and not grad[5].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_rows_of_weight_zero_are_not_read(cuda, dtype, tail):
    x, ids, lp = make(cuda, 6, 5001, 8, dtype, seed=4)
    x[2], lp[4] = float("nan"), float("nan")
    w = torch.tensor([1.0, 2.0, 0.0, 1.0, 0.0, 0.5], device=cuda)
    g = torch.ones(6, device=cuda)
    loss, grad = ops.distill_loss_and_grad(x, ids, lp, w, tail=tail)
    assert loss[2] == 0 and loss[4] == 0 and not grad[2].any() and not grad[4].any()
    live = [0, 1, 3, 5]
    want, want_grad = reference(x[live], ids[live], lp[live], w[live], 1.0, tail, g[live])
    close(loss[live], grad[live], want, want_grad, w[live], g[live], 1.0, x.dtype)


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_padding_and_empty_rows(cuda, tail):
    x, ids, lp = make(cuda, 6, 700, 12, "f32", seed=5)
    ids[0, 5:] = -1
    ids[1] = 700
    ids[2, ::2] = 2 ** 31 - 1
    ids[3, 1:] = -2 ** 31
    lp[4, 3:] = float("-inf")
    lp[0, 5:] = float("nan")     # what stands at padding is not used
    loss, grad = check(x, ids, lp, tail=tail)
    assert loss[1] == 0 and not grad[1].any()


def test_a_renormalised_row_of_infinities_is_empty(cuda):
    x, ids, lp = make(cuda, 3, 700, 12, "f32", seed=6)
    lp[1] = float("-inf")
    loss, grad = check(x, ids, lp)
    assert loss[1] == 0 and not grad[1].any()


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_entries_that_share_an_id_add_up(cuda, tail):
    x, ids, lp = make(cuda, 4, 900, 20, "f32", seed=7)
    ids[0, 7] = ids[0, 3]
    ids[1, 1:4] = ids[1, 0]
    ids[2, 10:] = ids[2, :10].clone()
    lp -= 1.0                    # so that the bucket's sum stays below 1
    check(x, ids, lp, tail=tail)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_masked_student_logits(cuda, dtype, tail):
    x, ids, lp = make(cuda, 5, 6007, 10, dtype, seed=8)
    lo = torch.finfo(DT[dtype]).min
    inside = torch.zeros((5, 6007), dtype=torch.bool, device=cuda).scatter_(1, ids.long(), True)
    x[0] = torch.where(inside[0], x[0], float("-inf"))      # only the entries are left
    x[1, :3000] = torch.where(inside[1, :3000], x[1, :3000], float("-inf"))
    x[2] = torch.where(inside[2], x[2], lo)                 # masks of the type's lowest value
    x[3, ::2] = torch.where(inside[3, ::2], x[3, ::2], lo)
    g = torch.ones(5, device=cuda)
    loss, grad = ops.distill_loss_and_grad(x, ids, lp, tail=tail)
    want, want_grad = reference(x, ids, lp, None, 1.0, tail, g)
    if tail == "bucket":         # a rest at the lowest value: log(s) is as large, in proportion to r
        assert torch.isfinite(loss).all() if dtype != "f32" else True
        rows = [0, 1, 3]
    else:
        rows = [0, 1, 2, 3, 4]
    close(loss[rows], grad[rows], want[rows], want_grad[rows], None, g[rows], 1.0, x.dtype)
    assert torch.isfinite(grad).all()


@pytest.mark.parametrize("gap", [20.0, 100.0, 300.0])
def test_a_rest_far_below_the_entries(cuda, gap):
    """s = e^-gap underflows beside the entries; log(s) and q / s do not."""
    x, ids, lp = make(cuda, 4, 3001, 10, "f32", seed=9)
    x.scatter_add_(1, ids.long(), torch.full((4, 10), gap, device=cuda))
    lp -= 0.5
    g = torch.ones(4, device=cuda)
    loss, grad = ops.distill_loss_and_grad(x, ids, lp, tail="bucket")
    want, want_grad = reference(x, ids, lp, None, 1.0, "bucket", g)
    assert ((loss.double() - want).abs() <= TOL * want.abs()).all()
    # the rest's share r q / s spans its own 20 nats: good to 1e-5 of itself
    assert ((grad.double() - want_grad).abs() <= 4 * TOL).all()


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_impossible_entries_and_broken_rows(cuda, tail):
    inf, nan = float("inf"), float("nan")
    x, ids, lp = make(cuda, 6, 800, 6, "f32", seed=10)
    x[0, ids[0, 2].long()] = -inf      # an entry the student cannot produce
    x[1] = -inf                        # nothing left
    x[2, 9] = nan
    x[3, 9] = inf
    lp[4, 1] = nan
    loss, grad = ops.distill_loss_and_grad(x, ids, lp, tail=tail)
    assert loss[0] == inf and torch.isfinite(grad[0]).all()
    assert loss[1] == inf and torch.isfinite(grad[1]).all()
    assert torch.isnan(loss[2:5]).all()
    want, want_grad = reference(x[5:], ids[5:], lp[5:], None, 1.0, tail, torch.ones(1, device=cuda))
    close(loss[5:], grad[5:], want, want_grad, None, torch.ones(1, device=cuda), 1.0, x.dtype)
    p = torch.exp(lp[0]) if tail == "bucket" else torch.softmax(lp[0], 0)
    assert abs(float(grad[0, ids[0, 2].long()]) + float(p[2])) <= TOL


@pytest.mark.parametrize("V", [4, 40])
def test_every_token_an_entry(cuda, V):
    x, ids, lp = make(cuda, 5, V, V, "f32", seed=V)
    for tail in ("renormalize", "bucket"):
        check(x, ids, lp, tail=tail)


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_against_differences(cuda, tail):
    """(L(x + h d) - L(x - h d)) / 2h against the gradient: h^2 / 6 of a third derivative below 8 |d|^3
    max norm 1, and 2^-23 of a loss below 8 over h: 1e-3 at h = 0.02 holds both."""
    x, ids, lp = make(cuda, 16, 2003, 12, "f32", seed=12, lift=6.0)
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(4)).to(cuda)
    d.scatter_(1, ids.long(), torch.sign(torch.randn(ids.shape, generator=torch.Generator().manual_seed(5))).to(cuda))
    d = d.clamp(-1, 1)
    h = 0.02
    _, grad = ops.distill_loss_and_grad(x, ids, lp, tail=tail)
    up, down = ops.distill_loss(x + h * d, ids, lp, tail=tail), ops.distill_loss(x - h * d, ids, lp, tail=tail)
    slope = (up.double() - down.double()) / (2 * h)
    assert ((slope - (grad.double() * d).sum(1)).abs() <= 1e-3).all()
    assert float((grad.double() * d).sum(1).abs().max()) > 0.05


def test_gradients_of_broadcast_inputs(cuda):
    x, ids, lp = make(cuda, 1, 3001, 9, "f32", seed=13)
    leaf = x.clone().requires_grad_(True)
    w = torch.tensor([1.0, 2.0, 0.0, 0.5], device=cuda)
    loss = ops.distill_loss(leaf.expand(4, -1), ids.expand(4, -1), lp.expand(4, -1), w)
    loss.sum().backward()
    _, one = ops.distill_loss_and_grad(x, ids, lp)
    assert torch.allclose(leaf.grad, 3.5 * one, rtol=0, atol=4 * TOL)


def test_teacher_is_what_the_sampler_returns(cuda):
    """Columns 1.. of the sampler's logprobs, as they are (strided)."""
    x, _, _ = make(cuda, 8, 8000, 4, "f32", seed=14)
    r = ops.sample(x, num_logprobs=20)
    ids, lp = r.logprob_ids[:, 1:], r.logprob_vals[:, 1:]
    student = x + torch.randn(x.shape, generator=torch.Generator().manual_seed(6)).to(cuda)
    check(student, ids, lp, tail="bucket")
    loss, grad = ops.distill_loss_and_grad(x, ids, lp, tail="bucket")
    assert loss.abs().max() <= TOL and grad.abs().max() <= TOL      # the teacher itself


def test_strides_and_alignment(cuda):
    x, ids, lp = make(cuda, 9, 4111, 11, "bf16", seed=15)
    want, want_grad = ops.distill_loss_and_grad(x, ids, lp, tail="bucket")
    for off in (1, 2, 5):
        wide = torch.full((9, 4150), float("nan"), dtype=x.dtype, device=cuda)
        wide[:, off:off + 4111] = x
        out = torch.full((9, 4180), 7.0, dtype=x.dtype, device=cuda)
        loss, grad = ops.distill_loss_and_grad(wide[:, off:off + 4111], ids, lp, tail="bucket", out=out[:, 3:4114])
        assert torch.allclose(loss, want, rtol=0, atol=TOL) and torch.equal(out[:, 3:4114], grad)
        assert torch.allclose(grad.float(), want_grad.float(), rtol=2 ** -7, atol=2 * TOL)
        assert bool((out[:, :3] == 7).all()) and bool((out[:, 4114:] == 7).all())
        # in place, in the padded tensor
        ops.distill_loss_and_grad(wide[:, off:off + 4111], ids, lp, tail="bucket", out=wide[:, off:off + 4111])
        assert torch.equal(wide[:, off:off + 4111], grad) and torch.isnan(wide[:, :off]).all()
        assert torch.isnan(wide[:, off + 4111:]).all()
    loss, grad = ops.distill_loss_and_grad(x.t().contiguous().t(), ids.long(), lp.double(), tail="bucket")
    assert torch.equal(grad, want_grad)


def test_more_rows_than_a_launch_takes(cuda):
    """Launches of 8192 rows: the boundary, and a short one after it that is split further."""
    N, V = 8192 + 7, 4300
    x, ids, lp = make(cuda, 40, V, 5, "bf16", seed=16)
    rep = -(-N // 40)
    x, ids, lp = x.repeat(rep, 1)[:N], ids.repeat(rep, 1)[:N], lp.repeat(rep, 1)[:N]
    g = torch.linspace(0.1, 1.0, N, device=cuda)
    for tail in ("renormalize", "bucket"):
        loss, grad = ops.distill_loss_and_grad(x, ids, lp, tail=tail, grad_output=g)
        for part in (slice(0, 40), slice(8180, N)):
            want, want_grad = reference(x[part], ids[part], lp[part], None, 1.0, tail, g[part])
            close(loss[part], grad[part], want, want_grad, None, g[part], 1.0, x.dtype)


def test_rows_past_32_bits(cuda):
    N, V = 8300, 262144          # 2.2e9 logits
    x = torch.zeros((N, V), dtype=torch.bfloat16, device=cuda)
    y, ids, lp = make(cuda, 4, V, 6, "bf16", seed=17)
    x[-4:] = y
    ids, lp = ids.repeat(N // 4, 1), lp.repeat(N // 4, 1)
    w = torch.zeros(N, device=cuda)
    w[-4:] = 1.0
    loss, grad = ops.distill_loss_and_grad(x, ids, lp, w, tail="bucket", out=x)
    want, want_grad = reference(y, ids[-4:], lp[-4:], None, 1.0, "bucket", torch.ones(4, device=cuda))
    close(loss[-4:], grad[-4:], want, want_grad, None, torch.ones(4, device=cuda), 1.0, y.dtype)
    assert not loss[:-4].any() and not grad[-6:-4].any()


def test_no_rows(cuda):
    x = torch.empty((0, 100), device=cuda, requires_grad=True)
    ids, lp = torch.empty((0, 4), dtype=torch.int32, device=cuda), torch.empty((0, 4), device=cuda)
    ops.distill_loss(x, ids, lp).sum().backward()
    assert x.grad.shape == (0, 100)
    loss, grad = ops.distill_loss_and_grad(x.detach(), ids, lp)
    assert loss.shape == (0,) and grad.shape == (0, 100)


@pytest.mark.parametrize("N", [3, 600])
def test_same_answer_each_time_and_on_another_stream(cuda, N):
    x, ids, lp = make(cuda, 3, 70001, 30, "bf16", seed=18)
    x, ids, lp = (t.repeat(N // 3, 1) for t in (x, ids, lp))
    want = ops.distill_loss_and_grad(x, ids, lp, tail="bucket")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            got.append(ops.distill_loss_and_grad(x, ids, lp, tail="bucket"))
    torch.cuda.synchronize()
    for loss, grad in got:
        assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])


def test_a_sampler_call_between_uses_the_same_workspace(cuda):
    """The counters of split rows lie in the region that every operation shares."""
    x, ids, lp = make(cuda, 4, 60000, 30, "f32", seed=19)
    want = ops.distill_loss(x, ids, lp)
    ref = ops.topk(x, 20)
    for _ in range(3):
        v, i = ops.topk(x, 20)
        assert torch.equal(i, ref[1]) and torch.equal(ops.distill_loss(x, ids, lp), want)
        ops.sample(x, temperature=1.0, rng_key=3)


def test_in_a_graph(cuda):
    x, ids, lp = make(cuda, 6, 60011, 30, "bf16", seed=20)
    y, ids2, lp2 = make(cuda, 6, 60011, 30, "bf16", seed=21)
    first = [t.clone() for t in (x, ids, lp)]
    ops.distill_loss_and_grad(x, ids, lp, tail="bucket")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = ops.distill_loss_and_grad(x, ids, lp, tail="bucket")
    for source in (first, (y, ids2, lp2), first, (y, ids2, lp2)):
        for a, b in zip((x, ids, lp), source):
            a.copy_(b)
        want, want_grad = ops.distill_loss_and_grad(*source, tail="bucket")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want) and torch.equal(grad, want_grad)


def test_refusals(cuda):
    x, ids, lp = make(cuda, 3, 300, 4, "f32", seed=22)
    for bad in (dict(tail="other"), dict(teacher_ids=ids[:2]), dict(teacher_logprobs=lp[:, :2]), dict(logits=x[0]),
                dict(logits=x.cpu()), dict(teacher_ids=ids.cpu()), dict(row_weight=torch.ones(2)),
                dict(teacher_ids=torch.zeros((3, 257), dtype=torch.int32, device=cuda),
                     teacher_logprobs=torch.zeros((3, 257), device=cuda)),
                dict(teacher_ids=ids[:, :0], teacher_logprobs=lp[:, :0])):
        with pytest.raises(ValueError):
            ops.distill_loss(**{**dict(logits=x, teacher_ids=ids, teacher_logprobs=lp), **bad})
    with pytest.raises(TypeError):
        ops.distill_loss(x.double(), ids, lp)
    for T in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(_lib.VwsError) as e:
            ops.distill_loss(x, ids, lp, temperature=T)
        assert e.value.status == _lib.ERR_INVALID_ARGUMENT
    for out in (torch.empty((3, 301), device=cuda), torch.empty((3, 300), device=cuda, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            ops.distill_loss_and_grad(x, ids, lp, out=out)
    wide = torch.zeros((6, 300), device=cuda)
    with pytest.raises(_lib.VwsError):       # overlaps the logits without being their memory
        ops.distill_loss_and_grad(wide[:3], ids, lp, out=wide[1:4])
    big = torch.zeros((1, (1 << 19) + 8), device=cuda)
    with pytest.raises(_lib.VwsError) as e:
        ops.distill_loss(big, ids[:1], lp[:1])
    assert e.value.status == _lib.ERR_LIMIT
