"""Log-probabilities of given tokens, with entropy, ranks, top alternatives and gradients, against 64-bit forms."""
from __future__ import annotations

import pytest
import torch

from tests import tree_ref as R
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def make(dev, N, V, dtype, seed=0, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn((N, V), generator=g, device=dev) * spread
    at = torch.randint(V, (N, min(8, V)), generator=g, device=dev)
    x.scatter_(1, at, x.gather(1, at) + 6.0)
    ids = torch.where(torch.rand(N, generator=g, device=dev) < 0.5, at[:, 0], torch.randint(V, (N,), generator=g, device=dev))
    return x.to(R.DTYPES[dtype]), ids.int()


def near(got, want, off, what=""):
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine) and torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)].double(), want[~fine & ~torch.isnan(want)]), what
    d = (got.double() - want).abs()[fine]
    assert bool((d <= off[fine]).all()), (what, float((d / off[fine]).max()))


def check(x, ids, temperature=1.0, top=5):
    r = ops.token_logprobs(x, ids, top, True, temperature)
    w = R.logprobs(x, ids, temperature, top)
    near(r.logprobs, w["logprobs"], w["logprobs_off"], "logprobs")
    near(r.entropy, w["entropy"], w["entropy_off"], "entropy")
    assert torch.equal(r.logprob_ids.long(), w["ids"])
    near(r.logprob_vals, w["vals"], w["vals_off"], "vals")
    assert torch.equal(r.logprob_ranks.long(), w["ranks"])
    # the other forms give the same
    for kw in (dict(), dict(entropy=True), dict(num_logprobs=top)):
        s = ops.token_logprobs(x, ids, temperature=temperature, **kw)
        near(s.logprobs, w["logprobs"], w["logprobs_off"], kw)
        assert (s.entropy is None) == ("entropy" not in kw) and (s.logprob_ids is None) == ("num_logprobs" not in kw)
        if "num_logprobs" in kw:
            assert torch.equal(s.logprob_ids, r.logprob_ids) and torch.equal(s.logprob_ranks, r.logprob_ranks)
    return r


@pytest.mark.parametrize("N,V,dtype,top,temperature", [
    (1, 1, "f32", 1, 1.0), (3, 5, "bf16", 5, 0.7), (2, 63, "f16", 0, 1.0), (1, 1000, "f32", 64, 2.0), (7, 50257, "f32", 5, 1.0),
    (1, 262144, "bf16", 64, 1.0), (33, 8191, "f16", 20, 0.5), (900, 4097, "bf16", 20, 1.0), (300, 32000, "f32", 1, 1.3),
    (2, 524288, "f32", 64, 1.0), (5, 151937, "bf16", 64, 1.0), (8200, 300, "f32", 3, 1.0), (17, 2049, "bf16", 64, 1.0),
])
def test_logprobs(cuda, N, V, dtype, top, temperature):
    x, ids = make(cuda, N, V, dtype, seed=N + V)
    check(x, ids, temperature, top)


def test_padding_rows(cuda):
    x, ids = make(cuda, 6, 9000, "f32", seed=1)
    wide = ids.long()
    wide[1], wide[3], wide[4] = -1, 9000, 2 ** 32 + 5
    x[[1, 3, 4]] = float("nan")
    r = ops.token_logprobs(x, wide, 4, True)
    live = [0, 2, 5]
    w = R.logprobs(x[live], ids[live], 1.0, 4)
    near(r.logprobs[live], w["logprobs"], w["logprobs_off"])
    for t in (r.logprobs, r.entropy, r.logprob_vals, r.logprob_ranks):
        assert not bool(t[[1, 3, 4]].any())
    assert bool((r.logprob_ids[[1, 3, 4]] == -1).all())


@pytest.mark.parametrize("V", [700, 40000])
@pytest.mark.parametrize("low", [-float("inf"), -1e10, -3.4028234663852886e38])
def test_masked_rows(cuda, V, low):
    """All but a few tokens masked: fewer than the alternatives that are asked for, by index then."""
    x, ids = make(cuda, 4, V, "f32", seed=2)
    keep = torch.zeros((4, V), dtype=torch.bool, device=cuda)
    keep[0, [3, V - 1]] = True
    keep[1, 100:130] = True
    keep[2] = True
    keep[2, ::2] = False
    keep[3, 7] = True
    x = torch.where(keep, x, low)
    ids = torch.tensor([3, 110, 1, 8], device=cuda).int()    # (the last a masked one)
    check(x, ids, 1.0, 20)


def test_ties(cuda):
    """Equal logits at the last place of the list, constant rows, zeros of both signs, one thread's logits above all others."""
    V = 60000
    x = torch.zeros((6, V), device=cuda)
    x[1] = -5.5
    x[2, ::3] = -0.0
    x[3] = torch.randn(V, device=cuda).round()
    x[4, 1024 * 4:1024 * 4 + 4] = 3.0
    for i in range(4):                                        # vectors of one thread: every 1024th element and the next three
        x[5, i + torch.arange(0, V - 8, 1024, device=cuda)] = torch.arange(0, V - 8, 1024, device=cuda).float() + 1.0
    ids = torch.tensor([V - 1, 0, 3, 17, 4097, 4096], device=cuda).int()
    for top in (1, 30, 64):
        check(x, ids, 1.0, top)
    check(x.bfloat16(), ids, 1.0, 64)


def test_many_above_the_threshold(cuda):
    """More than a candidate list's logits in few threads' shares."""
    V = 262144
    x = torch.randn((1, V), device=cuda) * 0.1
    at = torch.arange(V, device=cuda)
    mine = (at // 4) % 256 < 20                               # twenty threads' vectors
    x[0, mine] = 10.0 + torch.rand(int(mine.sum()), device=cuda)
    for n in (1, 900):
        check(x.expand(n, V)[:, :].contiguous() if n == 1 else x.expand(n, V)[:, :40000].contiguous(),
              torch.full((n,), 5, device=cuda).int(), 1.0, 64)


def test_rows_that_are_not_numbers(cuda):
    x, ids = make(cuda, 4, 5000, "f32", seed=3)
    x[0, 77] = float("nan")
    x[1, 99] = float("inf")
    x[2] = -float("inf")
    r = ops.token_logprobs(x, ids, 3, True)
    assert bool(torch.isnan(r.logprobs[:3]).all()) and bool(torch.isnan(r.entropy[:3]).all()) and bool(torch.isfinite(r.logprobs[3]))
    order = torch.sort(x[0].nan_to_num(-1e30), descending=True, stable=True).indices[:3]
    assert r.logprob_ids[0, 1:].tolist() == order.tolist() and int(r.logprob_ids[1, 1]) == 99
    assert r.logprob_ids[2, 1:].tolist() == [0, 1, 2]
    y = torch.full((1, 100), float("nan"), device=cuda)
    y[0, 5] = 1.0
    r = ops.token_logprobs(y, torch.tensor([5], device=cuda), 3)
    assert r.logprob_ids.tolist() == [[5, 5, -1, -1]] and bool(torch.isnan(r.logprob_vals).all())


def test_large_finite_logits(cuda):
    """A row far from zero, where a product's rounding would move every exponential."""
    x, ids = make(cuda, 3, 3001, "f32", seed=4)
    x[0] += 1e7
    x[1] -= 1e9
    x[2] = x[2] * 1e4
    check(x, ids, 1.0, 8)


@pytest.mark.parametrize("N,V,dtype,temperature", [(1, 1, "f32", 1.0), (5, 1003, "f32", 0.7), (40, 50257, "bf16", 1.0), (3, 262144, "f16", 1.5),
                                                    (600, 2048, "bf16", 1.0), (8200, 130, "f32", 2.0)])
def test_gradient(cuda, N, V, dtype, temperature):
    x, ids = make(cuda, N, V, dtype, seed=N)
    ids[::4] = -1
    g = torch.Generator(device=cuda).manual_seed(N)
    gl, gh = (torch.randn(N, generator=g, device=cuda) for _ in range(2))
    if N > 2:
        gl[1] = gh[1] = 0.0
    x.requires_grad_()
    for a, b in ((gl, gh), (gl, None), (None, gh)):
        r = ops.token_logprobs(x, ids, None if a is None else 0, True, temperature)
        got, = torch.autograd.grad([t for t, u in ((r.logprobs, a), (r.entropy, b)) if u is not None], [x],
                                   [u for u in (a, b) if u is not None])
        zero = torch.zeros(N, device=cuda)
        want, off = R.logprobs_grad(x.detach(), ids, zero if a is None else a, zero if b is None else b, temperature)
        assert got.dtype == x.dtype
        near(got, want, off)


def test_gradient_against_differences(cuda):
    x, ids = make(cuda, 2, 37, "f32", seed=6)
    x.requires_grad_()
    r = ops.token_logprobs(x, ids, entropy=True, temperature=0.8)
    (r.logprobs.sum() + 0.5 * r.entropy.sum()).backward()
    y = x.detach().double()

    def loss(z):
        w = R.logprobs(z, ids, 0.8)
        return float((w["logprobs"] + 0.5 * w["entropy"]).sum())

    for i, j in ((0, 0), (0, int(ids[0])), (1, 36), (1, int(ids[1])), (1, 5)):
        h = torch.zeros_like(y)
        h[i, j] = 1e-5
        d = (loss(y + h) - loss(y - h)) / 2e-5
        assert abs(d - float(x.grad[i, j])) < 1e-5     # (differences: some 1e-10 / 2e-5; the kernel: 2^-24 of terms of some 10)


def test_gradient_of_masked_rows(cuda):
    x, ids = make(cuda, 3, 5000, "f32", seed=7)
    x[0, 50:] = -float("inf")
    x[1, 50:] = -3.4028234663852886e38
    x[2] -= 1e9
    ids[:] = 4
    x.requires_grad_()
    r = ops.token_logprobs(x, ids, entropy=True)
    gl, gh = torch.tensor([1.0, 1.0, -2.0], device=cuda), torch.tensor([0.3, 0.3, 1.0], device=cuda)
    got, = torch.autograd.grad([r.logprobs, r.entropy], [x], [gl, gh])
    want, off = R.logprobs_grad(x.detach(), ids, gl, gh)
    near(got, want, off)
    assert not bool(got[:2, 50:].any())


def test_graphs_beside_each_other(cuda):
    """Two eager graphs of the same leaf, backward in either order; strided logits."""
    base, ids = make(cuda, 20, 1000, "bf16", seed=8)
    x = torch.zeros((20, 1100), dtype=torch.bfloat16, device=cuda)
    x[:, 30:1030] = base
    x.requires_grad_()
    a = ops.token_logprobs(x[:, 30:1030], ids, entropy=True)
    b = ops.token_logprobs(x[:, 30:1030], ids)
    gb, = torch.autograd.grad(b.logprobs.sum(), x)
    ga, = torch.autograd.grad(a.logprobs.sum(), x)
    assert torch.equal(ga, gb) and not bool(ga[:, :30].any()) and bool(ga[:, 30:].any())
    with torch.no_grad():
        r = ops.token_logprobs(x[:, 30:1030], ids)
    assert torch.equal(r.logprobs, a.logprobs) and not r.logprobs.requires_grad


def test_gradients_twice_and_not_of_gradients(cuda):
    """A retained graph gives its gradient again; with create_graph the gradient is the same and has none of its own; saved
    tensors that went through host memory, and logits changed in between."""
    x, ids = make(cuda, 7, 900, "f32", seed=10)
    x.requires_grad_()
    g = torch.linspace(-1, 1, 7, device=cuda)
    r = ops.token_logprobs(x, ids, 2, True)
    a, = torch.autograd.grad([r.logprobs, r.entropy], [x], [g, g], retain_graph=True)
    b, = torch.autograd.grad([r.logprobs, r.entropy], [x], [g, g], retain_graph=True)
    c, = torch.autograd.grad([r.logprobs, r.entropy], [x], [g, g], create_graph=True)
    assert torch.equal(a, b) and torch.equal(a, c) and a.data_ptr() != b.data_ptr()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(c.sum(), x)
    with torch.autograd.graph.save_on_cpu():
        r = ops.token_logprobs(x, ids, 2, True)
    d, = torch.autograd.grad([r.logprobs, r.entropy], [x], [g, g])
    assert torch.equal(a, d)
    e, = torch.autograd.grad((ops.token_logprobs(x, ids).logprobs.double() * g.double()).sum(), x)   # (an upstream of 64 bits)
    f, = torch.autograd.grad(ops.token_logprobs(x, ids).logprobs, x, g)
    assert torch.equal(e, f)
    with torch.no_grad():
        r = ops.token_logprobs(x, ids)
    y = x * 1.0
    r = ops.token_logprobs(y, ids)
    with torch.no_grad():
        y += 1.0
    with pytest.raises(RuntimeError):
        r.logprobs.sum().backward()


def test_overlapping_rows_are_copied(cuda):
    x, ids = make(cuda, 1, 3000, "f32", seed=9)
    wide, want = x.expand(5, 3000), x.repeat(5, 1)
    ids = torch.arange(5, device=cuda)
    assert torch.equal(ops.token_logprobs(wide, ids, 3).logprob_vals, ops.token_logprobs(want, ids, 3).logprob_vals)


def test_empty_and_refusals(cuda):
    x, ids = make(cuda, 3, 100, "f32")
    r = ops.token_logprobs(x[:0], ids[:0], 4, True)
    assert r.logprob_ids.shape == (0, 5) and r.logprobs.shape == (0,)
    for args in ((x[0], ids), (x, ids[:2]), (x, ids.float()), (x, ids.cpu()), (x, ids, 65), (x, ids, -1), (x[:, :3], ids, 4), (x, ids, 1, True, 0.0),
                 (x, ids, 1, True, float("nan")), (x, ids, 1, True, float("inf")), (x.cpu(), ids)):
        with pytest.raises(ValueError):
            ops.token_logprobs(*args)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.double(), ids)
