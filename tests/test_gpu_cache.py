"""The paged cache's writes against 64-bit forms: appended keys and values with the rotation, accepted nodes moved up."""
from __future__ import annotations

import pytest
import torch

from tests import tree_ref as R
from vllm_webgpu_amd import ops

pytestmark = pytest.mark.gpu


def packed(dev, T, heads, kv_heads, dim, dtype, seed=0):
    """q, k, v as views of one projection's output."""
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn((T, (heads + 2 * kv_heads) * dim), generator=g, device=dev).to(R.DTYPES[dtype])
    return [t.unflatten(1, (-1, dim)) for t in x.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)]


def freqs(dev, rotary, base=10000.0):
    return base ** (-torch.arange(0, rotary, 2, device=dev).float() / rotary)


def check(got, want, off, dtype):
    off = off + R.half_step(R.DTYPES[dtype]) * want.abs() + 1e-30
    bad = (got.double() - want).abs() > off
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / off).max()))


@pytest.mark.parametrize("T,heads,kv_heads,dim,rotary,page,dtype,interleaved", [
    (1, 4, 1, 64, 64, 16, "bf16", False), (7, 6, 2, 128, 128, 8, "f16", False), (65, 8, 8, 96, 48, 32, "bf16", True),
    (200, 3, 3, 256, 256, 64, "f16", True), (131, 10, 5, 192, 16, 256, "bf16", False), (64, 0, 2, 128, 0, 16, "bf16", False),
    (9000, 2, 1, 64, 32, 16, "f16", False),
])
def test_append(cuda, T, heads, kv_heads, dim, rotary, page, dtype, interleaved):
    q, k, v = packed(cuda, T, heads, kv_heads, dim, dtype, seed=T)
    pages = (T + T // 8 + page - 1) // page + 5
    kc, vc = R.make_cache(cuda, pages, kv_heads, page, dim, dtype, seed=1)
    g = torch.Generator().manual_seed(T)
    # runs of tokens from odd places on, some tokens nowhere
    order, slots = torch.randperm(pages, generator=g), []
    at = int(torch.randint(page, (1,), generator=g))
    for _ in range(T):
        slots.append(int(order[at // page]) * page + at % page)
        at += 1 if torch.rand(1, generator=g) < 0.98 else 2
        if at >= pages * page:
            at = 0
    slots = torch.tensor(slots, dtype=torch.int32)
    drop = torch.rand(T, generator=g) < 0.05
    slots[drop] = torch.tensor([-1, -7, pages * page, 2 ** 31 - 1], dtype=torch.int32)[torch.randint(4, (int(drop.sum()),), generator=g)]
    assert len(set(slots[~drop].tolist())) == int((~drop).sum())
    kw = {}
    if rotary:
        kw = dict(positions=torch.randint(0, 1 << 20, (T,), generator=g).int().to(cuda), inv_freq=freqs(cuda, rotary),
                  interleaved=interleaved, rope_scale=0.75)
    ref = dict(kw)
    if ref:
        ref["scale"] = ref.pop("rope_scale")
    wk, wv, off = R.append(k, v, kc, vc, slots, **ref)
    before = q.clone()
    out = ops.append_kv(k, v, kc, vc, slots.to(cuda), q=q if heads else None, **kw)
    check(kc, wk, off, dtype)
    assert torch.equal(vc.double(), wv)
    if heads:
        want, qoff = (q.double(), torch.zeros_like(q.double())) if not kw else R.rotate(q, **{k: v for k, v in ref.items()})
        check(out, want, qoff, dtype)
        assert torch.equal(q, before)
    else:
        assert out is None


def test_append_in_place_keeps_the_rest(cuda):
    """Queries turned where they lie, in one projection's output: its keys and values stay."""
    q, k, v = packed(cuda, 33, 4, 2, 128, "bf16", seed=3)
    kc, vc = R.make_cache(cuda, 6, 2, 16, 128, "bf16")
    pos, f = torch.arange(33, device=cuda).int() + 5, freqs(cuda, 128)
    slots = torch.arange(33, device=cuda).int() + 3
    k0, v0, want = k.clone(), v.clone(), ops.append_kv(k, v, kc.clone(), vc.clone(), slots, q=q, positions=pos, inv_freq=f)
    got = ops.append_kv(k, v, kc, vc, slots, q=q, positions=pos, inv_freq=f, out=q)
    assert got is q and torch.equal(q, want) and torch.equal(k, k0) and torch.equal(v, v0)


def test_append_pages_apart_and_wide_ids(cuda):
    """A layer's pages among other layers'; 64-bit slots and positions past 32 bits."""
    whole = torch.zeros((10, 3, 2, 16, 64), dtype=torch.float16, device=cuda)
    values = torch.zeros((10, 3, 2, 64, 16), dtype=torch.float16, device=cuda)
    q, k, v = packed(cuda, 20, 2, 2, 64, "f16", seed=4)
    slots = torch.arange(20, device=cuda) + 40
    slots[3], slots[5] = 2 ** 32 + 41, -2 ** 40
    ops.append_kv(k, v, whole[:, 1], values[:, 1], slots)
    wk, wv, _ = R.append(k, v, torch.zeros((10, 2, 16, 64), dtype=torch.float16, device=cuda),
                         torch.zeros((10, 2, 64, 16), dtype=torch.float16, device=cuda), slots)
    assert torch.equal(whole[:, 1].double(), wk) and torch.equal(values[:, 1].double(), wv)
    assert not bool(whole[:, [0, 2]].any()) and not bool(values[:, [0, 2]].any())


def test_far_positions_turn_exactly(cuda):
    """At position 2^31 - 1 a 32-bit angle would be off by tens of radians."""
    q = torch.ones((3, 1, 64), dtype=torch.bfloat16, device=cuda)
    kc, vc = R.make_cache(cuda, 1, 1, 8, 64, "bf16")
    pos, f = torch.tensor([2 ** 31 - 1, 2 ** 30 + 1, 0], device=cuda).int(), freqs(cuda, 64, 1e6)
    out = ops.append_kv(q, q, kc, vc, torch.tensor([0, 1, 2], device=cuda).int(), q=q, positions=pos, inv_freq=f)
    want, off = R.rotate(q, pos, f)
    check(out, want, off + 2.0 ** -21, "bf16")   # (2^31 turns in 64 bits leave 2^-22 of one)


def paths(B, width, nodes, g):
    rows = []
    for _ in range(B):
        n = int(torch.randint(0, min(width, nodes) + 1, (1,), generator=g))
        pick = sorted(torch.randperm(nodes - 1, generator=g)[:max(0, n - 1)].add(1).tolist())
        rows.append(([0] + pick if n else []) + [-1] * (width - (1 + len(pick) if n else 0)))
    return torch.tensor(rows, dtype=torch.int32)


@pytest.mark.parametrize("B,kv_heads,dim,page,width,nodes,dtype", [
    (1, 1, 64, 8, 3, 5, "bf16"), (5, 3, 128, 16, 9, 20, "f16"), (17, 2, 256, 32, 40, 256, "bf16"), (3, 4, 96, 64, 256, 256, "f16"),
    (2, 1, 192, 16, 1, 1, "bf16"),
])
def test_compact(cuda, B, kv_heads, dim, page, width, nodes, dtype):
    g = torch.Generator().manual_seed(width)
    context = torch.randint(0, 3 * page, (B,), generator=g)
    need = (3 * page + nodes + page - 1) // page
    kc, vc = R.make_cache(cuda, B * need + 2, kv_heads, page, dim, dtype)
    table = torch.randperm(B * need + 2, generator=g)[:B * need].view(B, need).int()
    path = paths(B, width, nodes, g)
    wk, wv = kc.clone(), vc.clone()
    for b in range(B):
        for j, node in enumerate(path[b].tolist()):
            if node >= 0:
                (p, i), (d, o) = divmod(int(context[b]) + node, page), divmod(int(context[b]) + j, page)
                wk[table[b, d], :, o], wv[table[b, d], :, :, o] = kc[table[b, p], :, i], vc[table[b, p], :, :, i]
    ops.compact_kv(kc, vc, table.to(cuda), context.int().to(cuda), path.to(cuda))
    assert torch.equal(kc, wk) and torch.equal(vc, wv)


def test_compact_leaves_what_lies_in_no_page(cuda):
    kc, vc = R.make_cache(cuda, 4, 2, 8, 64, "bf16")
    k0, v0 = kc.clone(), vc.clone()
    table = torch.tensor([[0, -1], [9, 1], [2, 3], [2, 3]], device=cuda).int()
    context = torch.tensor([5, 2, 14, -3], device=cuda).int()
    path = torch.tensor([[0, 4, 5], [0, 3, 4], [0, 2, 3], [0, 4, 6]], device=cuda).int()
    ops.compact_kv(kc, vc, table, context, path)   # (a source or target in no page, past the table, a bad context)
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


def test_offsets_past_32_bits(cuda):
    """Pages whose elements lie past 2^32 bytes and 2^31 elements."""
    pages, page, dim = 140000, 128, 128                      # 2.3e9 elements each
    kc = torch.zeros((pages, 1, page, dim), dtype=torch.bfloat16, device=cuda)
    vc = torch.zeros((pages, 1, dim, page), dtype=torch.bfloat16, device=cuda)
    q, k, v = packed(cuda, 40, 2, 1, dim, "bf16", seed=9)
    slots = torch.arange(40, device=cuda).int() + (pages - 1) * page + 3
    ops.append_kv(k, v, kc, vc, slots)
    assert torch.equal(kc[-1, 0, 3:43], k[:, 0]) and torch.equal(vc[-1, 0, :, 3:43].T, v[:, 0])
    assert not bool(kc[:-1].any()) and not bool(vc[:-1].any())
    table = torch.tensor([[pages - 1]], device=cuda).int()
    at = lambda *x: torch.tensor(x, device=cuda).int()  # noqa: E731
    cu = at(0, 3)
    out = ops.tree_attention(q[37:].contiguous(), kc, vc, table, at(40), cu, 3)
    want, bound = R.attention(q[37:], kc[-1:], vc[-1:], at(0).unsqueeze(0), [40], [0, 3], None)
    assert bool(((out.double() - want).abs() <= bound).all())
    ops.compact_kv(kc, vc, table, at(3), at(0, 5, 30).unsqueeze(0))
    assert torch.equal(kc[-1, 0, 4:6], k[[5, 30], 0]) and torch.equal(vc[-1, 0, :, 4:6].T, v[[5, 30], 0])


def test_refusals(cuda):
    q, k, v = packed(cuda, 4, 4, 2, 64, "bf16")
    kc, vc = R.make_cache(cuda, 3, 2, 16, 64, "bf16")
    s = torch.arange(4, device=cuda).int()
    f = freqs(cuda, 64)
    bad = [
        (TypeError, dict(k_cache=kc.float(), v_cache=vc.float())), (TypeError, dict(v_cache=vc.half())), (TypeError, dict(k=k.half())),
        (ValueError, dict(v_cache=kc)), (ValueError, dict(k=k[:, :1])), (ValueError, dict(slots=s[:3])), (ValueError, dict(slots=s.cpu())),
        (ValueError, dict(positions=s)), (ValueError, dict(inv_freq=f)), (ValueError, dict(positions=s, inv_freq=f[:5])),
        (ValueError, dict(positions=s, inv_freq=freqs(cuda, 128))), (ValueError, dict(positions=s[:2], inv_freq=f)),
        (ValueError, dict(q=q[:3])), (ValueError, dict(out=q)), (ValueError, dict(q=q, out=k.expand(4, 2, 64))),
        (ValueError, dict(q=q, out=q[:1].expand(4, 4, 64))), (ValueError, dict(k=k.clone().requires_grad_())),
        (ValueError, dict(k_cache=kc.transpose(1, 2), v_cache=vc)), (ops._lib.VwsError, dict(positions=s, inv_freq=f, rope_scale=float("inf"))),
        (ops._lib.VwsError, dict(k_cache=kc[..., :12, :].contiguous(), v_cache=vc[..., :12].contiguous())),
        (ops._lib.VwsError, dict(k=k[..., :32], v=v[..., :32], k_cache=kc[..., :32].contiguous(), v_cache=vc[..., :32, :].contiguous())),
    ]
    for error, change in bad:
        args = {**dict(k=k, v=v, k_cache=kc, v_cache=vc, slots=s), **change}
        with pytest.raises(error):
            ops.append_kv(**args)
    t, c = torch.zeros((1, 2), device=cuda).int(), torch.zeros(1, device=cuda).int()
    for table, context, path in ((t[0], c, t), (t, t, t), (t, c, t[0]), (t, c, torch.zeros((1, 257), device=cuda).int()),
                                 (t, c, torch.zeros((2, 2), device=cuda).int()), (t, c.cpu(), t)):
        with pytest.raises(ValueError):
            ops.compact_kv(kc, vc, table, context, path)


def test_no_tokens(cuda):
    kc, vc = R.make_cache(cuda, 2, 2, 16, 64, "bf16")
    k0 = kc.clone()
    e = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=cuda)
    out = ops.append_kv(e, e, kc, vc, torch.empty(0, device=cuda).int(), q=e)
    assert out.shape == (0, 2, 64) and torch.equal(kc, k0)


@pytest.mark.parametrize("T,interleaved", [(2051, True), (2047, False), (4098, False)])
def test_append_of_several_tokens_a_workgroup(cuda, T, interleaved):
    """Queries turned in place, the last workgroup's tokens fewer, every third head's stride apart."""
    wide = torch.randn((T, 9, 72), device=cuda, generator=torch.Generator(device=cuda).manual_seed(T)).bfloat16()
    q, k, v = wide[:, :4, :64], wide[:, 4:6, :64], wide[:, 6:8, 8:]
    kc, vc = R.make_cache(cuda, T // 16 + 2, 2, 16, 64, "bf16")
    slots, pos = torch.arange(T, device=cuda).flip(0).int(), torch.arange(T, device=cuda).int() * 37
    f = freqs(cuda, 48)
    want, off = R.rotate(q, pos, f, interleaved=interleaved)
    wk, wv, koff = R.append(k, v, kc, vc, slots.cpu(), positions=pos, inv_freq=f, interleaved=interleaved)
    rest = wide[:, 8].clone()
    out = ops.append_kv(k, v, kc, vc, slots, q=q, positions=pos, inv_freq=f, interleaved=interleaved, out=q)
    assert out.data_ptr() == wide.data_ptr() and torch.equal(wide[:, 8], rest)
    check(q, want, off, "bf16")
    check(kc, wk, koff, "bf16")
    assert torch.equal(vc.double(), wv)
