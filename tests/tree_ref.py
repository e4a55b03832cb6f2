"""Plain 64-bit forms of the paged cache's and drafted trees' operators and of the tokens' log-probabilities, with bounds on what
32-bit arithmetic and the outputs' rounding may be off."""
from __future__ import annotations

import math

import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


# ---- cache ----------------------------------------------------------------------------------------


def make_cache(dev, pages, kv_heads, page, dim, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    k = torch.randn((pages, kv_heads, page, dim), generator=g, device=dev).to(DTYPES[dtype])
    v = torch.randn((pages, kv_heads, dim, page), generator=g, device=dev).to(DTYPES[dtype])
    return k, v


def rotate(x, positions, inv_freq, scale=1.0, interleaved=False):
    """(rotated, bound on a 32-bit rotation's error before the rounding) of x [T, H, D], in 64 bits."""
    R = 2 * inv_freq.numel()
    angle = positions.double()[:, None, None] * inv_freq.double()
    c, s = torch.cos(angle) * scale, torch.sin(angle) * scale
    y, err = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    i = torch.arange(R // 2, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    a, b = x.double()[..., lo], x.double()[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    # the angle's fraction of a turn, its sine, the scale and two products and a sum, each within a few steps of 2^-24
    err[..., lo] = err[..., hi] = 16 * 2.0 ** -24 * abs(scale) * (a.abs() + b.abs())
    return y, err


def append(k, v, k_cache, v_cache, slots, positions=None, inv_freq=None, scale=1.0, interleaved=False):
    """(k_cache, v_cache) in 64 bits after the call, and the keys' bound."""
    page = k_cache.shape[2]
    kc, vc, err = k_cache.double(), v_cache.double(), torch.zeros(k_cache.shape, dtype=torch.float64, device=k.device)
    kr, ke = (k.double(), torch.zeros_like(k.double())) if positions is None else rotate(k, positions, inv_freq, scale, interleaved)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < k_cache.shape[0] * page:
            kc[s // page, :, s % page], vc[s // page, :, :, s % page] = kr[t], v[t].double()
            err[s // page, :, s % page] = ke[t]
    return kc, vc, err


# ---- trees ----------------------------------------------------------------------------------------


def random_tree(n, g, reach=5):
    return [-1] + [max(0, i - 1 - int(torch.randint(reach, (1,), generator=g))) for i in range(1, n)]


def sees(parents):
    """bool [n, n] of one tree: node i sees its ancestors and itself."""
    see = torch.eye(len(parents), dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            see[i] |= see[p]
    return see


def pack(see, width):
    """bool [T, n <= width] -> int32 words [T, ceil(width / 32)]."""
    b = torch.zeros((see.shape[0], (width + 31) // 32 * 32), dtype=torch.int64)
    b[:, :see.shape[1]] = see
    return (b.view(see.shape[0], -1, 32) << torch.arange(32)).sum(2).to(torch.int32)


def attention(q, k_cache, v_cache, table, context, cu, see, scale=None):
    """(out, bound) of every row in 64 bits; see: a list of bool [n, n] per request, or None (a chain)."""
    page, Hk, D = k_cache.shape[2], k_cache.shape[1], k_cache.shape[3]
    T, H = q.shape[:2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    eps = half_step(q.dtype)
    for b, c in enumerate(context):
        n = cu[b + 1] - cu[b]
        pos = torch.arange(c + n)
        pages = table[b].cpu()[pos // page].long().to(q.device)
        off = (pos % page).to(q.device)
        mask = torch.ones((n, c + n), dtype=torch.bool)
        mask[:, c:] = torch.ones((n, n), dtype=torch.bool).tril() if see is None else see[b]
        mask = mask.to(q.device).unsqueeze(1)
        for h in range(Hk):
            k, v = k_cache[pages, h, off].double(), v_cache[pages, h, :, off].double()
            mine = slice(h * (H // Hk), (h + 1) * (H // Hk))
            x = q[cu[b]:cu[b + 1], mine].double()
            s = (x @ k.T) * scale
            off_s = (x.abs() @ k.abs().T) * scale * (D + 4) * 2.0 ** -24     # a 32-bit product's error
            off_s = torch.where(mask, off_s, 0.0).amax(-1, keepdim=True)
            s = torch.where(mask, s, -math.inf)
            m = s.amax(-1, keepdim=True)
            e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
            w = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
            vv = torch.where(mask.any(1).any(0).unsqueeze(1), v, 0.0)        # (what nobody sees may be anything)
            if bool(torch.isfinite(vv).all()):
                o, near = w @ vv, w @ vv.abs()
            else:
                o = torch.where(mask.unsqueeze(-1), w.unsqueeze(-1) * vv, 0.0).sum(2)
                near = o.abs()
            out[cu[b]:cu[b + 1], mine] = o
            # weights rounded to the type, scores' errors in weight and sum, sums of 32 bits, the output's rounding
            bound[cu[b]:cu[b + 1], mine] = eps * o.abs() + near * (eps + 2.5 * off_s + (c + n) * 2.0 ** -24 / 4 + 2.0 ** -19) + 1e-30
            if q.dtype == torch.float16:
                # weights (up to 2^8 relative to the largest) below 2^-14 step by 2^-24
                bound[cu[b]:cu[b + 1], mine] += 2.0 ** -24 * vv.abs().nan_to_num(0, 0, 0).sum(0)
    return out, bound


def walk(sampled, tokens, parents, cu, width):
    """(tokens, path, num_accepted) as lists."""
    outs, paths, counts = [], [], []
    for b in range(len(cu) - 1):
        lo, n = cu[b], cu[b + 1] - cu[b]
        out, path, at = [], [], 0 if n > 0 else None
        while at is not None and len(path) < width:
            path.append(at)
            out.append(sampled[lo + at])
            fit = [j for j in range(at + 1, n) if parents[lo + j] == at and tokens[lo + j] == out[-1]]
            at = fit[0] if fit else None
        counts.append(len(path) - 1)
        outs.append(out + [-1] * (width - len(out)))
        paths.append(path + [-1] * (width - len(path)))
    return outs, paths, counts


# ---- log-probabilities ----------------------------------------------------------------------------


def logprobs(x, ids, temperature=1.0, top=None):
    """A dict in 64 bits: logprobs, entropy, ids, vals, ranks, and the bounds of the first two's errors (and vals')."""
    N, V = x.shape
    live = (ids >= 0) & (ids < V)
    at = torch.where(live, ids, 0).long().unsqueeze(1)
    z = x.double() / temperature
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    mine = torch.where(live, logp.gather(1, at).squeeze(1), 0.0)
    entropy = torch.where(live, -torch.where(p > 0, p * logp, 0.0).sum(1), 0.0)
    # a sum's 32-bit accumulators take V / 1024 terms each, then some merges; the exponents' rounding of |z - max|
    sums = (V / 1024 + 64) * 2.0 ** -24
    gap = (z - z.amax(1, keepdim=True)).abs()
    far = torch.where(p > 0, p * gap, 0.0).sum(1)
    o = {"logprobs": mine, "entropy": entropy, "live": live,
         "logprobs_off": sums + 2.0 ** -22 * (gap.gather(1, at).squeeze(1) + far + mine.abs() + 1),
         "entropy_off": (sums + 2.0 ** -22 * (1 + far)) * (2 + 2 * far + entropy)}
    if top is not None:
        xv = x.float() + 0.0
        # (the larger value, then the lower index; a NaN is never among them)
        key = torch.where(xv.isnan(), torch.tensor(-math.inf, device=x.device), xv)
        order = torch.sort(key, dim=1, descending=True, stable=True).indices
        order = torch.gather(order, 1, torch.sort(xv.gather(1, order).isnan().int(), dim=1, stable=True).indices)[:, :top]
        o["ids"] = torch.where(live.unsqueeze(1), torch.cat([at, order], 1), -1)
        o["vals"] = torch.where(live.unsqueeze(1), torch.cat([logp.gather(1, at), logp.gather(1, order)], 1), 0.0)
        o["vals_off"] = sums + 2.0 ** -22 * (torch.cat([gap.gather(1, at), gap.gather(1, order)], 1) + far.unsqueeze(1) + 1)
        o["ranks"] = torch.where(live, (x.float() >= x.float().gather(1, at)).sum(1), 0)
    return o


def logprobs_grad(x, ids, gl, gh, temperature=1.0):
    """(gradient, bound) in 64 bits."""
    N, V = x.shape
    live = ((ids >= 0) & (ids < V)).unsqueeze(1)
    at = torch.where(live, ids.unsqueeze(1), 0).long()
    logp = torch.log_softmax(x.double() / temperature, 1)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    H = -plogp.sum(1, keepdim=True)
    gl, gh = gl.double().unsqueeze(1) / temperature, gh.double().unsqueeze(1) / temperature
    one = torch.zeros_like(p).scatter_(1, at, 1.0)
    g = torch.where(live, gl * (one - p) - gh * (plogp + p * H), 0.0)
    part = gl.abs() * (one + p) + gh.abs() * (plogp.abs() + p * (H + 1))
    z = x.double() / temperature
    gap = torch.where(p > 0, (z - z.amax(1, keepdim=True)).abs(), 0.0)
    off = part * ((V / 1024 + 64) * 2.0 ** -24 * (4 + 2 * H) + 2.0 ** -22 * (gap + 4))
    return g, torch.where(live, off + half_step(x.dtype) * g.abs(), 0.0) + torch.finfo(x.dtype).smallest_normal * half_step(x.dtype) * 2
