"""Plain 64-bit references of draft verification and of the distillation loss, for the GPU tests."""
from __future__ import annotations

import numpy as np
import torch

from oracle import sampler as O


def kept_row(x, T, k, p, min_p):
    """(probabilities in float64 with zeros at cut tokens, whether the cut is a near tie) of one row
    by the sampler's rules: y = fl32(x / T); min-p on fl32(y - max); top-k keeps ties of the k-th;
    top-p removes, in (y, index) order from below, while the running mass stays <= (1 - p) W (a sum
    within 1e-6 W of that is decided by the masses floor(exp 2^44), as the sampler does)."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore", divide="ignore"):
        y = (x / np.float32(T)).astype(np.float32)
    ok = ~np.isnan(y)
    m = y[ok].max()
    with np.errstate(invalid="ignore"):
        d = (y - m).astype(np.float32)
        e = np.where(ok, np.exp(np.where(ok, d, 0).astype(np.float64)), 0.0)
    keep = ok.copy()
    near = False
    if min_p > 0:
        bound = np.log(np.float64(min(np.float32(min_p), 1.0)))
        keep &= np.where(ok, d, -np.inf) >= bound
        fin = d[ok & np.isfinite(d)].astype(np.float64)
        near |= bool((np.abs(fin - bound) < 1e-6).any()) and min_p < 1
    if 0 < k < x.size and k <= ok.sum():
        keep &= ok & (y >= np.sort(y[ok])[-k])
    q32 = np.float32(1.0) - np.float32(p)
    if q32 > 0:
        idx = np.nonzero(keep)[0]
        idx = idx[np.lexsort((idx, y[idx]))]
        c = np.cumsum(e[idx])
        W = c[-1]
        gone = c <= q32 * W if q32 < 1 else np.ones(idx.size, bool)
        gone[-1] = False
        if q32 < 1 and (np.abs(c[:-1] - q32 * W) < 1e-6 * W).any():
            # too close for approximate sums: the sampler's integer masses, which decide it
            mass = [O.mass(O.exp_det(float(v))) for v in d[idx]]
            total = [int(v) for v in np.cumsum(np.array(mass, np.uint64))]
            bound = O.scale_floor(float(q32), total[-1])
            gone = np.array([v <= bound for v in total])
            gone[-1] = False
        keep[idx[gone]] = False
    w = np.where(keep, e, 0.0)
    return w / w.sum(), near


def verify(logits, drafts, cu, K, q, T, k, p, min_p, au, u):
    """Verification of host arrays, request by request.  T, k, p, min_p: [B].  Returns tokens,
    accepted, logprobs and, per request, whether a decision was too close to call in 32 bits."""
    B = len(cu) - 1
    tokens = np.full((B, K + 1), -1, np.int32)
    accepted = np.zeros(B, np.int32)
    lps = np.zeros((B, K + 1), np.float64)
    near = np.zeros(B, bool)
    V = logits.shape[1]
    for b in range(B):
        n = cu[b + 1] - cu[b]
        for i in range(n + 1):
            x = np.asarray(logits[cu[b] + b + i], np.float32)
            fin = x[~np.isnan(x)]
            top = int(np.argmax(np.where(np.isnan(x), -np.inf, x))) if fin.size else 0
            if fin.size and fin.max() == -np.inf:
                top = int(np.nonzero(~np.isnan(x))[0][0])
            sure = not (T[b] >= 1e-5) or fin.size == 0 or not np.isfinite(fin.max())
            d = int(drafts[cu[b] + i]) if i < n else -1
            inside = 0 <= d < V
            if sure:
                if i < n and inside and d == top:
                    tokens[b, i] = d
                    continue
                tokens[b, i] = top
                accepted[b] = i
                break
            prob, nt = kept_row(x, T[b], k[b], p[b], min_p[b])
            near[b] |= nt
            weight = prob
            if i < n:
                row = None if q is None else np.asarray(q[cu[b] + i], np.float64)
                qd = 0.0 if not inside else (1.0 if q is None else row[d])
                pd = prob[d] if inside else 0.0
                lhs = float(au[cu[b] + i]) * qd
                near[b] |= abs(lhs - pd) <= 1e-5 * max(pd, 1e-300) and qd > 0
                if qd > 0 and lhs < pd:
                    tokens[b, i] = d
                    lps[b, i] = np.log(pd)
                    continue
                if q is not None:
                    weight = np.maximum(prob - row, 0.0)
                elif inside:
                    weight = prob.copy()
                    weight[d] = 0.0
            with np.errstate(divide="ignore", invalid="ignore"):
                key = np.where(weight > 0, weight / -np.log(u[b].astype(np.float64)), 0.0)
            order = np.argsort(-key, kind="stable")[:2]
            t = int(order[0]) if key[order[0]] > 0 else top
            # a residual p - q rounds to 2^-24 p: its relative error grows as it cancels
            slack = 1e-5 + (2e-7 * prob[order] / np.maximum(weight[order], 1e-300)).max()
            near[b] |= key.size > 1 and key[order[0]] > 0 and key[order[1]] >= key[order[0]] * (1 - slack)
            tokens[b, i] = t
            lps[b, i] = np.log(prob[t])
            accepted[b] = i
            break
    return tokens, accepted, lps, near


def distill(logits, ids, lp, weight=None, T=1.0, tail="renormalize"):
    """Loss [N] in float64, differentiable in ``logits`` (any device)."""
    N, V = logits.shape
    z = logits.double() / T
    logq = torch.log_softmax(z, 1)
    valid = (ids >= 0) & (ids < V)
    at = torch.where(valid, ids, 0).long()
    lq = logq.gather(1, at)
    l = torch.where(valid, lp.double(), float("-inf"))
    if tail == "renormalize":
        live = (l > float("-inf")).any(1)
        l = torch.log_softmax(torch.where(live.unsqueeze(1), l, 0.0) / T, 1)
    else:
        live = valid.any(1)
    p = torch.where(valid, l.exp(), 0.0)
    terms = torch.where(p > 0, p * (torch.where(p > 0, l, 0.0) - torch.where(p > 0, lq, 0.0)), 0.0)
    loss = terms.sum(1)
    if tail == "bucket":
        r = (1.0 - p.sum(1)).clamp(min=0.0)
        inside = torch.zeros((N, V + 1), dtype=torch.bool, device=logits.device)
        inside.scatter_(1, torch.where(valid, ids.long(), V), True)
        rest = torch.where(inside[:, :V], float("-inf"), z)
        have = torch.isfinite(rest).any(1)
        rest = torch.where(have.unsqueeze(1), rest, 0.0)
        log_s = torch.logsumexp(rest, 1) - torch.logsumexp(z, 1)
        on = have & (r > 0)
        loss = loss + torch.where(on, r * (torch.log(torch.where(on, r, 1.0)) - torch.where(on, log_s, 0.0)), 0.0)
    w = torch.ones(N, dtype=torch.float64, device=logits.device) if weight is None else weight.double()
    return torch.where(live & (w != 0), w * torch.where(live, loss, 0.0), 0.0)
