"""The 8-bit cache in plain 64-bit torch: codes and scales of pages, attention over them, and
log-probabilities of tokens.  Independent of the library."""
import math

import torch

F8 = torch.float8_e4m3fn


def scale_of(amax: torch.Tensor) -> torch.Tensor:
    """The smallest 2^e, e >= -126, with 448 * 2^e >= amax."""
    out = torch.full_like(amax, 2.0 ** -126)
    for e in range(-125, 121):
        out = torch.where(amax > 448 * 2.0 ** (e - 1), torch.tensor(2.0 ** e, dtype=amax.dtype,
                                                                    device=amax.device), out)
    return out


def round_codes(y: torch.Tensor) -> torch.Tensor:
    """y to the nearest e4m3 number, ties to even (|y| <= 448); what is not finite becomes NaN."""
    a = y.abs()
    step = torch.full_like(a, 2.0 ** -9)
    for e in range(-5, 9):
        step = torch.where(a >= 2.0 ** e, torch.tensor(2.0 ** (e - 3), dtype=a.dtype, device=a.device), step)
    return torch.where(torch.isfinite(y), torch.round(y / step) * step, math.nan)


def store(x, codes, scales, table, cu, slots, lens, page, cap):
    """The store of x [T, heads, dim]; codes [pages, page, heads, dim] and scales [pages, heads] in
    64 bits, changed in place."""
    n_pages = codes.shape[0]
    x = x.double()
    for b, slot in enumerate(slots):
        n = cu[b + 1] - cu[b]
        if slot < 0 or n == 0:
            continue
        start, last = lens[b] - n, (lens[b] - 1) // page
        for j in range(max(start // page, last - cap // page + 1), last + 1):
            pg = int(table[slot][j % (cap // page)])
            if not 0 <= pg < n_pages:
                continue
            p0, p1 = max(start, j * page), min(lens[b], (j + 1) * page)
            rows = x[cu[b] + p0 - start:cu[b] + p1 - start]
            amax = torch.where(torch.isfinite(rows), rows.abs(), 0.0).amax((0, 2))
            s, r0 = scale_of(amax), p0 - j * page
            if r0:
                s = torch.maximum(s, scales[pg])
                codes[pg, :r0] = round_codes(codes[pg, :r0] * (scales[pg] / s)[None, :, None])
            scales[pg] = s
            codes[pg, r0:r0 + p1 - p0] = round_codes(rows / s[None, :, None])


def visible(p, window, keep_first):
    lo = 0
    if window > 0:
        lo = max(0, p - window + 1)
    elif window < 0:
        lo = p - p % -window
    return list(range(min(keep_first, lo) if window else 0)) + list(range(lo, p + 1))


def attend(q, k_codes, k_scales, v_codes, v_scales, table, slots, positions, page, cap, nh, scale,
           window=0, keep_first=0, sinks=None, bias=None, softcap=0.0):
    """(out [B, nh, hdv], bound of the scores' magnitudes sum |q||k| scale [B, nh], max |v| [B, nh, hdv],
    keys seen [B]) in 64 bits."""
    nkv, hd, hdv = k_codes.shape[2], k_codes.shape[3], v_codes.shape[3]
    B = len(slots)
    q = q.double().reshape(B, nh, hd)
    out = torch.zeros((B, nh, hdv), dtype=torch.float64, device=q.device)
    mag = torch.zeros((B, nh), dtype=torch.float64, device=q.device)
    vmax = torch.zeros_like(out)
    for b in range(B):
        if slots[b] < 0:
            continue
        j = torch.tensor(visible(positions[b], window, keep_first), device=q.device)
        pg = table[slots[b]].long()[j % cap // page]
        k = k_codes[pg, j % page].double() * k_scales[pg].double()[:, :, None]
        v = v_codes[pg, j % page].double() * v_scales[pg].double()[:, :, None]
        for h in range(nh):
            g = h // (nh // nkv)
            s = k[:, g] @ q[b, h] * scale
            mag[b, h] = ((k[:, g].abs() @ q[b, h].abs()) * abs(scale)).max()
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if bias is not None:
                s = s + bias[h].double()[(positions[b] - j).clamp_max(bias.shape[1] - 1)]
            vals = v[:, g]
            vmax[b, h] = vals.abs().amax(0)
            if sinks is not None:
                s = torch.cat([s, sinks[h].double().reshape(1)])
                vals = torch.cat([vals, torch.zeros_like(vals[:1])])
            out[b, h] = torch.softmax(s, 0) @ vals
    return out, mag, vmax, [0 if s < 0 else len(visible(p, window, keep_first))
                            for s, p in zip(slots, positions)]


def logprobs(logits, tokens, top):
    """(logprob, entropy, rank, top ids, top logprobs, sum p |x - m|) of rows of logits."""
    x = logits.double()
    lp = torch.log_softmax(x, 1)
    R, V = x.shape
    logprob = torch.full((R,), math.nan, dtype=torch.float64, device=x.device)
    rank = torch.zeros(R, dtype=torch.int64, device=x.device)
    ids = torch.arange(V, device=x.device)
    for r, t in enumerate(tokens.tolist()):
        if 0 <= t < V:
            logprob[r] = lp[r, t]
            rank[r] = 1 + ((x[r] > x[r, t]) | ((x[r] == x[r, t]) & (ids < t))).sum()
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(1)
    spread = torch.where(p > 0, p * (x - x.amax(1, keepdim=True)).abs(), 0.0).sum(1)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return logprob, entropy, rank, order, lp.gather(1, order), spread
