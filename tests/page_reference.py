"""The ops over paged 8-bit caches and the choice of tokens in NumPy, 64 bits, from their definitions."""
import math

import numpy as np


def turn(heads, angle, turn_at, rot, layout):
    """heads [.., dk] at the angles [rot / 2], in 64 bits."""
    h = heads.astype(np.float64).copy()
    i = np.arange(rot // 2)
    x, y = (2 * i, 2 * i + 1) if layout == "pairs" else (i, i + rot // 2)
    x, y = x + turn_at, y + turn_at
    a, b, c, s = h[..., x].copy(), h[..., y].copy(), np.cos(angle), np.sin(angle)
    h[..., x], h[..., y] = a * c - b * s, a * s + b * c
    return h


def scale_for(most):
    """The smallest power of two, 2^-126 at least, of which 127 times reach `most`."""
    if not np.isfinite(most):
        return np.nan
    e = -126
    if most > 0:
        e = max(e, math.frexp(most)[1] - 8)
    while 127 * 2.0 ** e < most:
        e += 1
    return 2.0 ** e


def append(keys, values, scales, src, page_table, entries, live, prefix, cols, B, G, dk, dv, page, turn_at=0, rot=0, freqs=None, layout="pairs", q_heads=0, turned=None):
    """New codes, scales and turned queries; cols: key, value and query columns of src.  Codes of positions that nothing has written are whatever they were."""
    keys, values, scales = keys.astype(np.float64), values.astype(np.float64), scales.astype(np.float64)
    turned = None if turned is None else turned.astype(np.float64)
    pages, (slots, most) = len(keys), page_table.shape
    joins = {}
    for r in range(min(max(live, 0), B)):
        slot, length = entries[r][:2]
        if slot < 0:
            continue
        bad = slot >= slots or not 0 <= length <= most * page or prefix < 0
        if not bad and length > 0:
            p = page_table[slot, (length - 1) // page]
            bad = not 0 <= p < pages
            if not bad:
                joins.setdefault((slot, (length - 1) // page, int(p)), {})[(length - 1) % page] = r
        angle = (prefix + length - 1.0) * np.asarray(freqs if rot else [], np.float64)
        if q_heads:
            q = src[r, cols[2]:cols[2] + q_heads * dk].reshape(q_heads, dk)
            turned[r] = np.nan if bad else turn(q, angle, turn_at, rot, layout).ravel()
    for (slot, nth, p), tokens in joins.items():
        k = {}
        for t, r in tokens.items():
            angle = (prefix + nth * page + t + 0.0) * np.asarray(freqs if rot else [], np.float64)
            with np.errstate(all="ignore"):
                k[t] = turn(src[r, cols[0]:cols[0] + G * dk].reshape(G, dk), angle, turn_at, rot, layout).astype(np.float32).astype(np.float64)
        v = {t: src[r, cols[1]:cols[1] + G * dv].reshape(G, dv).astype(np.float64) for t, r in tokens.items()}
        for which, codes, new in ((0, keys, k), (1, values, v)):
            for g in range(G):
                before = 0.0 if 0 in tokens else scales[p, g, which]
                need = scale_for(max(np.abs(x[g]).max() if np.isfinite(x[g]).all() else np.inf for x in new.values()))
                after = np.nan if np.isnan(before) or np.isnan(need) else max(before, need)
                if 0 not in tokens and not np.isnan(after):
                    codes[p, g] = np.rint(codes[p, g] * (before / after))
                scales[p, g, which] = after
                for t, x in new.items():
                    if not np.isnan(after):
                        codes[p, g, t] = np.rint(x[g] / after)
    return keys, values, scales, turned


def read(keys, values, scales, page_table, entries, live, B, dst):
    """dst [B, G * (dk + dv)]."""
    dst, page, (slots, most) = dst.astype(np.float64), keys.shape[2], page_table.shape
    for r in range(min(max(live, 0), B)):
        slot, length = entries[r][:2]
        if slot < 0:
            continue
        if slot >= slots or not 0 <= length <= most * page:
            dst[r] = np.nan
        elif length == 0:
            dst[r] = 0.0
        else:
            p, t = page_table[slot, (length - 1) // page], (length - 1) % page
            dst[r] = np.nan if not 0 <= p < len(keys) else np.concatenate([(keys[p, :, t] * scales[p, :, :1]).ravel(), (values[p, :, t] * scales[p, :, 1:]).ravel()])
    return dst


def attend(dst, q, keys, values, scales, page_table, entries, live, B, scale, window=0, cap=0.0, sink=None):
    """(dst [B, H, dv], how far a kernel may be off).  A score is a sum of dk products of exact codes and queries of 45 bits of their largest element, exact but for the rounding of the parts that are joined:
    2^-21 of the sum of magnitudes, and 2^-23 of it for 16 products, are above both (as they are for operands of 22 bits).  Weights come from exponentials of base 2 (2^-22, and their argument's rounding) and are
    32 bits of the largest contribution, outputs exact sums that are rounded and joined after 512 tiles and between warps (a rounding for 32 keys is above that)."""
    dst, tol = dst.astype(np.float64), np.zeros(dst.shape)
    page, (slots, most), H = keys.shape[2], page_table.shape, q.shape[1]
    G, dk = keys.shape[1], keys.shape[3]
    for r in range(min(max(live, 0), B)):
        slot, length = entries[r][:2]
        if slot < 0:
            continue
        if slot >= slots or not 0 <= length <= most * page:
            dst[r] = np.nan
            continue
        lo = max(0, length - window) if window else 0
        ids = page_table[slot, lo // page:-(-length // page)]
        if length and ((ids < 0) | (ids >= len(keys))).any():
            dst[r] = np.nan
            continue
        if length == 0:
            dst[r] = 0.0
            continue
        at = np.arange(lo, length) - lo // page * page
        for g in range(G):
            k = (keys[ids, g] * scales[ids, g, 0].astype(np.float64)[:, None, None]).reshape(-1, dk)[at]
            v = (values[ids, g] * scales[ids, g, 1].astype(np.float64)[:, None, None]).reshape(-1, values.shape[3])[at]
            for h in range(g * (H // G), (g + 1) * (H // G)):
                with np.errstate(all="ignore"):
                    x = q[r, h].astype(np.float64)
                    s = k @ x * scale
                    off = abs(scale) * (np.abs(k) @ np.abs(x)) * (2.0 ** -21 + (dk + 15) // 16 * 2.0 ** -23) + 2.0 ** -22 * np.abs(s)
                    if cap:
                        s = cap * np.tanh(s / cap)
                    top = max(s.max(), -np.inf if sink is None else sink[h])
                    p = np.exp(s - top)
                    total = p.sum() + (0.0 if sink is None else math.exp(sink[h] - top))
                    dst[r, h] = p @ v / total
                    spread = np.abs(s - top)
                    error = off + 2.0 ** -21 + 2.0 ** -23 * np.minimum(spread, 200.0)
                    average = p @ error / total
                    tol[r, h] = (p * (error + average)) @ np.abs(v) / total + (p @ np.abs(v) / total) * (16 + len(at) / 32) * 2.0 ** -23 + 1e-37
    return dst, tol


def sample(logits, choice, u):
    """(token, probability) of one row; choice: (temperature, top_k, top_p, min_p)."""
    z, (temperature, top_k, top_p, min_p) = logits.astype(np.float64), choice
    temperature, top_p, min_p, u = (float(np.float32(x)) for x in (temperature, top_p, min_p, u))
    if np.isnan(z).any() or z.max() == -np.inf or not (0 <= temperature < np.inf and 0 <= top_p <= 1 and 0 <= min_p <= 1 and 0 <= u < 1):
        return -1, np.nan
    if temperature == 0:
        return int(np.argmax(z)), 1.0
    with np.errstate(all="ignore"):
        e = np.where(z == z.max(), 1.0, np.exp((z - z.max()) / temperature))
    order = np.argsort(-z, kind="stable")
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        sums = np.cumsum(e[order])
        order = order[:1 + int(np.searchsorted(sums, top_p * sums[-1], side="left"))]
    with np.errstate(all="ignore"):                      # (as exponents: e^x of a small negative x rounds to 1, which is not what a min_p of 1 lets through)
        exponent = np.where(z == z.max(), 0.0, (z - z.max()) / temperature)
        stays = np.sort(order[exponent[order] >= np.log(min_p)])
    sums = np.cumsum(e[stays])
    token = int(stays[np.searchsorted(sums, u * sums[-1], side="right")])
    return token, e[token] / sums[-1]
