"""The ops of a batched step in NumPy, 64 bits, from their definitions."""
import numpy as np


def words(a):
    """int32 words as the f32 slots that carry them."""
    return np.ascontiguousarray(a, np.int32).view(np.float32)


def append(cache, src, table_rows, live, prefix, src_col, cache_col, cols, key_heads, dim, turn_at, rot, base, layout, q_heads, q_col, turned, freqs=None):
    """Later rows over earlier ones.  cache [slots, R, width], src [B, rs], turned [B, q_heads * dim]."""
    cache, turned = cache.astype(np.float64), turned.astype(np.float64)
    f = np.asarray(freqs, np.float64) if freqs is not None else base ** (-2.0 * np.arange(rot // 2) / max(rot, 1))

    def turn(heads, angle):
        h = heads.astype(np.float64).copy()
        if rot:
            i = np.arange(rot // 2)
            x, y = (2 * i, 2 * i + 1) if layout == "pairs" else (i, i + rot // 2)
            x, y = x + turn_at, y + turn_at
            a, b, c, s = h[:, x].copy(), h[:, y].copy(), np.cos(angle), np.sin(angle)
            h[:, x], h[:, y] = a * c - b * s, a * s + b * c
        return h

    for r in range(min(live, len(table_rows))):
        slot, length, _ = table_rows[r]
        if slot < 0:
            continue
        bad = slot >= cache.shape[0] or not 0 <= length <= cache.shape[1] or prefix < 0
        angle = (prefix + length - 1.0) * f
        if not bad and length > 0:
            row = src[r, src_col:src_col + cols].astype(np.float64)
            if key_heads and rot:
                row[:key_heads * dim] = turn(row[:key_heads * dim].reshape(key_heads, dim), angle).ravel()
            cache[slot, length - 1, cache_col:cache_col + cols] = row
        if q_heads:
            turned[r] = np.nan if bad else turn(src[r, q_col:q_col + q_heads * dim].reshape(q_heads, dim), angle).ravel()
    return cache, turned


def attend(dst, q, kc, vc, kp, vp, table_rows, live, prefix, prefix_slot, scale, cap=0.0, sink=None):
    """q [B, H, dk], kc [slots, R, G, dk], vc [slots, R, G, dv], kp [prefix slots, Rp, G, dk] (or None), dst [B, H, dv] -> (dst, how far a result may be off)."""
    dst = dst.astype(np.float64)
    tol = np.zeros_like(dst)
    B, H, dk = q.shape
    G = kc.shape[2]
    for r in range(min(live, len(table_rows))):
        slot, length, _ = table_rows[r]
        if slot < 0:
            continue
        if slot >= kc.shape[0] or not 0 <= length <= kc.shape[1] or prefix < 0 or (prefix > 0 and (kp is None or prefix > kp.shape[1] or not 0 <= prefix_slot < kp.shape[0])):
            dst[r] = np.nan
            continue
        for h in range(H):
            g = h // (H // G)
            k, v = kc[slot, :length, g].astype(np.float64), vc[slot, :length, g].astype(np.float64)
            if prefix:
                k, v = np.concatenate([kp[prefix_slot, :prefix, g].astype(np.float64), k]), np.concatenate([vp[prefix_slot, :prefix, g].astype(np.float64), v])
            if not len(k):
                dst[r, h] = 0.0
                continue
            z = q[r, h].astype(np.float64)
            s = scale * (k @ z)
            # A product of dk f32 terms, each factor held to 2^-22 of the largest magnitude of its row, is off by at most this; a cap has slope one at most.
            off = abs(scale) * ((np.abs(k) @ np.abs(z)).max() * dk * 2.0 ** -24 + 3 * 2.0 ** -22 * np.abs(k).max() * np.abs(z).sum())
            if cap:
                s = cap * np.tanh(s / cap)
            off += 4 * 2.0 ** -24 * np.abs(s).max()
            top = s.max()
            p = np.exp(s - top)
            total = p.sum() + (np.exp(float(sink[h]) - top) if sink is not None else 0.0)
            dst[r, h] = p @ v / total
            # Weights are off by a factor e^(2 off), by a few roundings of exp and of sums that are formed in runs of at most 64 keys and joined in a tree, and by the
            # 2^-22 to which they and the values are held.
            tol[r, h] = (2 * off + (64 + 32) * 2.0 ** -24 + 4 * 2.0 ** -22) * (p @ np.abs(v) / total + np.abs(v).max() * 2.0 ** -14)
    return dst, tol


def adapt(dst, base, x, A, Bm, scales, table_rows, live):
    """A [adapters, rank, K], Bm [adapters, N, rank] -> (dst, how far a result may be off)."""
    dst = dst.astype(np.float64)
    tol = np.zeros_like(dst)
    for r in range(min(live, len(table_rows))):
        slot, _, a = table_rows[r]
        if slot < 0:
            continue
        if a >= len(A):
            dst[r] = np.nan
        elif a < 0:
            dst[r] = base[r]
        else:
            s = 1.0 if scales is None else float(scales[a])
            A64, B64, x64 = A[a].astype(np.float64), Bm[a].astype(np.float64), x[r].astype(np.float64)
            h = A64 @ x64
            dst[r] = base[r].astype(np.float64) + s * (B64 @ h)
            # two chained products: every term of either passes at most K (rank) additions and a few roundings
            grow = (len(x64) + len(h) + 16) * 2.0 ** -24
            tol[r] = grow * abs(s) * (np.abs(B64) @ (np.abs(A64) @ np.abs(x64))) + 2.0 ** -23 * (np.abs(dst[r]) + np.abs(base[r]))
    return dst, tol


def rules(dst, logits, rows, live, history, bias, masks):
    """rows: (slot, length, first, mask, bias first, bias count, repetition, presence, frequency) -> (dst, how far a result may be off)."""
    dst = dst.astype(np.float64)
    tol = np.zeros_like(dst)
    V = logits.shape[1]
    for r in range(min(live, len(rows))):
        slot, length, first, mask, b0, nb, rep, presence, frequency = rows[r]
        if slot < 0:
            continue
        z = logits[r].astype(np.float64)
        size = np.abs(np.where(np.isfinite(z), z, 0.0))
        tokens = np.asarray(history[slot, :length] if length else [], np.int64)
        inside = (tokens >= 0) & (tokens < V)
        seen = np.zeros(V, bool)
        seen[tokens[inside]] = True
        count = np.bincount(tokens[first:][inside[first:]], minlength=V).astype(np.float64)
        with np.errstate(invalid="ignore"):
            z = np.where(seen, np.where(z > 0, z / rep, z * rep), z)
        size = np.maximum(size, np.abs(np.where(np.isfinite(z), z, 0.0))) + presence * (count > 0) + abs(frequency) * count
        z = z - presence * (count > 0) - frequency * count
        for t, v in bias[b0:b0 + nb]:
            z[t] += v
            size[t] += abs(v)
        if mask >= 0:
            z[np.unpackbits(masks[mask].view(np.uint8), bitorder="little")[:V] == 0] = -np.inf
        dst[r] = z
        tol[r] = (6 + nb) * 2.0 ** -24 * size
    return dst, tol
