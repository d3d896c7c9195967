"""Plain numpy of the operators on a paged cache that requests share and that forgets, in whole
numbers and float64, and the bounds that rounding allows a kernel."""
import numpy as np


def sharing(lengths, q_start, holders, shared, P, T):
    """What pa_share_rows does: (start, rows, positions, prefix, low, high, first)."""
    R = len(lengths)
    n = np.diff(q_start)
    some = np.minimum(np.maximum(shared, 0), lengths) // P * P
    member = (holders >= 0) & (holders < R) & (n > 0) & (some > 0)
    start, rows, pos = [0], [], []
    prefix, low, high, first = (np.zeros(R, dtype=np.int64) for _ in range(4))
    for g in range(R):
        who = np.flatnonzero(member & (holders == g))
        if len(who) > 1:
            prefix[g] = some[who].min()
            first[who] = prefix[g]
            low[g], high[g] = (lengths - n)[who].min(), lengths[who].max() - 1
            for r in who:
                rows += range(q_start[r], q_start[r + 1])
                pos += range(lengths[r] - n[r], lengths[r])
        start.append(len(rows))
    fill = [-1] * (T - len(rows))
    return tuple(np.array(x, dtype=np.int64) for x in (start, rows + fill, pos + fill, prefix, low, high, first))


def weights(q, k, tables, lengths, q_start, lse, scores, live, scale, first):
    """float64 (scores, bound) of pa_paged_weights.

    A weight exp(x - lse) may be off by what moves its argument: a score's float32 products and sums, at
    most (D + 2) 2^-24 scale sum |q k|; the roundings of x c, of lse log2(e) and of c, each half a step
    of its value, within 2^-22 (|x| + |lse|); and 2^-20 relative for the exponential.  The sum of N of
    them rounds by 2^-24 of itself N times at most, and once more with the score."""
    T, Hq, D = q.shape
    pages, Hkv, P, _ = k.shape
    G = Hq // Hkv
    out, bound = scores.copy(), np.zeros(scores.shape)
    for r, L in enumerate(lengths):
        s, e = q_start[r], q_start[r + 1]
        n, pos = e - s, np.arange(L)
        if n == 0:
            continue
        page = tables[r, pos // P]
        there = (page >= 0) & (page < pages)
        ok = live(np.arange(L - n, L)[:, None], pos[None, :]) & there[None, :]
        at = there & (pos >= first[r])
        for h in range(Hkv):
            kh = np.where(ok.any(axis=0)[:, None], k[np.where(there, page, 0), h, pos % P], 0)
            w, ew = np.zeros(L), np.zeros(L)
            for j in range(h * G, (h + 1) * G):
                z = lse[s:e, j][:, None]
                has = ok & ~np.isneginf(z)
                x = (q[s:e, j] @ kh.T) * scale
                ab = (np.abs(q[s:e, j]) @ np.abs(kh).T) * scale
                with np.errstate(over="ignore", invalid="ignore"):
                    p = np.where(has, np.exp(x - z), 0)
                    d = np.where(has, (D + 2) * 2.0 ** -24 * ab + 2.0 ** -22 * (np.abs(x) + np.abs(z)) + 2.0 ** -20, 0)
                    w += p.sum(axis=0)
                    ew += np.where(has, p * np.expm1(d), 0).sum(axis=0)
            old = np.where(pos < L - n, out[np.where(there, page, 0), h, pos % P], 0)
            total = old + w
            out[page[at], h, pos[at] % P] = total[at]
            bound[page[at], h, pos[at] % P] = (1.01 * ew + (n * G + 8) * 2.0 ** -24 * w + 2.0 ** -24 * np.abs(total) + 1e-36)[at]
    return out, bound


def choose(scores, tables, lengths, keep, recent, limit, first):
    """What pa_choose_keys does, of one layer: (kept, lengths)."""
    pages, H, P = scores.shape
    R = len(lengths)
    kept, after = np.full((R, H, keep), -1, dtype=np.int64), np.array(lengths)
    for r, L in enumerate(lengths):
        f = min(max(first[r], 0), L)
        if L - f <= limit:
            continue
        after[r] = f + keep
        pos = np.arange(f, L - recent)
        page = tables[r, pos // P]
        there = (page >= 0) & (page < pages)
        for h in range(H):
            x = scores[np.where(there, page, 0), h, pos % P]
            # (no page below all numbers, NaN above; sorts are stable: the first of equal ones)
            rank = np.where(~there, 0, np.where(np.isnan(x), 3, np.where(x == np.inf, 2, 1)))
            x = np.where(np.isnan(x) | ~there, 0, x)
            order = np.lexsort((pos, -x, -rank))
            best = np.sort(pos[order[:keep - recent]])
            kept[r, h] = np.concatenate([best, np.arange(L - recent, L)])
    return kept, after


def evict(kept, x, tables, lengths, first):
    """Rows x [pages, H, P, ...] of one layer moved as pa_evict_rows does."""
    pages, H, P = x.shape[:3]
    out, reach = x.copy(), tables.shape[1] * P
    for r, L in enumerate(lengths):
        f = min(max(first[r], 0), L)
        for h in range(H):
            for j, of in enumerate(kept[r, h]):
                if of <= f + j or of >= reach:
                    continue
                a, b = tables[r, of // P], tables[r, (f + j) // P]
                if 0 <= a < pages and 0 <= b < pages:
                    out[b, h, (f + j) % P] = x[a, h, of % P]
    return out
