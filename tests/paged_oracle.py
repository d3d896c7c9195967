"""Plain numpy of the paged cache's operators, in whole numbers and float64, and the bounds that
rounding allows a kernel."""
import numpy as np
import torch

# a rounding to the type is off by at most half a step
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def tables_step(before, fresh, tables, free_list, free_count, P, tokens):
    """What pa_page_tables does: (lengths, q_start, slots, positions, free_count, status, tables)."""
    R, cols = tables.shape
    tables = tables.copy()
    n_pages = len(free_list)
    slots, pos = np.full(tokens, -1), np.full(tokens, -1)
    status, need = 0, 0
    for b, f in zip(before, fresh):
        if b < 0 or f < 0 or b + f > cols * P:
            status |= 2
        else:
            need += -(-(b + f) // P) - -(-b // P)
    if sum(f for b, f in zip(before, fresh) if b >= 0 and f >= 0 and b + f <= cols * P) > tokens:
        status |= 4
    if not 0 <= free_count <= n_pages or need > free_count:
        status |= 1
    if status:
        return before.copy(), np.zeros(R + 1, dtype=int), slots, pos, free_count, status, tables
    top, t = free_count, 0
    q_start = np.concatenate([[0], np.cumsum(fresh)])
    for r, (b, f) in enumerate(zip(before, fresh)):
        for c in range(-(-b // P), -(-(b + f) // P)):
            top -= 1
            tables[r, c] = free_list[top]
        for x in range(b, b + f):
            page = tables[r, x // P]
            slots[t] = page * P + x % P if 0 <= page < n_pages else -1
            pos[t] = x
            t += 1
    return before + fresh, q_start, slots, pos, top, 0, tables


def release(first, last, tables, free_list, free_count):
    """What pa_page_release does: (tables, free_list, free_count, status)."""
    R, cols = tables.shape
    tables, out, n = tables.copy(), free_list.copy(), len(free_list)
    back = []
    for r in range(R):
        for c in range(max(0, first[r]), min(cols, last[r])):
            if 0 <= tables[r, c] < n:
                back.append(tables[r, c])
                tables[r, c] = -1
    if not 0 <= free_count <= n or free_count + len(back) > n:
        return None, free_list.copy(), free_count, 1
    out[free_count:free_count + len(back)] = back
    return tables, out, free_count + len(back), 0


def attention(q, k, v, tables, lengths, q_start, live, scale, dtype):
    """float64 (o, lse, bound of o, bound of lse) of the packed rows; rows of no request are NaN.

    q [T, Hq, D], k / v [pages, Hkv, P, D] float64; live(q positions [n, 1], k positions [1, L]) ->
    bool.  A kernel's o may be off by: its rounding to the type and (16-bit types) that of each
    probability, half a step of each; the error of a score, at most (D + 2) 2^-24 scale sum |q k|
    in float32, twice relative in the probabilities (their own and the sum's); 2^-18 relative for
    the exponentials (their argument is rounded at up to 2^5 in size) and the sums; and float16
    loses probabilities below its smallest step, 2^-25 each of at least one in all."""
    T, Hq, D = q.shape
    pages, Hkv, P, _ = k.shape
    G, u = Hq // Hkv, HALF_STEP[dtype]
    o, lse = np.full(q.shape, np.nan), np.full((T, Hq), np.nan)
    eo, el = np.zeros(q.shape), np.zeros((T, Hq))
    for r, L in enumerate(lengths):
        s, e = q_start[r], q_start[r + 1]
        n, pos = e - s, np.arange(L)
        if n == 0:
            continue
        page = tables[r, pos // P] if L else np.zeros(0, dtype=int)
        there = (page >= 0) & (page < pages)
        ok = live(np.arange(L - n, L)[:, None], pos[None, :]) & there[None, :]
        page = np.where(there, page, 0)
        for h in range(Hq):
            kh, vh = k[page, h // G, pos % P], v[page, h // G, pos % P]
            # (what is dead contributes nothing, whatever it holds)
            seen = ok.any(axis=0)
            kh, vh = np.where(seen[:, None], kh, 0), np.where(seen[:, None], vh, 0)
            x = np.where(ok, (q[s:e, h] @ kh.T) * scale, -np.inf)
            ab = np.where(ok, (np.abs(q[s:e, h]) @ np.abs(kh).T) * scale, 0).max(axis=1, initial=0)
            m = x.max(axis=1, initial=-np.inf)
            p = np.exp(x - np.where(np.isfinite(m), m, 0)[:, None])
            l = p.sum(axis=1)
            some = l > 0
            w = p / np.where(some, l, 1)[:, None]
            o[s:e, h] = w @ vh
            with np.errstate(divide="ignore"):
                lse[s:e, h] = np.where(some, m + np.log(l), -np.inf)
            mass = w @ np.abs(vh)
            ds = (D + 2) * 2.0 ** -24 * ab[:, None]
            pu = 0 if dtype == torch.float32 else u
            few = ok.sum(axis=1)[:, None] * 2.0 ** -25 * np.abs(vh).max(initial=0) if dtype == torch.float16 else 0
            eo[s:e, h] = 1.01 * (u * np.abs(o[s:e, h]) + pu * mass) + (2 * ds + 2.0 ** -18) * mass + few
            el[s:e, h] = ds[:, 0] + 2.0 ** -18 + 2.0 ** -22 * np.abs(np.where(some, lse[s:e, h], 0))
    return o, lse, eo, el
