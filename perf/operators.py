"""Serving a batch of requests from a paged cache: its tables, the write into it, and the
attention of each request's new tokens to all its cached ones.

``listed`` holds the fixed cases, ``draw`` gives further ones of the same ranges.  ``run``
computes a case in plain torch, or, with ``own`` set, by the package's entry points;
``exact`` is the same result in float64.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one generated token for each of 256 requests: the tables grow by a page here and there
        dict(name="tables-token", op="tables", R=256, lo=1, hi=8192, fresh_lo=1, fresh_hi=1, pad=0, page=64, max_length=8448,
             pattern=1),
        # prompts that arrive together (some requests wait: no new token), in pages of 16, with
        # the token rows padded to a fixed size
        dict(name="tables-prompts", op="tables", R=96, lo=0, hi=4000, fresh_lo=0, fresh_hi=1400, pad=500, page=16,
             max_length=8192, pattern=2),
        # the new keys and values of 256 requests generating a token each, one layer
        dict(name="append-token", op="append", dtype="bf16", R=256, lo=1, hi=4096, fresh_lo=1, fresh_hi=1, pad=0, page=64,
             max_length=8192, Hkv=8, D=128, pattern=3),
        # the keys and values of whole prompts
        dict(name="append-prompts", op="append", dtype="f16", R=24, lo=0, hi=900, fresh_lo=100, fresh_hi=2000, pad=77,
             page=16, max_length=4096, Hkv=8, D=64, pattern=4),
        # the smallest attention call: one float32 request in a small model, where latency counts
        dict(name="token-f32-small", op="attn", dtype="f32", R=1, lo=1001, hi=1001, fresh_lo=1, fresh_hi=1, pad=0, page=16,
             max_length=1024, Hq=4, Hkv=4, D=64, mask="causal", p0=0, p1=0, trim=False, pattern=5),
        # a serving batch generating a token each over contexts of all lengths
        dict(name="token-batch", op="attn", dtype="bf16", R=64, lo=300, hi=8192, fresh_lo=1, fresh_hi=1, pad=0, page=64,
             max_length=8192, Hq=32, Hkv=8, D=128, mask="causal", p0=0, p1=0, trim=False, pattern=6),
        # two long documents being continued: few rows, one long axis
        dict(name="token-long", op="attn", dtype="f16", R=2, lo=65536, hi=131071, fresh_lo=1, fresh_hi=1, pad=0, page=64,
             max_length=131072, Hq=32, Hkv=8, D=128, mask="causal", p0=0, p1=0, trim=False, pattern=7),
        # a few drafted tokens per request under the band and lattice mask, rows padded
        dict(name="draft-lattice", op="attn", dtype="bf16", R=40, lo=100, hi=6000, fresh_lo=1, fresh_hi=5, pad=9, page=32,
             max_length=8192, Hq=16, Hkv=2, D=128, mask="local_strided", p0=256, p1=16, trim=False, pattern=8),
        # a long prompt's next chunk over what is cached of it: the largest work
        dict(name="chunk-long", op="attn", dtype="bf16", R=1, lo=30001, hi=30001, fresh_lo=2000, fresh_hi=2000, pad=0,
             page=64, max_length=32768, Hq=32, Hkv=8, D=128, mask="causal", p0=0, p1=0, trim=False, pattern=9),
        # chunks of prompts together with requests that generate, in one call
        dict(name="chunk-mixed", op="attn", dtype="f16", R=36, lo=17, hi=4000, fresh_lo=20, fresh_hi=1000, pad=30, page=16,
             max_length=4096, Hq=16, Hkv=8, D=64, mask="causal", p0=0, p1=0, trim=False, ones=0.7, pattern=10),
        # prompts streamed through a window of 1024 and 64 sinks, pages behind the window given back
        dict(name="sinks-chunk", op="attn", dtype="bf16", R=4, lo=5000, hi=32768, fresh_lo=1000, fresh_hi=4096, pad=0,
             page=64, max_length=32768, Hq=32, Hkv=8, D=128, mask="sinks", p0=1024, p1=64, trim=True, pattern=11),
        # a token each of endless streams with the same mask
        dict(name="sinks-token", op="attn", dtype="bf16", R=128, lo=700, hi=32768, fresh_lo=1, fresh_hi=1, pad=0, page=64,
             max_length=32768, Hq=32, Hkv=8, D=128, mask="sinks", p0=1024, p1=64, trim=True, pattern=12),
    ]


# ---- draws ---------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = _drawn(rng)
        w = work(c)
        if c["op"] != "attn":
            most = 1.5e8
        else:
            # below the listed largest of their kind: a long chunk, a batch of tokens; in float32,
            # whose rates are lower, a sixteenth
            cut = 16 if c["dtype"] == "f32" else 1
            if w["flops"] > 8e11 / cut:
                continue
            most = 1e9
        if w["bytes"] <= most:
            return c


def _drawn(rng):
    op = rng.choice(["tables", "append", "token", "token", "chunk", "chunk", "sinks", "sinks"])
    page, pattern = rng.choice([16, 32, 64, 128]), rng.randrange(1 << 30)
    if op in ("tables", "append"):
        one = rng.random() < 0.5
        R = _log(rng, 1, 600) if one else _log(rng, 1, 100)
        fresh = 1 if one else _log(rng, 2, 2000)
        lo, hi = rng.choice([0, 1]), _log(rng, 16, 8192)
        c = dict(op=op, R=R, lo=lo, hi=hi, fresh_lo=1 if one else rng.choice([0, 1, fresh // 2]), fresh_hi=fresh,
                 pad=rng.choice([0, 0, _log(rng, 1, 300)]), page=page, max_length=hi + fresh + rng.randrange(300),
                 pattern=pattern)
        if op == "append":
            c.update(dtype=rng.choice(["bf16", "f16", "f32"]), Hkv=rng.choice([1, 2, 4, 5, 8]), D=rng.choice([64, 128]))
        return c
    dtype = rng.choice(["bf16", "f16", "bf16", "f16", "f32"])
    Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 8])
    token = op == "token" or (op == "sinks" and rng.random() < 0.5)
    R = _log(rng, 1, 128) if token else _log(rng, 1, 24)
    fresh = rng.choice([1, 1, 1, 2, 7]) if token else _log(rng, 20, 3000)
    hi = _log(rng, 100, 32768) + fresh
    lo = max(fresh, _log(rng, 1, hi))
    if op == "sinks":
        mask, p0, p1 = "sinks", _log(rng, 16, 2048), rng.choice([1, 4, 16, 64])
    else:
        mask = rng.choice(["causal", "causal", "local_strided"])
        p0, p1 = (0, 0) if mask == "causal" else (_log(rng, 16, 512), rng.choice([8, 16, 32]))
    return dict(op="attn", dtype=dtype, R=R, lo=lo, hi=hi, fresh_lo=rng.choice([1, fresh]), fresh_hi=fresh,
                pad=rng.choice([0, 0, _log(rng, 1, 100)]), page=page, max_length=hi + rng.randrange(300), Hq=Hq, Hkv=Hkv, D=D,
                mask=mask, p0=p0, p1=p1, trim=op == "sinks" and rng.random() < 0.7,
                ones=0.0 if token else rng.choice([0.0, 0.6]), pattern=pattern)


# ---- sizes ---------------------------------------------------------------------------
def _sizes(case):
    """(tokens cached before, new tokens) of each request, numpy int64: log-uniform contexts,
    lo .. hi tokens with the new ones in an attention case and before them in the others."""
    rng = random.Random(case["pattern"])
    fresh = [rng.randint(case["fresh_lo"], case["fresh_hi"]) for _ in range(case["R"])]
    # (the share of the requests that generate a token each beside the others' chunks)
    fresh = [1 if rng.random() < case.get("ones", 0.0) else f for f in fresh]
    length = [_log(rng, max(1, case["lo"]), max(1, case["hi"])) if case["hi"] > case["lo"] else case["hi"] for _ in fresh]
    if case["op"] == "attn":
        before = [max(0, n - f) for n, f in zip(length, fresh)]
    else:
        before = [n if rng.random() > 0.1 else case["lo"] for n in length]
    return np.array(before, dtype=np.int64), np.array(fresh, dtype=np.int64)


def _tokens(case):
    return int(_sizes(case)[1].sum()) + case["pad"]


def _live(case, q, k):
    """Whether a key at position k is live for a query at position q (torch or numpy integers)."""
    d = q - k
    if case["mask"] == "sinks":
        return (d >= 0) & ((d < case["p0"]) | (k < case["p1"]))
    if case["mask"] == "local_strided":
        return (d >= 0) & ((d < case["p0"]) | (d % case["p1"] == 0))
    return d >= 0


def _counts(case):
    """(live pairs, keys live for some new token) over all requests, of one head."""
    pairs = keys = 0
    for b, f in zip(*_sizes(case)):
        q = np.arange(b, b + f)
        n = int(b + f)
        if case["mask"] == "sinks":
            first = np.maximum(0, q - case["p0"] + 1)
            pairs += int((q + 1 - first + np.minimum(first, case["p1"])).sum())
            keys += n - int(first[0]) + min(int(first[0]), case["p1"]) if f else 0
        elif case["mask"] == "local_strided":
            w, s = case["p0"], case["p1"]
            pairs += int((np.minimum(q + 1, w) + np.maximum(0, q // s - (w - 1) // s)).sum())
            seen = np.zeros(n, dtype=bool)
            for i in range(min(int(f), s)):  # the lattice repeats after s rows
                seen |= _live(case, q[-1 - i], np.arange(n))
            seen[max(0, int(b) - w + 1):] |= f > 0
            keys += int(seen.sum())
        else:
            pairs += int((q + 1).sum())
            keys += n if f else 0
    return pairs, keys


def work(case):
    before, fresh = _sizes(case)
    T, page = _tokens(case), case["page"]
    if case["op"] == "tables":
        new = (-(-(before + fresh) // page) - -(-before // page)).sum()
        half = ((fresh > 0) & (before % page > 0)).sum()  # requests whose last page goes on
        # the free pages taken and written into the tables, lengths and new tokens in, lengths and
        # starts out, a slot and a position per token
        return dict(bytes=float(8 * new + 4 * half + 16 * case["R"] + 8 * T), flops=0.0)
    if case["op"] == "append":
        return dict(bytes=4.0 * int(fresh.sum()) * case["Hkv"] * case["D"] * ESIZE[case["dtype"]] + 4.0 * T, flops=0.0)
    pairs, keys = _counts(case)
    rows = int(fresh.sum()) * case["Hq"]
    return dict(flops=4.0 * case["D"] * case["Hq"] * pairs,
                bytes=2.0 * case["D"] * ESIZE[case["dtype"]] * (keys * case["Hkv"] + rows) + 4.0 * rows
                + 4.0 * keys / page + 8.0 * case["R"])


# ---- inputs --------------------------------------------------------------------------
def _columns(case):
    return -(-case["max_length"] // case["page"])


def _held(case):
    """bool [R, columns]: the pages that hold a cached token before the call (attention: with the
    new tokens, without what the window has left behind where the pages are given back)."""
    before, fresh = _sizes(case)
    n = before + fresh if case["op"] == "attn" else before
    col = np.arange(_columns(case))[None, :]
    held = col < -(-n // case["page"])[:, None]
    if case["op"] == "attn" and case["trim"]:
        first = np.maximum(0, before - case["p0"] + 1) // case["page"]
        held &= (col >= first[:, None]) | (col < -(-case["p1"] // case["page"]))
    return held


def _dev(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32).cuda()


def _pages(case, seed):
    """(tables int32 [R, columns] with -1 for no page, the free pages, pages in all): page ids in an
    order that a cache in use has, that is none."""
    held = _held(case)
    before, fresh = _sizes(case)
    n, spare = int(held.sum()), 7
    if case["op"] != "attn":
        spare += int((-(-(before + fresh) // case["page"])).sum())
    ids = np.random.default_rng(seed).permutation(n + spare)
    tables = np.full(held.shape, -1, dtype=np.int64)
    tables[held] = ids[:n]
    return tables, ids[n:], n + spare


def _randn(seed, dtype, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if dtype == torch.float32 else torch.float16).to(dtype)


def _positions(case, pad_value):
    """Per row of the packed tokens: its request and its position, numpy (pad rows: pad_value)."""
    before, fresh = _sizes(case)
    req = np.repeat(np.arange(case["R"]), fresh)
    pos = np.arange(len(req)) - np.repeat(np.cumsum(fresh) - fresh, fresh) + np.repeat(before, fresh)
    pad = np.full(case["pad"], pad_value)
    return np.concatenate([req, pad]), np.concatenate([pos, pad])


def _data(case, seed):
    """The tensors of a case, on the GPU."""
    before, fresh = _sizes(case)
    tables, free, pages = _pages(case, seed)
    T = _tokens(case)
    s = dict(case=case, T=T, pages=pages, before=_dev(before), fresh=_dev(fresh), tables=_dev(tables),
             q_start=_dev(np.concatenate([[0], np.cumsum(fresh)])), lengths=_dev(before + fresh))
    if case["op"] == "tables":
        # a pool in use: some of the list's end is free
        s.update(free_list=_dev(np.concatenate([free, np.full(pages - len(free), -1)])), free_count=_dev([len(free)]))
        return s
    dt, P, Hkv, D = DTYPES[case["dtype"]], case["page"], case["Hkv"], case["D"]
    if case["op"] == "append":
        # the tables after the call: the new tokens' pages are free ones
        col = np.arange(tables.shape[1])[None, :]
        new = (tables < 0) & (col < -(-(before + fresh) // P)[:, None])
        tables[new] = free[:int(new.sum())]
        req, pos = _positions(case, -1)
        slots = np.where(pos < 0, -1, tables[req, np.maximum(pos, 0) // P] * P + np.maximum(pos, 0) % P)
        s.update(k_new=_randn(seed + 1000003, dt, T, Hkv, D), v_new=_randn(seed + 2000003, dt, T, Hkv, D), slots=_dev(slots))
    else:
        s.update(q=_randn(seed + 1000003, dt, T, case["Hq"], D), max_fresh=int(fresh.max()),
                 o=torch.zeros(T, case["Hq"], D, dtype=dt, device="cuda"),
                 lse=torch.zeros(T, case["Hq"], dtype=torch.float32, device="cuda"))
    s.update(k=_randn(seed + 3000003, dt, pages, Hkv, P, D), v=_randn(seed + 4000003, dt, pages, Hkv, P, D))
    if case.get("mask") == "sinks":
        # sink tokens have larger keys, as trained models do
        first = tables[:, :case["p1"] // P]
        s["k"][torch.as_tensor(first[first >= 0], device="cuda")] *= 4
    return s


def prepare(case, seed):
    s = _data(case, seed)
    if case["op"] == "attn":
        # requests that the plain form pads to one size, so that its scores stay within 16 GB
        before, fresh = _sizes(case)
        s["groups"], lo = [], 0
        for hi in range(1, case["R"] + 1):
            span = slice(lo, hi + 1)
            if hi == case["R"] or (hi + 1 - lo) * case["Hq"] * fresh[span].max() * (before + fresh)[span].max() > 1 << 32:
                s["groups"].append((lo, hi, int(fresh[lo:hi].max()), int((before + fresh)[lo:hi].max())))
                lo = hi
    if own:
        s["call"] = _own_call(s)
    return s


# ---- the framework's operators ----------------------------------------------------------
def _own_call(s):
    """The launch that a serving program keeps for its buffers."""
    from polyhedral_amd import paged
    from polyhedral_amd.polyattn import masks
    case = s["case"]
    if case["op"] == "tables":
        return paged.prepare_tables(s["before"], s["fresh"], s["tables"], s["free_list"], s["free_count"], case["page"], s["T"])
    if case["op"] == "append":
        return paged.prepare_append(s["k_new"], s["v_new"], s["slots"], s["k"], s["v"])
    mask = {"causal": masks.Causal, "sinks": lambda: masks.SinksWindow(case["p1"], case["p0"]),
            "local_strided": lambda: masks.LocalStrided(case["p0"], case["p1"])}[case["mask"]]()
    return paged.prepare_attention(s["q"], s["k"], s["v"], s["tables"], s["lengths"], s["q_start"], mask,
                                   max_fresh=s["max_fresh"], out=s["o"], lse=s["lse"])


def run(state):
    op = state["case"]["op"]
    if own:
        done = state["call"]()
        if op == "tables":
            return (state["tables"], done.lengths, done.q_start, done.slots, done.positions, done.free_count, done.status)
        return (state["k"], state["v"]) if op == "append" else (state["o"], state["lse"])
    return {"tables": _plain_tables, "append": _plain_append, "attn": _plain_attention}[op](state)


# ---- the same in plain torch -------------------------------------------------------------
def _plain_tables(s):
    P, T, tables = s["case"]["page"], s["T"], s["tables"]
    before, fresh = s["before"].long(), s["fresh"].long()
    lengths = before + fresh
    first = (before + P - 1) // P
    need = (lengths + P - 1) // P - first
    base = need.cumsum(0) - need
    req = torch.repeat_interleave(need)
    j = torch.arange(req.numel(), device=req.device)
    tables[req, first[req] + j - base[req]] = s["free_list"][s["free_count"].long() - 1 - j]
    q_start = torch.cat([fresh.new_zeros(1), fresh.cumsum(0)])
    t = torch.arange(T, device=req.device)
    r = torch.searchsorted(q_start[1:].contiguous(), t, right=True)
    inside = r < fresh.numel()
    r = r.clamp(max=fresh.numel() - 1)
    pos = before[r] + t - q_start[r]
    slot = tables[r, (pos // P).clamp(max=tables.shape[1] - 1)].long() * P + pos % P
    status = ((need.sum() > s["free_count"][0]).int() + 2 * (lengths > tables.shape[1] * P).any().int()
              + 4 * (q_start[-1] > T).int())
    i32 = torch.int32
    return (tables, lengths.to(i32), q_start.to(i32), torch.where(inside, slot, -1).to(i32),
            torch.where(inside, pos, -1).to(i32), (s["free_count"] - need.sum()).to(i32), status.reshape(1))


def _plain_append(s):
    P, k, v = s["case"]["page"], s["k"], s["v"]
    rows = torch.nonzero(s["slots"] >= 0)[:, 0]
    slot = s["slots"][rows].long()
    k[slot // P, :, slot % P] = s["k_new"][rows]
    v[slot // P, :, slot % P] = s["v_new"][rows]
    return k, v


def _plain_attention(s):
    case, q, o, lse = s["case"], s["q"], s["o"], s["lse"]
    P, Hkv, D = case["page"], case["Hkv"], case["D"]
    G = case["Hq"] // Hkv
    for lo, hi, rows, keys in s["groups"]:
        n = (s["q_start"][lo + 1:hi + 1] - s["q_start"][lo:hi]).long()
        L = s["lengths"][lo:hi].long()
        i = torch.arange(rows, device=q.device)
        t = torch.arange(keys, device=q.device)
        row = s["q_start"][lo:hi].long()[:, None] + torch.minimum(i, (n - 1).clamp(min=0)[:, None])
        page = s["tables"][lo:hi, t // P].clamp(min=0).long()
        qs = q[row.clamp(max=q.shape[0] - 1)].float().view(hi - lo, rows, Hkv, G, D).transpose(1, 2).reshape(hi - lo, Hkv, rows * G, D)
        ks = s["k"][page, :, t % P].float().permute(0, 2, 3, 1).contiguous()
        vs = s["v"][page, :, t % P].float().transpose(1, 2).contiguous()
        pos = (L - n)[:, None] + i
        live = _live(case, pos[:, :, None], t) & (t < L[:, None, None]) & (i < n[:, None])[:, :, None]
        x = (qs @ ks).mul_(D ** -0.5).view(hi - lo, Hkv, rows, G, keys)
        x.masked_fill_(~live[:, None, :, None, :], -math.inf)
        m = x.amax(-1, keepdim=True)
        m = torch.where(m == -math.inf, 0.0, m)
        p = x.sub_(m).exp_()
        total = p.sum(-1, keepdim=True)
        out = (p.view(hi - lo, Hkv, rows * G, keys) @ vs).view(hi - lo, Hkv, rows, G, D) / torch.where(total == 0, 1.0, total)
        valid = i < n[:, None]
        at = row[valid]
        o[at] = out.permute(0, 2, 1, 3, 4)[valid].reshape(-1, Hkv * G, D).to(o.dtype)
        lse[at] = (m + total.log()).permute(0, 2, 1, 3, 4)[valid].reshape(-1, Hkv * G)
    return o, lse


# ---- float64 -----------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "append":
        # every row where it belongs, the others as they were
        s = _data(case, seed)
        new = {int(x): t for t, x in enumerate(s["slots"].tolist()) if x >= 0}
        at = torch.tensor(list(new.keys()), device="cuda", dtype=torch.long)
        of = torch.tensor(list(new.values()), device="cuda", dtype=torch.long)
        out = []
        for pool, rows in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
            flat = pool.double().transpose(1, 2).reshape(-1, case["Hkv"], case["D"])
            flat[at] = rows[of].double()
            out.append(flat.view(s["pages"], case["page"], case["Hkv"], case["D"]).transpose(1, 2).contiguous())
        return tuple(out)
    if case["op"] != "attn":
        return None
    s = _data(case, seed)
    before, fresh = _sizes(case)
    tables = s["tables"].long()
    G, P, D = case["Hq"] // case["Hkv"], case["page"], case["D"]
    o = torch.zeros(s["T"], case["Hq"], D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["T"], case["Hq"], dtype=torch.float64, device="cuda")
    t0 = 0
    for r in range(case["R"]):
        b, f = int(before[r]), int(fresh[r])
        k_pos = torch.arange(b + f, device="cuda")
        q_pos = torch.arange(b, b + f, device="cuda")
        # only positions live for some row: what the window left behind has no page
        kept = k_pos[tables[r, k_pos // P] >= 0]
        page, off = tables[r, kept // P], kept % P
        for h in range(case["Hkv"]):
            kh, vh = s["k"][page, h, off].double(), s["v"][page, h, off].double()
            step = max(1, (1 << 27) // max(1, G * len(kept)))
            for i in range(0, f, step):
                rows = slice(t0 + i, t0 + min(f, i + step))
                x = torch.einsum("ngd,kd->ngk", s["q"][rows, h * G:(h + 1) * G].double(), kh) / math.sqrt(D)
                x.masked_fill_(~_live(case, q_pos[i:i + step, None], kept)[:, None, :], -math.inf)
                z = torch.logsumexp(x, -1)
                lse[rows, h * G:(h + 1) * G] = z
                o[rows, h * G:(h + 1) * G] = torch.exp(x - z[..., None]) @ vh
        t0 += f
    return o, lse
