"""A paged cache whose requests share a prefix, and that forgets: attention that reads a shared
prefix once for all its requests, the attention weight that every cached key has received, the
choice of the keys that stay, and their move to the front of a request's pages.

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
        # four samples of one short prompt in a small float32 model: the smallest call
        dict(name="prefix-token-f32-small", op="attn", dtype="f32", R=4, groups=1, alone=0, prefix_lo=512, prefix_hi=512,
             own_lo=20, own_hi=100, fresh_lo=1, fresh_hi=1, pad=0, page=16, Hq=4, Hkv=4, D=64, mask="causal", p0=0, p1=0,
             pattern=1),
        # users behind one system prompt, generating a token each
        dict(name="prefix-token-batch", op="attn", dtype="bf16", R=64, groups=1, alone=0, prefix_lo=8192, prefix_hi=8192,
             own_lo=16, own_hi=2000, fresh_lo=1, fresh_hi=1, pad=0, page=64, Hq=32, Hkv=8, D=128, mask="causal", p0=0, p1=0,
             pattern=2),
        # drafted tokens of requests behind five prompts, and some behind none, rows padded
        dict(name="prefix-draft-groups", op="attn", dtype="f16", R=34, groups=5, alone=6, prefix_lo=500, prefix_hi=6000,
             own_lo=10, own_hi=800, fresh_lo=1, fresh_hi=5, pad=9, page=32, Hq=16, Hkv=2, D=64, mask="causal", p0=0, p1=0,
             pattern=3),
        # many samples over one long document
        dict(name="prefix-token-long", op="attn", dtype="bf16", R=32, groups=1, alone=0, prefix_lo=65536, prefix_hi=65536,
             own_lo=1, own_hi=4000, fresh_lo=1, fresh_hi=1, pad=0, page=64, Hq=32, Hkv=8, D=128, mask="causal", p0=0, p1=0,
             pattern=4),
        # questions of some hundred tokens over two documents: the largest work
        dict(name="prefix-chunk", op="attn", dtype="bf16", R=12, groups=2, alone=0, prefix_lo=12000, prefix_hi=16384,
             own_lo=100, own_hi=1000, fresh_lo=100, fresh_hi=600, pad=0, page=64, Hq=32, Hkv=8, D=128, mask="causal", p0=0,
             p1=0, pattern=5),
        # the weights of one token over one short context
        dict(name="weights-token-f32-small", op="weights", dtype="f32", R=1, lo=1001, hi=1001, fresh_lo=1, fresh_hi=1, pad=0,
             page=16, Hq=4, Hkv=4, D=64, mask="causal", p0=0, p1=0, first=0, pattern=6),
        # a serving batch generating a token each, the first tokens exempt
        dict(name="weights-token-batch", op="weights", dtype="bf16", R=64, lo=300, hi=8192, fresh_lo=1, fresh_hi=1, pad=0,
             page=64, Hq=32, Hkv=8, D=128, mask="causal", p0=0, p1=0, first=4, pattern=7),
        # chunks of prompts
        dict(name="weights-chunk", op="weights", dtype="f16", R=8, lo=1000, hi=8000, fresh_lo=256, fresh_hi=1500, pad=20,
             page=16, Hq=32, Hkv=8, D=128, mask="causal", p0=0, p1=0, first=0, pattern=8),
        # one layer of a few short contexts
        dict(name="choose-few", op="choose", layers=1, R=4, lo=900, hi=1100, keep=512, recent=64, limit=512, first=0, page=16,
             Hkv=4, pattern=9),
        # all requests past the limit, eight layers at once, sinks kept
        dict(name="choose-batch", op="choose", layers=8, R=32, lo=1500, hi=16384, keep=2048, recent=256, limit=2304, first=4,
             page=64, Hkv=8, pattern=10),
        # the rows that stay of one layer of a small float32 model
        dict(name="evict-few", op="evict", dtype="f32", layers=1, R=2, lo=900, hi=1100, keep=512, recent=64, limit=512,
             first=0, page=16, Hkv=4, D=64, pattern=11),
        # and of four layers of a serving batch: the most bytes
        dict(name="evict-batch", op="evict", dtype="bf16", layers=4, R=32, lo=1500, hi=9000, keep=2048, recent=256, limit=2304,
             first=4, page=64, Hkv=8, D=128, pattern=12),
    ]


# ---- draws ---------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = _drawn(rng)
        w = work(c)
        # below the listed largest of their kind; in float32, whose rates are lower, a sixteenth
        cut = 16 if c.get("dtype") == "f32" else 1
        most = {"attn": (5e8, 8e11 / cut), "weights": (5e8, 4e11 / cut), "choose": (6e7, 1), "evict": (1e9, 1)}[c["op"]]
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and _plain_bytes(c) < 1.6e10:
            return c


def _drawn(rng):
    op = rng.choice(["attn", "attn", "weights", "choose", "evict"])
    page, pattern = rng.choice([16, 32, 64, 128]), rng.randrange(1 << 30)
    if op in ("choose", "evict"):
        keep = _log(rng, 64, 4096)
        c = dict(op=op, layers=rng.choice([1, 2, 4, 8]), R=_log(rng, 1, 64), lo=_log(rng, max(1, keep // 2), 2 * keep),
                 hi=2 * keep + _log(rng, 1, 12000), keep=keep, recent=rng.randint(0, keep // 2),
                 limit=keep + rng.choice([0, 0, keep // 8]), first=rng.choice([0, 0, 1, 4, page]), page=page,
                 Hkv=rng.choice([1, 2, 4, 5, 8]), pattern=pattern)
        if op == "evict":
            c.update(dtype=rng.choice(["bf16", "f16", "f32"]), D=rng.choice([64, 128]))
        return c
    dtype = rng.choice(["bf16", "f16", "bf16", "f16", "f32"])
    Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 8])
    token = rng.random() < 0.6
    fresh = rng.choice([1, 1, 1, 2, 7]) if token else _log(rng, 20, 1000)
    mask = rng.choice(["causal", "causal", "causal", "sinks", "local_strided"])
    p0, p1 = {"causal": (0, 0), "sinks": (_log(rng, 16, 4096), rng.choice([1, 4, 16, 64])),
              "local_strided": (_log(rng, 16, 512), rng.choice([8, 16, 32]))}[mask]
    c = dict(op=op, dtype=dtype, fresh_lo=rng.choice([1, fresh]), fresh_hi=fresh, pad=rng.choice([0, 0, _log(rng, 1, 100)]),
             page=page, Hq=Hq, Hkv=Hkv, D=D, mask=mask, p0=p0, p1=p1, pattern=pattern)
    if op == "weights":
        hi = _log(rng, 100, 32768) + fresh
        c.update(R=_log(rng, 1, 128) if token else _log(rng, 1, 16), lo=max(fresh, _log(rng, 1, hi)), hi=hi,
                 first=rng.choice([0, 0, 1, 4, page]))
        return c
    groups = rng.choice([1, 1, 1, 2, 3, 6])
    prefix = _log(rng, 100, 65536)
    own_hi = _log(rng, 20, 4000) + fresh
    c.update(R=2 * groups + (_log(rng, 1, 100) if token else _log(rng, 1, 12)), groups=groups, alone=rng.choice([0, 0, 1, 5]),
             prefix_lo=max(page, prefix // rng.choice([1, 4])), prefix_hi=max(page, prefix),
             own_lo=max(fresh, _log(rng, 1, own_hi)), own_hi=own_hi)
    return c


# ---- sizes ---------------------------------------------------------------------------
def _sizes(case):
    """Per request, numpy int64: its length with the new tokens, the new tokens, the request whose
    prefix it shares (-1: none) and the tokens of that.  The prefixes are held by requests without
    new tokens, the last ``groups`` of an attention case."""
    rng = random.Random(case["pattern"])
    draw_len = lambda lo, hi: _log(rng, max(1, lo), max(1, hi)) if hi > lo else hi  # noqa: E731
    if case["op"] != "attn":
        fresh = [rng.randint(case.get("fresh_lo", 0), case.get("fresh_hi", 0)) for _ in range(case["R"])]
        n = [max(f, draw_len(case["lo"], case["hi"])) for f in fresh]
        return tuple(np.array(x, dtype=np.int64) for x in (n, fresh, [-1] * case["R"], [0] * case["R"]))
    page, groups, total = case["page"], case["groups"], case["R"] + case["alone"]
    prefix = [max(1, draw_len(case["prefix_lo"], case["prefix_hi"]) // page) * page for _ in range(groups)]
    of = [i % groups for i in range(case["R"])] + [-1] * case["alone"]
    rng.shuffle(of)
    fresh = [rng.randint(case["fresh_lo"], case["fresh_hi"]) for _ in of]
    mine = [max(f, draw_len(case["own_lo"], case["own_hi"])) for f in fresh]
    shared = [prefix[g] if g >= 0 else 0 for g in of]
    holder = [total + g if g >= 0 else -1 for g in of]
    return tuple(np.array(x, dtype=np.int64) for x in ([s + m for s, m in zip(shared, mine)] + prefix, fresh + [0] * groups,
                                                       holder + [-1] * groups, shared + [0] * groups))


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


def _seen(case, q, lo, hi):
    """bool over the keys lo .. hi - 1: live for one of the queries at positions q."""
    if case["mask"] == "causal":
        return np.arange(lo, hi) <= q.max(initial=-1)
    seen = np.zeros(hi - lo, dtype=bool)
    for x in q:
        seen |= _live(case, x, np.arange(lo, hi))
    return seen


def _pairs(case, q):
    """Live pairs of queries at positions q, each with all keys up to its own."""
    if case["mask"] == "sinks":
        first = np.maximum(0, q - case["p0"] + 1)
        return int((q + 1 - first + np.minimum(first, case["p1"])).sum())
    if case["mask"] == "local_strided":
        w, s = case["p0"], case["p1"]
        return int((np.minimum(q + 1, w) + np.maximum(0, q // s - (w - 1) // s)).sum())
    return int((q + 1).sum())


def _counts(case):
    """(live pairs, keys live for some new token) of one head; a prefix's keys count once."""
    length, fresh, holder, shared = _sizes(case)
    pairs = keys = 0
    for n, f, s in zip(length, fresh, shared):
        q = np.arange(n - f, n)
        pairs += _pairs(case, q)
        if f:
            # (a lattice repeats after its stride)
            some = q if case["mask"] == "sinks" else q[-max(1, case["p1"]):]
            seen = _seen(case, some, s, n)
            if case["mask"] != "causal":
                seen[max(0, q[0] - case["p0"] + 1 - s):] = True
            keys += int(seen.sum())
    for g in np.unique(holder[holder >= 0]):
        members = np.nonzero(holder == g)[0]
        keys += int(_seen(case, np.unique(np.concatenate([np.arange(length[r] - fresh[r], length[r]) for r in members])), 0,
                          int(shared[members[0]])).sum())
    return pairs, keys


def _chosen(case):
    """bool [R]: the requests that give up keys."""
    return _sizes(case)[0] - case["first"] > case["limit"]


def work(case):
    length = _sizes(case)[0]
    if case["op"] in ("choose", "evict"):
        rows = case["layers"] * case["Hkv"] * int(_chosen(case).sum()) * case["keep"]
        lists = 8.0 * case["R"] + 4.0 * (length / case["page"]).sum()
        if case["op"] == "choose":
            # the scores that compete, in; the places chosen, out
            held = np.where(_chosen(case), length - case["first"] - case["recent"], 0)
            return dict(bytes=4.0 * case["layers"] * case["Hkv"] * float(held.sum()) + 4.0 * rows + lists, flops=0.0)
        # (the share of the chosen rows that lie where they belong is small: all count as moved)
        return dict(bytes=rows * (2.0 * (2 * case["D"] * ESIZE[case["dtype"]] + 4) + 4.0) + lists, flops=0.0)
    pairs, keys = _counts(case)
    rows, D, e = int(_sizes(case)[1].sum()) * case["Hq"], case["D"], ESIZE[case["dtype"]]
    if case["op"] == "weights":
        # keys, queries and their log-sum-exps in; scores in and out
        return dict(flops=2.0 * D * case["Hq"] * pairs, bytes=keys * case["Hkv"] * (D * e + 8.0) + rows * (D * e + 4.0)
                    + 4.0 * keys / case["page"] + 12.0 * case["R"])
    return dict(flops=4.0 * D * case["Hq"] * pairs, bytes=2.0 * D * e * (keys * case["Hkv"] + rows) + 4.0 * rows
                + 4.0 * keys / case["page"] + 16.0 * case["R"])


def _plain_bytes(case):
    """Memory of the plain form's largest tensor."""
    length, fresh, holder, shared = _sizes(case)
    if case["op"] in ("choose", "evict"):
        return 8.0 * case["layers"] * case["R"] * case["Hkv"] * float(length.max())
    most = 4.0 * len(length) * float((length - shared)[fresh > 0].max()) * max(case["Hq"] * float(fresh.max()), case["Hkv"] * case["D"])
    if case["op"] == "attn":
        rows = max(int(fresh[holder == g].sum()) for g in np.unique(holder[holder >= 0]))
        most = max(most, 4.0 * case["groups"] * float(shared.max()) * max(case["Hq"] * rows, case["Hkv"] * case["D"]))
    return most


# ---- inputs --------------------------------------------------------------------------
def _dev(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32).cuda()


def _randn(seed, dtype, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if dtype == torch.float32 else torch.float16).to(dtype)


def _pages(case, seed):
    """(tables int32 [R, columns] with -1 for no page, pages in all): page ids in an order that a
    cache in use has, that is none; who shares a prefix has its holder's pages in front."""
    length, fresh, holder, shared = _sizes(case)
    P = case["page"]
    col = np.arange(-(-int(length.max()) // P) + 2)[None, :]
    mine = (col < -(-length // P)[:, None]) & (col >= shared[:, None] // P)
    n = int(mine.sum())
    ids = np.random.default_rng(seed).permutation(n + 7)
    tables = np.full(mine.shape, -1, dtype=np.int64)
    tables[mine] = ids[:n]
    tables = np.where(col < shared[:, None] // P, tables[holder], tables)
    return tables, n + 7


def _data(case, seed):
    """The tensors of a case, on the GPU."""
    length, fresh, holder, shared = _sizes(case)
    tables, pages = _pages(case, seed)
    P, Hkv = case["page"], case["Hkv"]
    s = dict(case=case, pages=pages, tables=_dev(tables), lengths=_dev(length))
    if case["op"] in ("choose", "evict"):
        # weights as softmaxes give them: a few keys have most, many have none that is left in 32 bits
        x = _randn(seed + 1000003, torch.float32, case["layers"], pages, Hkv, P)
        s.update(scores=torch.where(x < -0.8, 0.0, (2.0 * x).exp()), first=_dev(np.full(case["R"], case["first"])))
        if case["op"] == "evict":
            shape = (case["layers"], pages, Hkv, P, case["D"])
            s.update(k=_randn(seed + 3000003, DTYPES[case["dtype"]], *shape), v=_randn(seed + 4000003, DTYPES[case["dtype"]], *shape))
        return s
    dt, D, T = DTYPES[case["dtype"]], case["D"], _tokens(case)
    s.update(q_start=_dev(np.concatenate([[0], np.cumsum(fresh)])), max_fresh=int(fresh.max()), longest=int((length - shared)[fresh > 0].max()),
             q=_randn(seed + 1000003, dt, T, case["Hq"], D), k=_randn(seed + 3000003, dt, pages, Hkv, P, D))
    if case["mask"] == "sinks":
        # sink tokens have larger keys, as trained models do
        sinks = tables[:, :case["p1"] // P]
        s["k"][torch.as_tensor(sinks[sinks >= 0], device="cuda")] *= 4
    if case["op"] == "weights":
        s.update(first=_dev(np.full(case["R"], case["first"])),
                 scores=_randn(seed + 5000003, torch.float32, pages, Hkv, P).abs() * 0.01,  # of some steps before
                 lse=torch.zeros(T, case["Hq"], dtype=torch.float32, device="cuda"))
        return s
    s.update(v=_randn(seed + 4000003, dt, pages, Hkv, P, D), holders=_dev(holder), shared=_dev(shared), prefix=int(shared.max()),
             o=torch.zeros(T, case["Hq"], D, dtype=dt, device="cuda"), lse=torch.zeros(T, case["Hq"], dtype=torch.float32, device="cuda"))
    # for the plain form: the tokens of each prefix's requests side by side, filled up with token T
    req = np.repeat(np.arange(len(fresh)), fresh)
    groups = [np.nonzero(holder[req] == g)[0] for g in np.unique(holder[holder >= 0])]
    rows = np.full((len(groups), max(map(len, groups))), T)
    for i, x in enumerate(groups):
        rows[i, :len(x)] = x
    s.update(group_rows=_dev(rows).long(), group_holder=_dev(np.unique(holder[holder >= 0])).long())
    return s


def prepare(case, seed):
    s = _data(case, seed)
    if case["op"] == "weights":
        _rows_scores(s, s["lse"])  # the log-sum-exps of the attention that came before
    if case["op"] == "evict":
        s["kept"] = _plain_choose(s)[0]
    if own:
        s["call"] = _own_call(s)
    return s


# ---- the framework's operators ----------------------------------------------------------
def _own_call(s):
    """The launches that a serving program keeps for its buffers."""
    from polyhedral_amd import paged
    from polyhedral_amd.polyattn import masks
    case = s["case"]
    if case["op"] == "choose":
        return [paged.prepare_choose(s["scores"], s["tables"], s["lengths"], case["keep"], case["recent"], limit=case["limit"],
                                     first=s["first"])]
    if case["op"] == "evict":
        return [paged.prepare_evict(s["kept"], s["k"], s["v"], s["scores"], s["tables"], s["lengths"], first=s["first"])]
    mask = {"causal": masks.Causal, "sinks": lambda: masks.SinksWindow(case["p1"], case["p0"]),
            "local_strided": lambda: masks.LocalStrided(case["p0"], case["p1"])}[case["mask"]]()
    if case["op"] == "weights":
        return [paged.prepare_weights(s["q"], s["k"], s["tables"], s["lengths"], s["q_start"], s["lse"], s["scores"], mask,
                                      first=s["first"], max_fresh=s["max_fresh"])]
    # which tokens share a prefix changes with every step, as the lengths do: found in the call
    sharing = paged.prepare_sharing(s["lengths"], s["q_start"], s["holders"], s["shared"], case["page"], s["q"].shape[0])
    return [sharing, paged.prepare_shared_attention(s["q"], s["k"], s["v"], s["tables"], s["lengths"], s["q_start"], sharing.result,
                                                    mask, max_fresh=s["max_fresh"], out=s["o"], lse=s["lse"])]


def run(state):
    op = state["case"]["op"]
    if own:
        for call in state["call"]:
            done = call()
        return (state["o"], state["lse"]) if op == "attn" else done
    return {"attn": _plain_attention, "weights": _plain_weights, "choose": _plain_choose, "evict": _plain_evict}[op](state)


# ---- the same in plain torch -------------------------------------------------------------
def _rows_scores(s, lse=None):
    """Of all requests' new rows, filled up to one number, and their keys from ``first_key`` on:
    (scores scale q . k in float32 [R, Hkv, rows, G, keys], -inf where a key is not live; the rows'
    places [R, rows], T for none; the keys' positions [R, keys]).  lse: is given each row's."""
    case, q = s["case"], s["q"]
    Hkv, D, P, T = case["Hkv"], case["D"], case["page"], q.shape[0]
    G = case["Hq"] // Hkv
    n = (s["q_start"][1:] - s["q_start"][:-1]).long()
    L = s["lengths"].long()
    i = torch.arange(s["max_fresh"], device=q.device)
    from_key = s["shared"].long()[:, None] if "shared" in s else 0
    t = torch.arange(s["longest"], device=q.device)[None, :] + from_key
    t = t.expand(len(n), -1)
    row = torch.where(i < n[:, None], s["q_start"][:-1].long()[:, None] + i, T)
    page = s["tables"].gather(1, (t // P).clamp(max=s["tables"].shape[1] - 1)).clamp(min=0).long()
    qs = torch.cat([q.float(), q.new_zeros(1, case["Hq"], D).float()])[row].view(len(n), -1, Hkv, G, D).transpose(1, 2)
    ks = s["k"][page, :, t % P].float().permute(0, 2, 3, 1)
    x = (qs.reshape(len(n), Hkv, -1, D) @ ks.contiguous()).mul_(D ** -0.5).view(len(n), Hkv, -1, G, t.shape[1])
    pos = (L - n)[:, None] + i
    live = _live(case, pos[:, :, None], t[:, None, :]) & (t < L[:, None])[:, None, :] & (i < n[:, None])[:, :, None]
    x.masked_fill_(~live[:, None, :, None, :], -math.inf)
    if lse is not None:
        z = torch.cat([lse, lse[:1]])
        z[row] = x.logsumexp(-1).permute(0, 2, 1, 3).reshape(len(n), -1, Hkv * G)
        lse.copy_(z[:-1])
    return x, row, t


def _state(x, v):
    """Maximum, sum and sums of values of rows of scores: m, l [...], o [..., D]."""
    m = x.amax(-1, keepdim=True)
    p = (x - torch.where(m == -math.inf, 0.0, m)).exp_()
    return m[..., 0], p.sum(-1), (p.flatten(2, 3) @ v).view(*x.shape[:-1], v.shape[-1])


def _plain_attention(s):
    case, q, o, lse = s["case"], s["q"], s["o"], s["lse"]
    Hkv, D, P, T = case["Hkv"], case["D"], case["page"], q.shape[0]
    G = case["Hq"] // Hkv
    # what each token sees of its prefix, and of its request's own keys
    m = q.new_full((2, T + 1, Hkv, G), -math.inf, dtype=torch.float32)
    l, acc = torch.zeros_like(m), q.new_zeros((2, T + 1, Hkv, G, D), dtype=torch.float32)
    rows, holder = s["group_rows"], s["group_holder"]
    t = torch.arange(s["prefix"], device=q.device)
    page = s["tables"][holder][:, t // P].clamp(min=0).long()
    qs = torch.cat([q.float(), q.new_zeros(1, case["Hq"], D).float()])[rows].view(len(rows), -1, Hkv, G, D).transpose(1, 2)
    ks = s["k"][page, :, t % P].float().permute(0, 2, 3, 1)
    vs = s["v"][page, :, t % P].float().transpose(1, 2)
    x = (qs.reshape(len(rows), Hkv, -1, D) @ ks.contiguous()).mul_(D ** -0.5).view(len(rows), Hkv, -1, G, len(t))
    n = s["q_start"][1:] - s["q_start"][:-1]
    req = torch.repeat_interleave(n, output_size=T - case["pad"])
    pos = torch.zeros(T + 1, dtype=torch.long, device=q.device)
    pos[:len(req)] = torch.arange(len(req), device=q.device) + (s["lengths"] - s["q_start"][1:])[req]
    live = _live(case, pos[rows][:, :, None], t) & (t < s["lengths"].long()[holder][:, None])[:, None, :]
    x.masked_fill_(~live[:, None, :, None, :], -math.inf)
    for part, at in zip((m, l, acc), _state(x, vs.contiguous())):
        part[0, rows] = at.transpose(1, 2)
    del x, ks, vs
    x, rows, t = _rows_scores(s)
    page = s["tables"].gather(1, (t // P).clamp(max=s["tables"].shape[1] - 1)).clamp(min=0).long()
    vs = s["v"][page, :, t % P].float().transpose(1, 2)
    for part, at in zip((m, l, acc), _state(x, vs.contiguous())):
        part[1, rows] = at.transpose(1, 2)
    # the two together
    m, l, acc = m[:, :len(req)], l[:, :len(req)], acc[:, :len(req)]
    top = m.amax(0)
    top = torch.where(top == -math.inf, 0.0, top)
    f = (m - top).exp()
    total = (f * l).sum(0)
    o[:len(req)] = ((f[..., None] * acc).sum(0) / torch.where(total == 0, 1.0, total)[..., None]).view(-1, Hkv * G, D).to(o.dtype)
    lse[:len(req)] = (top + total.log()).view(-1, Hkv * G)
    return o, lse


def _plain_weights(s):
    case, P, scores = s["case"], s["case"]["page"], s["scores"]
    x, row, t = _rows_scores(s)
    lse = torch.cat([s["lse"], s["lse"].new_zeros(1, case["Hq"])])[row].view(*row.shape, case["Hkv"], -1).transpose(1, 2)
    w = x.sub_(lse[..., None]).exp_().sum((2, 3))
    n, L = (s["q_start"][1:] - s["q_start"][:-1]).long(), s["lengths"].long()
    r, i = torch.nonzero((t >= s["first"][:, None]) & (t < L[:, None]), as_tuple=True)
    at = t[r, i]
    page, off = s["tables"][r, at // P].long(), at % P
    old = torch.where((at < (L - n)[r])[:, None], scores[page, :, off], 0.0)
    scores[page, :, off] = old + w[r, :, i]
    return scores


def _plain_choose(s):
    case, P = s["case"], s["case"]["page"]
    L, first = s["lengths"].long(), s["first"].long()
    t = torch.arange(s["tables"].shape[1] * P, device=L.device)
    x = s["scores"][:, s["tables"].clamp(min=0).long()].permute(0, 1, 3, 2, 4).flatten(3)
    # first the recent ones, then by score, ties by place, then those that are no candidates
    x = torch.where((t >= (L - case["recent"])[:, None])[None, :, None, :], math.inf, x)
    x = torch.where(((t < first[:, None]) | (t >= L[:, None]))[None, :, None, :], -math.inf, x)
    kept = x.sort(dim=-1, descending=True, stable=True)[1][..., :case["keep"]].sort(dim=-1)[0]
    kept = torch.cat([kept, kept.new_zeros(*kept.shape[:-1], case["keep"] - kept.shape[-1])], -1)
    gives = L - first > case["limit"]
    return (torch.where(gives[None, :, None, None], kept, -1).to(torch.int32),
            torch.where(gives, first + case["keep"], L).to(torch.int32))


def _plain_evict(s):
    P, kept, tables = s["case"]["page"], s["kept"], s["tables"].long()
    layer, r, h, j = torch.nonzero(kept >= 0, as_tuple=True)
    of = kept[layer, r, h, j].long()
    to = s["first"].long()[r] + j
    for x in (s["k"], s["v"], s["scores"]):
        x[layer, tables[r, to // P], h, to % P] = x[layer, tables[r, of // P], h, of % P]
    return s["k"], s["v"], s["scores"]


# ---- float64 -----------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "choose":
        return None
    if case["op"] == "evict":
        return _exact_evict(prepare(case, seed))
    s = _data(case, seed)
    length, fresh, _, _ = _sizes(case)
    G, P, D, Hkv = case["Hq"] // case["Hkv"], case["page"], case["D"], case["Hkv"]
    weigh = case["op"] == "weights"
    if weigh:
        s["lse"] = prepare(case, seed)["lse"]
        scores = s["scores"].double()
    else:
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    tables, t0 = s["tables"].long(), 0
    for r in range(len(length)):
        n, f = int(length[r]), int(fresh[r])
        k_pos = torch.arange(n, device="cuda")
        page, off = tables[r, k_pos // P], k_pos % P
        new = torch.arange(n - f, n, device="cuda")
        for h in range(Hkv if f else 0):
            kh = s["k"][page, h, off].double()
            vh = None if weigh else s["v"][page, h, off].double()
            w = torch.zeros(n, dtype=torch.float64, device="cuda")
            step = max(1, (1 << 27) // (G * n))
            for i in range(0, f, step):
                rows, heads = slice(t0 + i, t0 + min(f, i + step)), slice(h * G, (h + 1) * G)
                qh = s["q"][rows, heads].double()
                x = (qh.reshape(-1, D) @ kh.T).view(-1, G, n) / math.sqrt(D)
                x.masked_fill_(~_live(case, new[i:i + step, None], k_pos)[:, None, :], -math.inf)
                if weigh:
                    w += torch.exp(x - s["lse"][rows, heads].double()[..., None]).sum((0, 1))
                else:
                    z = torch.logsumexp(x, -1)
                    lse[rows, heads] = z
                    o[rows, heads] = (torch.exp(x - z[..., None]).view(-1, n) @ vh).view(-1, G, D)
            if weigh:
                a = case["first"]
                old = torch.where(k_pos < n - f, scores[page, h, off], 0.0)
                scores[page[a:], h, off[a:]] = (old + w)[a:]
        t0 += f
    return scores if weigh else (o, lse)


def _exact_evict(s):
    """Every kept row where it belongs, the others as they were."""
    case, tables = s["case"], s["tables"].long()
    P, out = case["page"], []
    places = torch.arange(tables.shape[1] * P, device="cuda")
    for x in (s["k"], s["v"], s["scores"][..., None]):
        y = x.double()
        for r in np.nonzero(_chosen(case))[0]:
            slots = tables[r, places // P] * P + places % P
            to = slots[case["first"]:case["first"] + case["keep"]]
            for layer in range(case["layers"]):
                for h in range(case["Hkv"]):
                    of = slots[s["kept"][layer, r, h].long()]
                    y[layer, to // P, h, to % P] = x[layer, of // P, h, of % P].double()
        out.append(y)
    return out[0], out[1], out[2][..., 0]
