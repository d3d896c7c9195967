"""Calls that the paged cache's documentation allows (polyhedral_amd.paged), beside those of
tests/test_gpu_paged.py."""
import numpy as np
import pytest
import torch

from polyhedral_amd import _lib, paged
from polyhedral_amd.polyattn import masks as pm
from tests.test_gpu_paged import Batch

pytestmark = pytest.mark.gpu

I32 = torch.int32


@pytest.mark.parametrize("device", [None, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda", 0)], ids=str)
def test_a_cache_on_any_name_of_its_device(gpu, device):
    cache = paged.PagedKVCache(2, 64, 8, 2, 64, torch.float16, 16, device=device)
    assert cache.device == cache.k.device == gpu
    new = torch.ones(5, 2, 64, dtype=torch.float16, device=gpu)
    step = cache.begin([3, 2])
    cache.append(new, new, step)
    assert torch.equal(cache.attend(new, pm.Causal(), step), new)
    cache.begin(torch.ones(2, dtype=I32, device="cuda"), 2)
    cache.trim(4)
    cache.finish([True, False])
    assert cache.lengths.tolist() == [0, 3]
    cache.check()


# ---- tensors that are parts of one buffer -------------------------------------------------------
@pytest.mark.parametrize("dtype,D,sizes", [(torch.float32, 64, [(1, 300), (3, 40)]), (torch.bfloat16, 128, [(1, 3000), (150, 400)]),
                                           (torch.float16, 64, [(40, 90)])])
def test_outputs_beside_inputs_in_one_buffer(gpu, dtype, D, sizes):
    """q and out are heads of one buffer in turn, or halves of its rows; out and lse are packed; K and V
    of a page lie side by side."""
    b = Batch(gpu, dtype, D, 16, 4, 2, sizes)
    want, wl = b.run(pm.Causal())
    kv = torch.stack([b.k, b.v], dim=1)
    k, v = kv[:, 0], kv[:, 1]
    heads = torch.full((b.T, 4, 2, D), 7.0, dtype=dtype, device=gpu)
    heads[:, :, 0] = b.q
    halves = torch.full((b.T, 8, D), 7.0, dtype=dtype, device=gpu)
    halves[:, 4:] = b.q
    lse = torch.full((b.T, 4), 7.0, device=gpu)
    for q, o in ((heads[:, :, 0], heads[:, :, 1]), (halves[:, 4:], halves[:, :4])):
        paged.attention(q, k, v, *b.dev(), pm.Causal(), out=o, lse=lse)
        assert torch.equal(o, want) and torch.equal(lse, wl) and torch.equal(q, b.q)
    if dtype == torch.float32:
        packed = torch.full((b.T, 4, D + 4), 7.0, device=gpu)
        paged.attention(b.q, k, v, *b.dev(), pm.Causal(), out=packed[..., :D], lse=packed[..., D])
        assert torch.equal(packed[..., :D], want) and torch.equal(packed[..., D], wl) and (packed[..., D + 1:] == 7).all()


def test_outputs_that_share_memory_are_refused(gpu):
    b = Batch(gpu, torch.float16, 64, 16, 4, 2, [(1, 20), (2, 30)])
    shape = (b.T, 4, 64)
    lse = torch.zeros(b.T, 4, device=gpu)

    def refused(match, **change):
        before = {n: t.clone() for n, t in (("q", b.q), ("k", b.k), ("v", b.v))}
        with pytest.raises(_lib.PolyattnError, match=match):
            paged.attention(b.q, b.k, b.v, *b.dev(), pm.Causal(), **change)
        assert all(torch.equal(t.nan_to_num(), getattr(b, n).nan_to_num()) for n, t in before.items())
    refused("rows of o overlap", out=torch.zeros(1, 4, 64, dtype=b.dtype, device=gpu).expand(shape))
    refused("rows of o overlap", out=torch.zeros(b.T, 1, 64, dtype=b.dtype, device=gpu).expand(shape))
    refused("rows of lse overlap", lse=torch.zeros(1, 4, device=gpu).expand(b.T, 4))
    refused("rows of lse overlap", lse=torch.zeros(b.T, 1, device=gpu).expand(b.T, 4))
    refused("o and q", out=b.q)
    refused("o and k", out=b.k.view(-1, 4, 64)[:b.T])
    both = torch.zeros(b.T, 4, 64, dtype=torch.float32, device=gpu)
    refused("o and lse", out=both.view(torch.float16)[..., :64], lse=both[..., 0])
    paged.attention(b.q, b.k, b.v, *b.dev(), pm.Causal(), lse=lse)


@pytest.mark.parametrize("layout", ["[pages, 2, H, P, D]", "[pages, H, P, 2, D]", "[2, pages, H, P, D]", "[pages, P, 2, H, D]",
                                    "[2 pages, H, P, D]", "v before k", "v a page on", "v two pages on", "k is v"])
def test_append_into_one_buffer_of_keys_and_values(gpu, layout):
    pages, H, P, D = 5, 3, 16, 64
    order = {"[pages, 2, H, P, D]": (0, 4, 1, 2, 3), "[pages, H, P, 2, D]": (0, 1, 2, 4, 3), "[pages, P, 2, H, D]": (0, 2, 4, 1, 3),
             "[2 pages, H, P, D]": (0, 4, 1, 2, 3)}.get(layout, (4, 0, 1, 2, 3))
    sizes = (pages, H, P, D, 2)
    buf = torch.zeros([sizes[i] for i in order], dtype=torch.float16, device=gpu)
    kv = buf.permute([order.index(i) for i in (4, 0, 1, 2, 3)])
    if layout.endswith("on"):
        on = 1 if layout == "v a page on" else 2
        buf = torch.zeros(pages + on, 2, H, P, D, dtype=torch.float16, device=gpu)
        kv = buf[:pages, 0], buf[on:, 1]
    k, v = (kv[1], kv[0]) if layout == "v before k" else (kv[0], kv[0 if layout == "k is v" else 1])
    new = torch.randn(2, 7, H, D, device=gpu).half()
    kn, vn = new[0], new[0 if layout == "k is v" else 1]
    slots = torch.tensor([0, 17, -1, 79, 33, 5, 80], dtype=I32, device=gpu)
    want = [torch.zeros(pages, H, P, D, dtype=torch.float16, device=gpu) for _ in range(2)]
    for w, n in zip(want, (kn, vn)):
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < pages * P:
                w[s // P, :, s % P] = n[i]
    paged.append(kn, vn, slots, k, v)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_strides_of_one_entry_do_not_matter(gpu):
    """One token, one head or one page: whatever stride its dimension has."""
    H, P, D = 2, 16, 64
    k, v = (torch.zeros(4, H, P, D, dtype=torch.float16, device=gpu) for _ in range(2))
    fused = torch.randn(2, 3 * H * D + 5, device=gpu).half()
    part = lambda i: fused.as_strided((1, H, D), (3 * H * D + 5, D, 1), i * H * D)  # noqa: E731
    slot = torch.tensor([20], dtype=I32, device=gpu)
    # k_new a part of a row whose pitch is no multiple of 16 bytes, v_new a tensor of its own
    kn, vn = part(1), torch.randn(1, H, D, device=gpu).half()
    assert kn.stride() != vn.stride()
    paged.append(kn, vn, slot, k, v)
    assert torch.equal(k[1, :, 4], kn[0]) and torch.equal(v[1, :, 4], vn[0]) and int((k != 0).any(-1).sum()) == H
    # one head
    two = torch.randn(3, 2, D, device=gpu).half()
    k1, v1 = (torch.zeros(4, 1, P, D, dtype=torch.float16, device=gpu) for _ in range(2))
    paged.append(two.as_strided((3, 1, D), (2 * D, 5, 1)), two[:, 1:], torch.tensor([1, 2, 3], dtype=I32, device=gpu), k1, v1)
    assert torch.equal(k1[0, 0, 1:4], two[:, 0]) and torch.equal(v1[0, 0, 1:4], two[:, 1])
    # one page and one token: its query heads in a row of the fused projection, of an odd pitch
    q = part(0)
    page_k = k.as_strided((1, H, P, D), (1, P * D, D, 1), H * P * D)
    page_v = v[1:2]
    i32 = lambda *x: torch.tensor(x, dtype=I32, device=gpu)  # noqa: E731
    args = (torch.zeros(1, 1, dtype=I32, device=gpu), i32(5), i32(0, 1), pm.SlidingWindow(1))
    out = torch.empty(H * D, dtype=torch.float16, device=gpu).as_strided((1, H, D), (H * D + 3, D, 1))
    assert torch.equal(paged.attention(q, page_k, page_v, *args, out=out), vn) and out.stride() != vn.stride()
    # strides that do count are still compared
    with pytest.raises(ValueError, match="share strides"):
        paged.append(two, two.transpose(0, 1).contiguous().transpose(0, 1), i32(1, 2, 3), k, v)


# ---- what is out of range ---------------------------------------------------------------------------
def test_lengths_and_starts_out_of_range_are_clamped(gpu):
    """Lengths to what the table reaches, starts to the rows there are and to those before them."""
    b = Batch(gpu, torch.bfloat16, 128, 16, 4, 2, [(2, 50), (1, 30), (40, 90)], pad=0)
    cols = b.tables.shape[1]
    for lengths, starts in (([1 << 30, -5, 90], [0, 2, 3, 43]), ([50, 30, 90], [0, 100, 3, 1 << 30]), ([1, 0, 1], [0, 2, 3, 43]),
                            ([50, 30, 90], [-9, 2, 1, 43]), ([50, 30, 90], [5, 7, 8, 20])):
        b.lengths = np.array(lengths)
        b.q_start = np.array(starts)
        o, lse = b.run(pm.Causal())
        s = np.maximum.accumulate(np.clip(starts, 0, b.T))
        c = Batch(gpu, torch.bfloat16, 128, 16, 4, 2, [(2, 50), (1, 30), (40, 90)], pad=0)
        c.lengths, c.q_start = np.clip(lengths, 0, cols * 16), s
        want, wl = c.run(pm.Causal())
        assert torch.equal(torch.nan_to_num(o.float()), torch.nan_to_num(want.float())) and torch.equal(lse.isnan(), wl.isnan())
        assert torch.equal(torch.nan_to_num(lse), torch.nan_to_num(wl))
        outside = torch.ones(b.T, dtype=torch.bool, device=gpu)
        outside[int(s[0]):int(s[-1])] = False
        assert (o[outside] == 7).all() and (lse[outside] == 7).all()


# ---- what waits for the device ----------------------------------------------------------------------
def test_counts_in_a_list_do_not_wait_for_the_device(gpu):
    """begin and finish return while the work before them still runs, and take the counts they were given
    even where the same memory is given again before the device has read it."""
    cache = paged.PagedKVCache(3, 256, 60, 1, 64, torch.float16, 16, device=gpu)
    cache.begin([1, 0, 2])
    cache.finish([False, True, False])
    a = torch.randn(8192, 8192, device=gpu).bfloat16()
    out = torch.empty_like(a)
    torch.mm(a, a, out=out)
    torch.cuda.synchronize()
    for _ in range(40):
        torch.mm(a, a, out=out)
    done = torch.cuda.Event()
    done.record()
    steps = [cache.begin([i, 2 * i, 1]) for i in range(8)]
    cache.finish([False, True, False])
    cache.begin([0, 7, 0])
    waited = done.query()
    torch.cuda.synchronize()
    assert not waited
    assert cache.lengths.tolist() == [1 + 28, 7, 2 + 8]
    assert [s.q_start.tolist() for s in steps] == [[0, i, 3 * i, 3 * i + 1] for i in range(8)]
    cache.check()


def test_counts_in_a_list_are_refused_in_a_capture(gpu):
    """A graph would replay the copy of memory that has gone on to other uses."""
    cache = paged.PagedKVCache(2, 64, 8, 1, 64, torch.float16, 16, device=gpu)
    for call in (lambda: cache.begin([1, 1]), lambda: cache.finish([True, False])):
        with pytest.raises(RuntimeError, match="capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        torch.cuda.synchronize()
    cache.begin([1, 1])
    assert cache.lengths.tolist() == [1, 1]


def test_captured_finish_and_trim(gpu):
    """A whole round of a server in one graph, finish and trim with masks on the device among it, on a
    stream of its own; replays against a second cache stepped eagerly."""
    R, H, D, P = 5, 2, 64, 16
    mask = pm.SinksWindow(3, 40)
    a, e = (paged.PagedKVCache(R, 400, 100, H, D, torch.bfloat16, P, 1, gpu) for _ in range(2))
    gen, rng = torch.Generator().manual_seed(3), np.random.default_rng(3)
    T = 30
    fresh, done = torch.zeros(R, dtype=I32, device=gpu), torch.zeros(R, dtype=torch.bool, device=gpu)
    kn, vn, q = (torch.zeros(T, n, D, dtype=torch.bfloat16, device=gpu) for n in (H, H, 2 * H))
    oa, oe = (torch.zeros(T, 2 * H, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))

    def a_round(cache, out):
        cache.finish(done)
        step = cache.begin(fresh, T)
        cache.append(kn, vn, step)
        cache.attend(q, mask, step, out=out)
        cache.trim(40, 3)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        a_round(a, oa)
    for i in range(30):
        n = rng.integers(0, 6, R)
        fresh.copy_(torch.as_tensor(n, dtype=I32))
        done.copy_(torch.as_tensor(rng.random(R) < 0.15))
        for x in (kn, vn, q):
            x.copy_(torch.randn(x.shape, generator=gen))
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph.replay()
        a_round(e, oe)
        torch.cuda.current_stream().wait_stream(stream)
        for x, y in ((a.tables, e.tables), (a.lengths, e.lengths), (a.free_count, e.free_count), (oa, oe)):
            assert torch.equal(x, y), i
        used = a.tables.cpu().numpy()
        used = used[used >= 0]
        free = a.free_list.cpu().numpy()[:int(a.free_count)]
        assert sorted(np.concatenate([used, free]).tolist()) == list(range(a.pages)), i
    a.check()
    e.check()


@pytest.mark.parametrize("dtype,n", [(torch.float16, 1), (torch.bfloat16, 40), (torch.float32, 2)])
def test_millions_of_tokens(gpu, dtype, n):
    """One request of 3 million tokens whose keys are all alike: the mean of its values, row by row."""
    L, P, D, G = 3_000_001, 256, 64, 4
    pages = -(-L // P)
    k = torch.ones(pages, 1, P, D, dtype=dtype, device=gpu)
    v = torch.randn(pages, 1, P, D, device=gpu).add_(1.0).to(dtype)
    perm = torch.randperm(pages, device=gpu)
    q = torch.randn(n, G, D, device=gpu).to(dtype)
    lse = torch.zeros(n, G, device=gpu)
    o = paged.attention(q, k, v, perm[None].to(I32), torch.tensor([L], dtype=I32, device=gpu),
                        torch.tensor([0, n], dtype=I32, device=gpu), pm.Causal(), lse=lse)
    rows = v[perm].reshape(-1, D).double()
    # every P is the same, 1 but for the rounding of its maximum in log2 units (2^-21 of it), which all sums
    # share; O and the sum of P are two chains of at most 2^11 additions, in a share and over the shares, each
    # off by 2^-24 of what is summed: 2^-12 in all; scores by (D + 2) 2^-24 of their terms
    for i in range(n):
        m = L - n + i + 1
        want, mass = rows[:m].mean(0), rows[:m].abs().mean(0)
        u = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
        assert ((o[i].double() - want).abs() <= 1.01 * u * want.abs() + 2.0 ** -11 * mass).all(), i   # (O and its divisor)
        x = q[i].double().sum(-1) * D ** -0.5
        terms = q[i].double().abs().sum(-1).max() * D ** -0.5
        assert (lse[i].double() - x - np.log(m)).abs().max() <= 2.0 ** -12 + (D + 2) * 2.0 ** -24 * terms
