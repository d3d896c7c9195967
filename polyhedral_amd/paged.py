"""Serving a batch of requests from a paged key / value cache.

The reference has no serving path; ``decode.KVCache`` keeps one length for all its heads in
``capacity`` rows each.  Here a layer's keys and values are pages of ``page_size`` tokens, K and
V [pages, heads, page_size, D], and request r's token at position t is row t % page_size of page
tables[r, t // page_size].  A step of a batch of requests, each with any number of new tokens
(none, one, a chunk of its prompt), packed one after the other:

1. ``build_tables``: from the tokens each request has and gets, on the device: pages taken from
   the free list, the tables, the packed rows' starts, slots and positions (pa_page_tables);
2. ``append``: the new keys and values to their slots (pa_paged_append);
3. ``attention``: every new token to all cached ones of its request, under any mask but an
   explicit matrix, query heads sharing KV heads in groups (pa_paged_attn).

``release`` gives pages back (pa_page_release).  Lengths, tables and counts stay on the device:
nothing here waits for it, and a step can be captured in a graph and replayed.  ``prepare_*``
validate once and return a launch that a program keeps for its buffers; ``PagedKVCache`` holds
the state of all this for a model's layers.
"""
import ctypes
import math
from collections import namedtuple

import torch

from . import _lib
from .spec import DENSE, DeviceMask, MaskSpec, _terms_by_name

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_POSITION = (1 << 30) - 1   # lengths stay at or below it

# status bits of a TableStep
SHORT_OF_PAGES, TOO_LONG, TOO_MANY_TOKENS = 1, 2, 4
LIST_FULL = 8   # in PagedKVCache.failed: a release that would have passed the free list's length

TableStep = namedtuple("TableStep", "lengths q_start slots positions free_count status")
TableStep.__doc__ = """int32 device tensors of a step: tokens of each request with the new ones, the packed rows'
starts [R + 1], each row's slot (page * page_size + row in the page) and position (-1 for rows of
no request), pages left free [1], status [1] (0, or SHORT_OF_PAGES + TOO_LONG + TOO_MANY_TOKENS:
nothing was taken then, and no row has a slot)."""


class PagedLaunch:
    """A validated call of the library with the tensors its pointers refer to; __call__ launches
    it on the current stream of its device and returns its result.  Runs of one launch share its
    outputs and its workspace: they must not overlap (runs in one stream do not), and a run on another
    stream than the one the launch was prepared on comes after that one's earlier work.  Keep it until
    its runs, or the graphs that hold them, are done."""

    def __init__(self, entry, call_args, keep, anchor, result, zero=None):
        self.entry, self.keep, self.anchor, self.result = entry, keep, anchor, result
        self._fn, self._args = getattr(_lib.lib(), entry), call_args
        self._zero = zero   # memory that is zero before the first run, and left zero by each

    def __call__(self):
        t = self.anchor
        if t.device.index == torch.cuda.current_device():
            return self._run(t)
        with torch.cuda.device(t.device):
            return self._run(t)

    def _run(self, t):
        if self._zero is not None:
            # (in the stream of the first run; a run that is only captured has not cleared it)
            self._zero.zero_()
            if not torch.cuda.is_current_stream_capturing():
                self._zero = None
        _lib.check(self._fn(*self._args, _lib.stream_of(t)), self.entry)
        return self.result


def _ints(t, name, shape=None, device=None):
    _lib.require_device(t)
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.numel() > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} needs a unit stride in its last dimension")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the others on {device}")
    return t


def _page_size(page_size):
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size={page_size}: one of {PAGE_SIZES}")


def _tables(t, R, page_size, device=None):
    _ints(t, "tables", device=device)
    if t.dim() != 2 or t.shape[0] != R:
        raise ValueError(f"tables must be [{R}, columns], got {tuple(t.shape)}")
    if t.shape[1] * page_size > MAX_POSITION:
        raise ValueError(f"{t.shape[1]} columns of {page_size} tokens pass the longest length, {MAX_POSITION}")
    # (one row has no pitch; a table whose rows overlap would be written through both)
    pitch = t.stride(0) if R > 1 else t.shape[1]
    if pitch < t.shape[1]:
        raise ValueError("the rows of tables overlap")
    return pitch


def prepare_tables(before, fresh, tables, free_list, free_count, page_size, tokens, out=None):
    """A PagedLaunch of one step of the tables; its result is a TableStep.

    before, fresh: int32 [R], the tokens each request holds and is to get.  tables: int32 [R,
    columns], written where a request gets a page (entries of pages it holds are read).
    free_list: int32 [pages], the free pages' ids in its first free_count[0] entries; they are
    taken from the end.  tokens: rows of the packed step (rows past the last request get slot and
    position -1).  out: a TableStep to write into (lengths may be ``before`` itself and free_count
    the given one: the state then advances with every run)."""
    _page_size(page_size)
    R = before.shape[0] if before.dim() == 1 else -1
    _ints(before, "before", (R,) if R >= 0 else (0,))
    dev = before.device
    _ints(fresh, "fresh", (R,), dev)
    pitch = _tables(tables, R, page_size, dev)
    if _ints(free_list, "free_list", device=dev).dim() != 1:
        raise ValueError("free_list must be [pages]")
    if free_list.shape[0] * page_size >= 1 << 31:
        raise ValueError(f"{free_list.shape[0]} pages of {page_size} rows: slots stay below 2^31")
    _ints(free_count, "free_count", (1,), dev)
    tokens = int(tokens)
    if not 0 <= tokens <= MAX_POSITION:
        raise ValueError(f"tokens={tokens} outside 0..{MAX_POSITION}")
    if out is None:
        new = lambda n: torch.empty(n, dtype=torch.int32, device=dev)  # noqa: E731
        out = TableStep(new(R), new(R + 1), new(tokens), new(tokens), new(1), new(1))
    else:
        for t, n, name in zip(out, (R, R + 1, tokens, tokens, 1, 1), TableStep._fields):
            _ints(t, f"out.{name}", (n,), dev)
    ws = torch.empty(3 * R + 2, dtype=torch.int32, device=dev)
    a = _lib.PaTablesArgs()
    ptr = _lib.address
    a.before, a.fresh, a.R = ptr(before), ptr(fresh), R
    a.free_list, a.free_count, a.n_pages = ptr(free_list), ptr(free_count), free_list.shape[0]
    a.page_size, a.tables, a.pitch, a.cols, a.tokens = page_size, ptr(tables), pitch, tables.shape[1], tokens
    a.lengths, a.q_start, a.slots, a.positions = ptr(out.lengths), ptr(out.q_start), ptr(out.slots), ptr(out.positions)
    a.free_left, a.status, a.workspace = ptr(out.free_count), ptr(out.status), ptr(ws)
    return PagedLaunch("pa_page_tables", (ctypes.byref(a),), [a, before, fresh, tables, free_list, free_count, ws, out],
                       before, out)


def build_tables(before, fresh, tables, free_list, free_count, page_size, tokens, out=None):
    """One step of the tables: see prepare_tables."""
    return prepare_tables(before, fresh, tables, free_list, free_count, page_size, tokens, out)()


def prepare_release(first, last, tables, free_list, free_count, out=None):
    """A PagedLaunch that gives back the pages first[r] .. last[r] - 1 (columns of the table; the
    range is clamped to it) of every request; entries without a page are skipped.  The pages go to
    the end of the free list in order of (request, column).  Its result is (free_count int32 [1],
    status int32 [1]: 1 when the list would pass its length, and then nothing changes); ``out``
    gives these tensors (free_count may be the given one)."""
    R = first.shape[0] if first.dim() == 1 else -1
    _ints(first, "first", (R,) if R >= 0 else (0,))
    dev = first.device
    _ints(last, "last", (R,), dev)
    pitch = _tables(tables, R, 1, dev)
    if _ints(free_list, "free_list", device=dev).dim() != 1:
        raise ValueError("free_list must be [pages]")
    _ints(free_count, "free_count", (1,), dev)
    if out is None:
        out = tuple(torch.empty(1, dtype=torch.int32, device=dev) for _ in range(2))
    else:
        for t, name in zip(out, ("free_count", "status")):
            _ints(t, f"out {name}", (1,), dev)
    ws = torch.empty(max(R, 1), dtype=torch.int32, device=dev)
    p = _lib.ptr
    args = (p(first), p(last), R, p(tables), pitch, tables.shape[1], p(free_list), p(free_count), free_list.shape[0],
            p(out[0]), p(out[1]), p(ws))
    return PagedLaunch("pa_page_release", args, [first, last, tables, free_list, free_count, ws, out], first, tuple(out))


def release(first, last, tables, free_list, free_count, out=None):
    """Pages back to the free list: see prepare_release."""
    return prepare_release(first, last, tables, free_list, free_count, out)()


def _strides(t):
    """The strides of all dimensions but the last; 0 where there is one entry, which no step leaves."""
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape, t.stride()[:-1]))


def _cache(k, v):
    """The checked shape (pages, heads, page_size, D) of a cache's tensors."""
    _lib.require_device(k, v)
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or _strides(k) != _strides(v) or k.device != v.device:
        raise ValueError("k and v must be [pages, heads, page_size, D] of one shape, dtype, strides and device")
    _lib.dtype_code(k)
    pages, H, P, D = k.shape
    _page_size(P)
    if D not in (64, 128):
        raise ValueError(f"D={D} (64 or 128)")
    if k.numel() and (k.stride(3) != 1 or v.stride(3) != 1):
        raise ValueError("the cache needs a unit stride in its last dimension")
    return pages, H, P, D


def _rows(t, name, shape, like):
    _lib.require_device(t)
    if t.dim() != 3 or tuple(t.shape) != tuple(shape) or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {list(shape)} {like.dtype} on {like.device}, got {list(t.shape)} {t.dtype} on "
                         f"{t.device}")
    if t.numel() and t.stride(2) != 1:
        raise ValueError(f"{name} needs a unit stride in its last dimension")


def prepare_append(k_new, v_new, slots, k, v):
    """A PagedLaunch that writes k_new, v_new [tokens, heads, D] (of the same strides, and no rows that
    slots name) to their slots (int32 [tokens], distinct; a slot outside the cache, as -1, is skipped)
    of k, v [pages, heads, page_size, D], whose rows do not overlap; its result is (k, v)."""
    pages, H, P, D = _cache(k, v)
    T = k_new.shape[0]
    _rows(k_new, "k_new", (T, H, D), k)
    _rows(v_new, "v_new", (T, H, D), k)
    if _strides(k_new) != _strides(v_new):
        raise ValueError("k_new and v_new must share strides")
    _ints(slots, "slots", (T,), k.device)
    p = _lib.ptr
    args = (p(k_new), p(v_new), *_strides(k_new), p(slots), T, p(k), p(v), *_strides(k), pages, P, H, D, _lib.dtype_code(k))
    return PagedLaunch("pa_paged_append", args, [k_new, v_new, slots, k, v], k, (k, v))


def append(k_new, v_new, slots, k, v):
    """New keys and values to their slots: see prepare_append."""
    return prepare_append(k_new, v_new, slots, k, v)()


def _paged_mask(mask):
    """The DeviceMask of a mask that has terms (no matrix, no tables)."""
    if isinstance(mask, MaskSpec):
        mask = DeviceMask(mask)
    if not isinstance(mask, DeviceMask):
        terms = _terms_by_name(mask)
        if terms is None:
            raise ValueError(f"{mask!r} is not a mask of positions: a matrix or a permuted mask has no meaning for requests "
                             "of different lengths")
        mask = DeviceMask(MaskSpec(tuple(terms[0]), tuple(terms[1])))
    if mask.perm_q is not None or mask.perm_kv is not None:
        raise ValueError("the mask takes no permutation tables: it is evaluated at the tokens' positions")
    if any(t[0] == DENSE for t in mask.spec.include + mask.spec.exclude):
        raise ValueError("a mask matrix has no meaning for requests of different lengths")
    return mask


def prepare_attention(q, k, v, tables, lengths, q_start, mask, scale=None, max_fresh=None, out=None, lse=None):
    """A PagedLaunch of the requests' newest tokens against all their cached ones.

    q [tokens, Hq, D]: rows q_start[r] .. q_start[r + 1] - 1 are request r's newest tokens, at
    positions lengths[r] - n .. lengths[r] - 1 (their keys and values appended already).  k, v
    [pages, Hkv, page_size, D]; query head h reads KV head h // (Hq // Hkv).  tables int32 [R,
    columns], lengths int32 [R], q_start int32 [R + 1], on the device.  mask: a polyattn mask
    object, a MaskSpec or a DeviceMask without tables, evaluated at positions; keys
    past a request's length are never live, and neither are keys whose table entry names no page.
    scale: positive, 1/sqrt(D) by default.  max_fresh: the most new tokens of a request, where the
    program knows it (it selects kernels; any value gives right results).  out: [tokens, Hq, D];
    lse: None or float32 [tokens, Hq], the natural-log sum-exp; neither shares memory with an
    input, the other or itself (a call that does is refused when it is launched).  A row with no
    live key gives 0 and -inf; rows of no request are left as they are (in a new ``out``: as its
    memory was).  The result is out."""
    pages, Hkv, P, D = _cache(k, v)
    if q.dim() != 3:
        raise ValueError("q must be [tokens, heads, D]")
    T, Hq = q.shape[0], q.shape[1]
    _rows(q, "q", (T, Hq, D), k)
    if Hq < 1 or Hkv < 1 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads are no multiple of {Hkv} KV heads")
    dev = k.device
    R = lengths.shape[0] if lengths.dim() == 1 else -1
    _ints(lengths, "lengths", (R,) if R >= 0 else (0,), dev)
    _ints(q_start, "q_start", (R + 1,), dev)
    pitch = _tables(tables, R, P, dev)
    dm = _paged_mask(mask)
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError(f"scale={scale} must be positive")
    max_fresh = T if max_fresh is None else int(max_fresh)
    if max_fresh < 0:
        raise ValueError(f"max_fresh={max_fresh} < 0")
    o = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    _rows(o, "out", (T, Hq, D), k)
    a = _lib.PaPagedArgs()
    ptr = _lib.address
    a.q, (a.q_st, a.q_sh) = ptr(q), _strides(q)
    a.k, a.v = ptr(k), ptr(v)
    a.c_sp, a.c_sh, a.c_sn = _strides(k)
    a.n_pages, a.page_size = pages, P
    a.tables, a.pitch, a.cols = ptr(tables), pitch, tables.shape[1]
    a.lengths, a.q_start, a.R, a.T, a.max_fresh = ptr(lengths), ptr(q_start), R, T, min(max_fresh, T)
    a.Hq, a.Hkv, a.D, a.dtype, a.scale = Hq, Hkv, D, _lib.dtype_code(q), scale
    a.mask = dm.struct()
    a.o, (a.o_st, a.o_sh) = ptr(o), _strides(o)
    if lse is not None:
        _lib.require_device(lse)
        if lse.dtype != torch.float32 or lse.shape != (T, Hq) or lse.device != dev:
            raise ValueError(f"lse must be float32 [{T}, {Hq}] on {dev}")
        a.lse, a.lse_st, a.lse_sh = ptr(lse), lse.stride(0), lse.stride(1)
    nbytes, zero = ctypes.c_int64(0), ctypes.c_int64(0)
    _lib.check(_lib.lib().pa_paged_workspace(ctypes.byref(a), ctypes.byref(nbytes), ctypes.byref(zero)), "pa_paged_workspace")
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ptr(ws), nbytes.value
    return PagedLaunch("pa_paged_attn", (ctypes.byref(a),), [a, q, k, v, tables, lengths, q_start, dm, o, lse, ws], k, o,
                       zero=ws[:zero.value])


def attention(q, k, v, tables, lengths, q_start, mask, scale=None, max_fresh=None, out=None, lse=None):
    """o [tokens, Hq, D]: see prepare_attention."""
    return prepare_attention(q, k, v, tables, lengths, q_start, mask, scale, max_fresh, out, lse)()


def _on_device(values, dtype, device):
    """A list's values on the device, through pinned memory that its allocator keeps until they have been
    read: the host does not wait."""
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("values from the host have no place in a graph's capture: give a tensor on the device")
        return torch.as_tensor(values, dtype=dtype).pin_memory().to(device, non_blocking=True)


class PagedKVCache:
    """Keys and values of up to ``requests`` requests at once, for ``layers`` layers that share
    their tables: k, v [layers, pages, heads, page_size, D].

    A step: ``step = cache.begin(fresh)``, then for each layer ``cache.append(k_new, v_new, step,
    layer)`` and ``cache.attend(q, mask, step, layer)``, before the next begin, trim or finish.
    ``trim`` gives back what a window has left behind, ``finish`` all of some requests' pages (their
    rows then start anew).  All state is in tensors on the device that stay where they are, so a
    whole step with counts on the device can be captured in a graph, and every replay is a step;
    only ``check`` waits for the device."""

    def __init__(self, requests, max_length, pages, heads, D, dtype=torch.bfloat16, page_size=64, layers=1, device=None):
        _page_size(page_size)
        if requests < 1 or max_length < 1 or pages < 1 or heads < 1 or layers < 1:
            raise ValueError("requests, max_length, pages, heads and layers must be at least 1")
        if pages * page_size >= 1 << 31:
            raise ValueError(f"{pages} pages of {page_size} rows: slots stay below 2^31")
        if max_length > MAX_POSITION - page_size:
            raise ValueError(f"max_length={max_length} passes {MAX_POSITION - page_size}")
        dev = torch.device("cuda" if device is None else device)
        if dev.type == "cuda" and dev.index is None:   # (tensors name their device by its index)
            dev = torch.device("cuda", torch.cuda.current_device())
        i32 = dict(dtype=torch.int32, device=dev)
        self.k = torch.zeros(layers, pages, heads, page_size, D, dtype=dtype, device=dev)
        self.v = torch.zeros_like(self.k)
        _cache(self.k[0], self.v[0])
        self.requests, self.page_size, self.pages, self.device = requests, page_size, pages, dev
        self.tables = torch.full((requests, -(-max_length // page_size)), -1, **i32)
        self.max_length = self.tables.shape[1] * page_size   # whole pages
        self.lengths = torch.zeros(requests, **i32)
        self.free_list = torch.arange(pages - 1, -1, -1, **i32)   # page 0 is taken first
        self.free_count = torch.full((1,), pages, **i32)
        self.failed = torch.zeros(1, **i32)    # the status bits of all steps so far
        self._last = (None, None)              # the newest step and its most new tokens of a request

    def begin(self, fresh, tokens=None):
        """Room for fresh[r] more tokens of every request (int32 [requests] on the device, or a list
        of counts, which a graph's capture does not take), packed into ``tokens`` rows (default, for a
        list: their sum; rows beyond are padding).  Returns the TableStep; lengths count the new tokens from here on.  A step that
        does not fit (pages, max_length, rows) takes nothing, gives no row a slot, and shows in
        step.status and ``check``."""
        most = None
        if not isinstance(fresh, torch.Tensor):
            fresh = [int(f) for f in fresh]
            most = max(fresh, default=0)
            tokens = sum(fresh) if tokens is None else tokens
            fresh = _on_device(fresh, torch.int32, self.device)
        if tokens is None:
            raise ValueError("tokens (the rows of the packed step) is needed with counts on the device")
        _ints(fresh, "fresh", (self.requests,), self.device)
        new = lambda n: torch.empty(n, dtype=torch.int32, device=self.device)  # noqa: E731
        out = TableStep(self.lengths, new(self.requests + 1), new(tokens), new(tokens), self.free_count, new(1))
        step = build_tables(self.lengths, fresh, self.tables, self.free_list, self.free_count, self.page_size, tokens, out)
        with torch.cuda.device(self.device):
            self.failed |= step.status
        self._last = (step, most)
        return step

    def append(self, k_new, v_new, step, layer=0):
        """k_new, v_new [tokens, heads, D] of a step into a layer's pages."""
        append(k_new, v_new, step.slots, self.k[layer], self.v[layer])

    def attend(self, q, mask, step, layer=0, scale=None, max_fresh=None, out=None, lse=None):
        """o [tokens, Hq, D] of a step's tokens against a layer's pages (see prepare_attention; of the
        newest step max_fresh is known where its counts were a list)."""
        if max_fresh is None and step is self._last[0]:
            max_fresh = self._last[1]
        return attention(q, self.k[layer], self.v[layer], self.tables, step.lengths, step.q_start, mask, scale, max_fresh,
                         out, lse)

    def _release(self, first, last):
        status = torch.empty(1, dtype=torch.int32, device=self.device)
        release(first, last, self.tables, self.free_list, self.free_count, (self.free_count, status))
        with torch.cuda.device(self.device):
            self.failed |= status * LIST_FULL

    def finish(self, done):
        """Gives back the pages of the requests where done (bool [requests], on the device, or a list,
        which a graph's capture does not take) is true and sets their lengths to 0."""
        if not (isinstance(done, torch.Tensor) and done.is_cuda):
            done = _on_device(done, torch.bool, self.device)
        done = done.to(device=self.device, dtype=torch.bool)
        if done.shape != (self.requests,):
            raise ValueError(f"done must be [{self.requests}], got {list(done.shape)}")
        with torch.cuda.device(self.device):
            last = done.to(torch.int32) * self.tables.shape[1]
            self._release(torch.zeros_like(last), last)
            self.lengths.masked_fill_(done, 0)

    def trim(self, window, sinks=0):
        """Gives back the pages that neither the next token's window nor the first ``sinks`` tokens
        need: with a SinksWindow(sinks, window) mask no later token sees them."""
        if window < 1 or sinks < 0:
            raise ValueError(f"window={window} must be at least 1 and sinks={sinks} at least 0")
        P = self.page_size
        with torch.cuda.device(self.device):
            last = ((self.lengths - int(min(window, MAX_POSITION)) + 1).clamp(min=0) // P).to(torch.int32)
            first = torch.full_like(last, min(-(-int(sinks) // P), self.tables.shape[1]))
            self._release(first, last)

    def check(self):
        """Waits for the device and raises if a step so far did not fit."""
        bits = int(self.failed.item())
        if bits:
            why = [w for b, w in ((SHORT_OF_PAGES, "too few free pages"), (TOO_LONG, f"a request past {self.max_length} tokens"),
                                  (TOO_MANY_TOKENS, "more new tokens than rows"),
                                  (LIST_FULL, "more pages given back than there are")) if bits & b]
            raise RuntimeError("a step did not fit: " + ", ".join(why))
