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

``release`` gives pages back (pa_page_release).

Requests whose tables name the same pages in front share a prefix: ``sharing`` finds which of a step's
tokens do (pa_share_rows), once for all layers, and ``shared_attention`` reads each prefix once for all
of them (pa_shared_attn).  Keys can be given up one by one: ``weights`` adds up the attention that
each has received (pa_paged_weights), ``choose`` picks those that stay (pa_choose_keys), and ``evict`` moves
them to the front of their request's pages (pa_evict_rows), after which their places count as their
positions.

Lengths, tables and counts stay on the device:
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

SHARED = 16      # there too: a prefix that could not be shared, or its request finished before those that share it
TRIMMED = 32     # there too: a request that was to be evicted had given back pages in front

TableStep = namedtuple("TableStep", "lengths q_start slots positions free_count status")
TableStep.__doc__ = """int32 device tensors of a step: tokens of each request with the new ones, the packed rows'
starts [R + 1], each row's slot (page * page_size + row in the page) and position (-1 for rows of
no request), pages left free [1], status [1] (0, or SHORT_OF_PAGES + TOO_LONG + TOO_MANY_TOKENS:
nothing was taken then, and no row has a slot)."""


Sharing = namedtuple("Sharing", "start rows positions prefix low high first")
Sharing.__doc__ = """int32 device tensors: which of a step's tokens share a prefix.  The tokens of the requests that
share request g's are rows[start[g]:start[g + 1]] of the packed step, at positions[..]; prefix[g] (tokens
of the prefix), low[g] and high[g] (the least and largest position) are 0 where there is no group;
first[r] is prefix[g] for the requests of a group, 0 for others."""

Choice = namedtuple("Choice", "kept lengths")
Choice.__doc__ = """int32 device tensors: the places that stay [layers,] requests, heads, keep], ascending (-1: the request
keeps all), and each request's length after their move."""


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


def _scale(scale, D):
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError(f"scale={scale} must be positive")
    return scale


def _workspace(sizes, a, device):
    """The workspace of the call with arguments ``a``, whose pointer is set, and the part of it that is zero
    before the first run (None: none)."""
    nbytes, zero = ctypes.c_int64(0), ctypes.c_int64(0)
    _lib.check(getattr(_lib.lib(), sizes)(ctypes.byref(a), ctypes.byref(nbytes), ctypes.byref(zero)), sizes)
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = _lib.address(ws), nbytes.value
    return ws, ws[:zero.value] if zero.value else None


def _attention_launch(entry, q, k, v, tables, lengths, q_start, sharing, mask, scale, max_fresh, out, lse):
    """The PagedLaunch of prepare_attention and prepare_shared_attention."""
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
    scale = _scale(scale, D)
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
    call, sizes = (ctypes.byref(a),), entry + "_workspace"
    if sharing is not None:
        s = _sharing_struct(sharing, R, T, dev)
        call += (ctypes.byref(s),)
    ws, zero = _workspace(sizes, a, dev)
    return PagedLaunch(entry + "_attn", call, [call, a, q, k, v, tables, lengths, q_start, sharing, dm, o, lse, ws], k, o,
                       zero=zero)


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
    return _attention_launch("pa_paged", q, k, v, tables, lengths, q_start, None, mask, scale, max_fresh, out, lse)


def attention(q, k, v, tables, lengths, q_start, mask, scale=None, max_fresh=None, out=None, lse=None):
    """o [tokens, Hq, D]: see prepare_attention."""
    return prepare_attention(q, k, v, tables, lengths, q_start, mask, scale, max_fresh, out, lse)()


def prepare_sharing(lengths, q_start, holders, shared, page_size, tokens, out=None):
    """A PagedLaunch that finds which tokens of a step share a prefix; its result is a Sharing, which
    holds for all layers of the step.

    lengths, q_start: as in prepare_attention.  holders, shared: int32 [R], the request whose first
    shared[r] tokens request r shares (-1: none), with that request's pages in its own table; only whole
    pages are shared.  The length of a request that shares holds its new tokens and lies within its table.  A request may be its own holder.  A prefix that one request alone has tokens for
    is no group.  tokens: rows of the packed step.  out: a Sharing to write into."""
    _page_size(page_size)
    R = lengths.shape[0] if lengths.dim() == 1 else -1
    _ints(lengths, "lengths", (R,) if R >= 0 else (0,))
    dev = lengths.device
    _ints(q_start, "q_start", (R + 1,), dev)
    _ints(holders, "holders", (R,), dev)
    _ints(shared, "shared", (R,), dev)
    tokens = int(tokens)
    if not 0 <= tokens <= MAX_POSITION:
        raise ValueError(f"tokens={tokens} outside 0..{MAX_POSITION}")
    sizes = (R + 1, tokens, tokens, R, R, R, R)
    if out is None:
        out = Sharing(*(torch.empty(n, dtype=torch.int32, device=dev) for n in sizes))
    else:
        for t, n, name in zip(out, sizes, Sharing._fields):
            _ints(t, f"out.{name}", (n,), dev)
        out = Sharing(*out)
    ws = torch.empty(max(8 * R, 1), dtype=torch.int32, device=dev)
    a = _lib.PaShareArgs()
    ptr = _lib.address
    a.lengths, a.q_start, a.holders, a.shared = ptr(lengths), ptr(q_start), ptr(holders), ptr(shared)
    a.R, a.page_size, a.T, a.workspace = R, page_size, tokens, ptr(ws)
    for name, t in zip(Sharing._fields, out):
        setattr(a, name, ptr(t))
    return PagedLaunch("pa_share_rows", (ctypes.byref(a),), [a, lengths, q_start, holders, shared, ws, out], lengths, out)


def sharing(lengths, q_start, holders, shared, page_size, tokens, out=None):
    """Which tokens of a step share a prefix: see prepare_sharing."""
    return prepare_sharing(lengths, q_start, holders, shared, page_size, tokens, out)()


def _sharing_struct(sharing, R, T, device):
    s = _lib.PaSharing()
    for t, n, name in zip(sharing, (R + 1, T, T, R, R, R, R), Sharing._fields):
        _ints(t, f"sharing.{name}", (n,), device)
        setattr(s, name, _lib.address(t))
    return s


def prepare_shared_attention(q, k, v, tables, lengths, q_start, sharing, mask, scale=None, max_fresh=None, out=None, lse=None):
    """A PagedLaunch of prepare_attention's result where requests share prefixes: the keys of a shared
    prefix are read once for all rows of its group, from its holder's table, and each request's own from
    its.  sharing: the Sharing of this step; the other arguments and the result as in prepare_attention."""
    return _attention_launch("pa_shared", q, k, v, tables, lengths, q_start, sharing, mask, scale, max_fresh, out, lse)


def shared_attention(q, k, v, tables, lengths, q_start, sharing, mask, scale=None, max_fresh=None, out=None, lse=None):
    """o [tokens, Hq, D]: see prepare_shared_attention."""
    return prepare_shared_attention(q, k, v, tables, lengths, q_start, sharing, mask, scale, max_fresh, out, lse)()


def _scores(t, shape, device):
    """The checked strides of scores of all dimensions but the last."""
    _lib.require_device(t)
    if t.dtype != torch.float32 or tuple(t.shape) != tuple(shape) or t.device != device:
        raise ValueError(f"scores must be float32 {list(shape)} on {device}, got {list(t.shape)} {t.dtype} on {t.device}")
    if t.numel() and t.stride(-1) != 1:
        raise ValueError("scores need a unit stride in their last dimension")
    return _strides(t)


def _first(t, R, device):
    return None if t is None else _ints(t, "first", (R,), device)


def prepare_weights(q, k, tables, lengths, q_start, lse, scores, mask, scale=None, first=None, max_fresh=None):
    """A PagedLaunch that adds to every cached key's score the attention weight it has from the step's
    tokens: over the tokens of its request and the query heads that read its head, the sum of exp(scale
    q . k - lse) where the key is live.

    q, k, tables, lengths, q_start, mask, scale, max_fresh: as in prepare_attention.  lse: float32 [tokens, Hq], of
    that attention (a row with -inf has no weight).  scores: float32 [pages, Hkv, page_size], as the
    cache's rows, updated in place: the keys of this step's tokens start from 0, whatever their score
    was.  first: int32 [R], places whose scores stay as they are are those below it (default: none); pages
    that requests share lie below it.  The result is scores."""
    pages, Hkv, P, D = _cache(k, k)
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
    first = _first(first, R, dev)
    dm = _paged_mask(mask)
    scale = _scale(scale, D)
    max_fresh = T if max_fresh is None else int(max_fresh)
    if max_fresh < 0:
        raise ValueError(f"max_fresh={max_fresh} < 0")
    _lib.require_device(lse)
    if lse.dtype != torch.float32 or lse.shape != (T, Hq) or lse.device != dev:
        raise ValueError(f"lse must be float32 [{T}, {Hq}] on {dev}")
    a = _lib.PaWeightsArgs()
    ptr = _lib.address
    a.q, (a.q_st, a.q_sh) = ptr(q), _strides(q)
    a.k, (a.c_sp, a.c_sh, a.c_sn) = ptr(k), _strides(k)
    a.n_pages, a.page_size = pages, P
    a.tables, a.pitch, a.cols = ptr(tables), pitch, tables.shape[1]
    a.lengths, a.q_start, a.first, a.R = ptr(lengths), ptr(q_start), ptr(first), R
    a.T, a.max_fresh, a.Hq, a.Hkv, a.D, a.dtype, a.scale = T, min(max_fresh, T), Hq, Hkv, D, _lib.dtype_code(q), scale
    a.mask = dm.struct()
    a.lse, a.lse_st, a.lse_sh = ptr(lse), lse.stride(0), lse.stride(1)
    a.scores, (a.s_sp, a.s_sh) = ptr(scores), _scores(scores, (pages, Hkv, P), dev)
    ws, zero = _workspace("pa_weights_workspace", a, dev)
    return PagedLaunch("pa_paged_weights", (ctypes.byref(a),), [a, q, k, tables, lengths, q_start, lse, scores, first, dm, ws], k,
                       scores, zero=zero)


def weights(q, k, tables, lengths, q_start, lse, scores, mask, scale=None, first=None, max_fresh=None):
    """Attention weights added to scores: see prepare_weights."""
    return prepare_weights(q, k, tables, lengths, q_start, lse, scores, mask, scale, first, max_fresh)()


def _layered(t, dims, name):
    """(layers, stride of the layer) of a tensor of ``dims`` dimensions or, before them, layers."""
    _lib.require_device(t)
    if t.dim() not in (dims, dims + 1):
        raise ValueError(f"{name} must have {dims} dimensions, or layers before them, got {list(t.shape)}")
    return (1, 0) if t.dim() == dims else (t.shape[0], t.stride(0) if t.shape[0] > 1 else 0)


def prepare_choose(scores, tables, lengths, keep, recent, limit=None, first=None, out=None, missing=None, missing_bits=1):
    """A PagedLaunch that says which cached keys stay; its result is a Choice.

    scores: float32 [pages, heads, page_size], or [layers, ...]: every layer, request and head chooses by
    its own.  tables int32 [R, columns], lengths int32 [R].  first: int32 [R], the tokens in front that
    always stay (sinks, a shared prefix; default none).  A request of more than ``limit`` (default
    keep) tokens behind those keeps ``keep`` of them: the ``recent`` newest, and of the others those with
    the largest scores (of equal ones those in front; NaN is above every number; a key without a page is
    below all).  out: a Choice to write into; its lengths are not the given ones.  missing: int32 [1]; given, a
    request past the limit that lacks a page from first on keeps all its keys, which then have no place to
    go to, and missing gets missing_bits."""
    layers, s_sl = _layered(scores, 3, "scores")
    pages, Hkv, P = scores.shape[-3:]
    _page_size(P)
    dev = scores.device
    s_sp, s_sh = _scores(scores, scores.shape, dev)[-2:]
    R = lengths.shape[0] if lengths.dim() == 1 else -1
    _ints(lengths, "lengths", (R,) if R >= 0 else (0,), dev)
    pitch = _tables(tables, R, P, dev)
    first = _first(first, R, dev)
    keep, recent = int(keep), int(recent)
    limit = keep if limit is None else int(limit)
    if not 0 <= recent <= keep <= limit <= MAX_POSITION or keep < 1:
        raise ValueError(f"recent={recent}, keep={keep}, limit={limit}: 0 <= recent <= keep <= limit <= {MAX_POSITION}, keep >= 1")
    shape = (R, Hkv, keep) if scores.dim() == 3 else (layers, R, Hkv, keep)
    if out is None:
        out = Choice(torch.empty(shape, dtype=torch.int32, device=dev), torch.empty(R, dtype=torch.int32, device=dev))
    else:
        out = Choice(*out)
        if not _ints(out.kept, "out.kept", shape, dev).is_contiguous():
            raise ValueError("out.kept must be contiguous")
        _ints(out.lengths, "out.lengths", (R,), dev)
    if missing is not None:
        _ints(missing, "missing", (1,), dev)
    held, kept = scores, out.kept
    if not layers:   # (one layer and head stand for none: the lengths do not depend on them)
        layers, Hkv, s_sp, s_sh = 1, 1, 0, 0
        held, kept = torch.zeros(P, device=dev), torch.empty(R, keep, dtype=torch.int32, device=dev)
    a = _lib.PaChooseArgs()
    ptr = _lib.address
    a.scores, a.s_sl, a.s_sp, a.s_sh = ptr(held), s_sl, s_sp, s_sh
    a.n_pages, a.page_size, a.tables, a.pitch, a.cols = pages, P, ptr(tables), pitch, tables.shape[1]
    a.lengths, a.first, a.layers, a.R, a.Hkv = ptr(lengths), ptr(first), layers, R, Hkv
    a.keep, a.recent, a.limit, a.kept, a.after = keep, recent, limit, ptr(kept), ptr(out.lengths)
    a.missing, a.missing_bits = ptr(missing), int(missing_bits)
    return PagedLaunch("pa_choose_keys", (ctypes.byref(a),), [a, held, kept, tables, lengths, first, missing, out], scores, out)


def choose(scores, tables, lengths, keep, recent, limit=None, first=None, out=None, missing=None, missing_bits=1):
    """Which cached keys stay: see prepare_choose."""
    return prepare_choose(scores, tables, lengths, keep, recent, limit, first, out, missing, missing_bits)()


def prepare_evict(kept, k, v, scores, tables, lengths, first=None):
    """A PagedLaunch that moves the rows of the keys that stay to the front, in place: in every layer and
    head, row kept[.., r, h, j] of request r goes to place first[r] + j.

    kept: int32 [R, heads, keep], or [layers, ...], as choose gives it (entries below their own place, as
    -1, move nothing).  k, v [pages, heads, page_size, D] and scores [pages, heads, page_size] (or None), or
    [layers, ...].  tables, lengths (before the move), first: as choose was given them.  The result is (k,
    v, scores)."""
    layers, c_sl = _layered(k, 4, "k")
    _lib.require_device(v)
    lead = k.shape[:-4]
    if v.shape != k.shape or _strides(v) != _strides(k):
        raise ValueError("k and v must share shape and strides")
    pages, Hkv, P, D = _cache(*((k, v) if not lead else (k[0], v[0]) if layers else (k.new_empty(k.shape[1:]),) * 2))
    dev = k.device
    R = lengths.shape[0] if lengths.dim() == 1 else -1
    _ints(lengths, "lengths", (R,) if R >= 0 else (0,), dev)
    pitch = _tables(tables, R, P, dev)
    first = _first(first, R, dev)
    keep = kept.shape[-1] if kept.dim() else 0
    if not _ints(kept, "kept", (*lead, R, Hkv, keep), dev).is_contiguous():
        raise ValueError("kept must be contiguous")
    a = _lib.PaEvictArgs()
    ptr = _lib.address
    if scores is not None:
        a.scores, (a.s_sp, a.s_sh) = ptr(scores), _scores(scores, (*lead, pages, Hkv, P), dev)[-2:]
        a.s_sl = scores.stride(0) if lead and layers > 1 else 0
    a.kept, a.layers, a.R, a.Hkv, a.keep = ptr(kept), layers, R, Hkv, keep
    a.k, a.v, a.c_sl = ptr(k), ptr(v), c_sl
    a.c_sp, a.c_sh, a.c_sn = _strides(k)[-3:]
    a.n_pages, a.page_size, a.tables, a.pitch, a.cols = pages, P, ptr(tables), pitch, tables.shape[1]
    a.lengths, a.first, a.D, a.dtype = ptr(lengths), ptr(first), D, _lib.dtype_code(k)
    return PagedLaunch("pa_evict_rows", (ctypes.byref(a),), [a, kept, k, v, scores, tables, lengths, first], k, (k, v, scores))


def evict(kept, k, v, scores, tables, lengths, first=None):
    """The rows that stay moved to the front: see prepare_evict."""
    return prepare_evict(kept, k, v, scores, tables, lengths, first)()


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
    rows then start anew).

    ``share`` gives requests the first tokens of another one, whose pages they then read with it.  With
    ``weigh``, scores [layers, pages, heads, page_size] are held too: ``cache.weigh(q, lse, mask, step, layer)``
    after a layer's attend adds to them the attention that its keys have received, and ``evict`` gives
    up the keys that had least, between steps.

    All state is in tensors on the device that stay where they are, so a
    whole step with counts on the device can be captured in a graph, and every replay is a step;
    only ``check`` waits for the device."""

    def __init__(self, requests, max_length, pages, heads, D, dtype=torch.bfloat16, page_size=64, layers=1, device=None,
                 weigh=False):
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
        self.holders = torch.full((requests,), -1, **i32)   # the request whose prefix each shares (itself: its own is shared)
        self.shared = torch.zeros(requests, **i32)          # tokens of that
        self.scores = torch.zeros(self.k.shape[:-1], dtype=torch.float32, device=dev) if weigh else None
        self._shares = False                   # whether requests may share prefixes
        self._trims = False                    # whether pages in front may be missing
        self._last = (None, None, None)        # the newest step, its most new tokens of a request, its Sharing

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
        which = sharing(self.lengths, step.q_start, self.holders, self.shared, self.page_size, tokens) if self._shares else None
        self._last = (step, most, which)
        return step

    def append(self, k_new, v_new, step, layer=0):
        """k_new, v_new [tokens, heads, D] of a step into a layer's pages."""
        append(k_new, v_new, step.slots, self.k[layer], self.v[layer])

    def attend(self, q, mask, step, layer=0, scale=None, max_fresh=None, out=None, lse=None):
        """o [tokens, Hq, D] of a step's tokens against a layer's pages (see prepare_attention; of the
        newest step max_fresh is known where its counts were a list, and shared prefixes are read once)."""
        newest = step is self._last[0]
        if max_fresh is None and newest:
            max_fresh = self._last[1]
        if newest and self._last[2] is not None:
            return shared_attention(q, self.k[layer], self.v[layer], self.tables, step.lengths, step.q_start, self._last[2],
                                    mask, scale, max_fresh, out, lse)
        return attention(q, self.k[layer], self.v[layer], self.tables, step.lengths, step.q_start, mask, scale, max_fresh,
                         out, lse)

    def share(self, holder, members, tokens):
        """Requests ``members`` (a list; without tokens so far) begin with the first ``tokens`` tokens of
        request ``holder``, whole pages that they read and do not copy.  The holder may go on; it keeps
        these pages, neither weighed nor evicted, until it finishes, which it can once the members have.  Members of
        one holder are read together as far as the one that shares least.  Where that cannot be (the holder has fewer tokens, or
        has given some of their pages back, or begins with fewer of another's itself; a member is not empty)
        nothing happens, and ``check`` says so.  Not to be captured; steps captured before the first call read
        a shared prefix as often as there are requests."""
        members = [int(m) for m in members]
        holder, tokens = int(holder), int(tokens)
        if not all(0 <= m < self.requests for m in members + [holder]) or holder in members:
            raise ValueError(f"members {members} and holder {holder}: different ones of {self.requests} requests")
        if not 0 < tokens <= self.max_length or tokens % self.page_size:
            raise ValueError(f"tokens={tokens}: whole pages of {self.page_size}, up to {self.max_length}")
        if not members:
            return
        at = _on_device(members + [holder], torch.int64, self.device)
        n = tokens // self.page_size
        with torch.cuda.device(self.device):
            m, h = at[:-1], at[-1:]
            of = self.holders[h]
            second = (of >= 0) & (of != h)       # the holder shares another's prefix itself
            root = torch.where(second, of, h)    # .. which is then theirs too
            ok = ((self.lengths[h] >= tokens) & (~second | (self.shared[h] >= tokens)) & (self.tables[root, :n] >= 0).all()
                  & (self.lengths[m] == 0) & (self.holders[m] < 0))
            i32 = lambda x: x.to(torch.int32)  # noqa: E731
            self.tables[m, :n] = torch.where(ok[:, None], self.tables[root, :n], self.tables[m, :n])
            for state, new in ((self.lengths, torch.full_like(m, tokens)), (self.shared, torch.full_like(m, tokens)),
                               (self.holders, root.expand(len(members)))):
                state[m] = torch.where(ok, i32(new), state[m])
            some = ok.any()
            self.holders[root] = torch.where(some, i32(root), self.holders[root])
            self.shared[root] = torch.where(some, self.shared[root].clamp(min=tokens), self.shared[root])
            self.failed |= i32((~ok).any()) * SHARED
        self._shares = True

    def weigh(self, q, lse, mask, step, layer=0, scale=None):
        """Adds the attention that a step's tokens have paid to a layer's keys to their scores (see
        prepare_weights; lse: what attend wrote).  Called for every step: a step's own keys start from 0 there.  A
        shared prefix is not weighed."""
        if self.scores is None:
            raise RuntimeError("the cache holds no scores: make it with weigh=True")
        most = self._last[1] if step is self._last[0] else None
        weights(q, self.k[layer], self.tables, step.lengths, step.q_start, lse, self.scores[layer], mask, scale, self.shared, most)

    def evict(self, keep, recent, limit=None, sinks=0):
        """Every request of more than ``limit`` (default keep) tokens behind its first ``sinks`` ones (and
        those that it shares) keeps ``keep`` of them, in each layer and head the ``recent`` newest and those
        with the largest scores, moved together in their order; pages that this leaves go back.  From then
        on a token's position is its place among those kept: a mask that counts distances counts them
        there.  Not in a cache that is trimmed: there may be no page where they go.  (A replay of an eviction
        that was captured before leaves requests with such places as they are, and ``check`` says so.)"""
        if self.scores is None:
            raise RuntimeError("the cache holds no scores: make it with weigh=True")
        if self._trims:
            raise RuntimeError("the cache has been trimmed: its requests have no pages in front to move keys to")
        if sinks < 0:
            raise ValueError(f"sinks={sinks} < 0")
        P = self.page_size
        with torch.cuda.device(self.device):
            first = self.shared.clamp(min=min(int(sinks), self.max_length))
            choice = choose(self.scores, self.tables, self.lengths, keep, recent, limit, first, None, self.failed, TRIMMED)
            evict(choice.kept, self.k, self.v, self.scores, self.tables, self.lengths, first)
            pages = lambda n: ((n + (P - 1)) // P).to(torch.int32)  # noqa: E731
            self._release(pages(choice.lengths), pages(self.lengths))
            self.lengths.copy_(choice.lengths)

    def _release(self, first, last):
        status = torch.empty(1, dtype=torch.int32, device=self.device)
        release(first, last, self.tables, self.free_list, self.free_count, (self.free_count, status))
        with torch.cuda.device(self.device):
            self.failed |= status * LIST_FULL

    def finish(self, done):
        """Gives back the pages of the requests where done (bool [requests], on the device, or a list,
        which a graph's capture does not take) is true and sets their lengths to 0.  One whose tokens
        others share that are not done stays as it is, and ``check`` says so."""
        if not (isinstance(done, torch.Tensor) and done.is_cuda):
            done = _on_device(done, torch.bool, self.device)
        done = done.to(device=self.device, dtype=torch.bool)
        if done.shape != (self.requests,):
            raise ValueError(f"done must be [{self.requests}], got {list(done.shape)}")
        done = done.contiguous()
        # (a step captured before the first prefix is shared is right after it too: the state is on the device)
        first, last, busy = (torch.empty(self.requests, dtype=torch.int32, device=self.device) for _ in range(3))
        a = _lib.PaFinishArgs()
        ptr = _lib.address
        a.done, a.holders, a.shared, a.lengths = ptr(done), ptr(self.holders), ptr(self.shared), ptr(self.lengths)
        a.R, a.page_size = self.requests, self.page_size
        a.tables, a.pitch, a.cols = ptr(self.tables), self.tables.stride(0), self.tables.shape[1]
        a.refused, a.refused_bits, a.first, a.last, a.workspace = ptr(self.failed), SHARED, ptr(first), ptr(last), ptr(busy)
        PagedLaunch("pa_page_finish", (ctypes.byref(a),), [a, done, first, last, busy], self.lengths, None)()
        self._release(first, last)

    def trim(self, window, sinks=0):
        """Gives back the pages that neither the next token's window nor the first ``sinks`` tokens
        need: with a SinksWindow(sinks, window) mask no later token sees them."""
        if window < 1 or sinks < 0:
            raise ValueError(f"window={window} must be at least 1 and sinks={sinks} at least 0")
        self._trims = True
        P = self.page_size
        with torch.cuda.device(self.device):
            last = (self.lengths - int(min(window, MAX_POSITION) - 1)).clamp_(min=0) // P
            # (nor what requests share)
            first = (self.shared // P).clamp_(min=min(-(-int(sinks) // P), self.tables.shape[1]))
            self._release(first, last)

    def check(self):
        """Waits for the device and raises if a step so far did not fit."""
        bits = int(self.failed.item())
        if bits:
            why = [w for b, w in ((SHORT_OF_PAGES, "too few free pages"), (TOO_LONG, f"a request past {self.max_length} tokens"),
                                  (TOO_MANY_TOKENS, "more new tokens than rows"),
                                  (LIST_FULL, "more pages given back than there are"),
                                  (SHARED, "a prefix that could not be shared, or was finished before those that share it"),
                                  (TRIMMED, "a request without the pages in front was to be evicted"))
                   if bits & b]
            raise RuntimeError("a step did not fit: " + ", ".join(why))
