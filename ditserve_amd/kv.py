"""Paged key-value caches: what a generating model keeps of its sequences.

A `PagedCache` holds keys and values in pages; a table names each sequence's pages, and
`lengths` says how many of its slots are filled.  Tables and lengths are device tensors, so
a loop of steps runs (and is captured into a graph) without the host:

    cache = kv.PagedCache.empty(pages, kv_heads, head_dim, page=64, device="cuda")
    out = ops.flash_attn_causal(q, k, v, seg, seg, heads, kv_heads, head_dim)    # the prompts
    lengths = kv.append(cache, k, v, table, lengths, seg)
    ...                                                                          # a step
    lengths = kv.append(cache, k, v, table, lengths)
    out = kv.decode_attn(q, cache, table, lengths, heads, weights="add")
    ...                                                                          # when it is full
    lengths = kv.evict(cache, table, lengths, new_table, keep=4096, recent=512)

Checks, streams and errors are those of ditserve_amd.ops.  A length outside what a table
holds is clamped to it, and a page that the cache lacks is neither read nor written (its
slots count as absent); both are reported by a later call or by check_tables(), as an
invalid cu_seqlens table is.  The pages a call writes must belong to one sequence; pages
that are only read may be shared.  The cache serves single tokens: no call attends several
new tokens over it, so the next part of a prompt (ops.flash_attn_causal) needs the keys and
values of its earlier parts as packed rows as well.  The reference has no counterpart: its models attend over
whole videos.
"""
import ctypes
import math

import torch

from . import _lib, ops
from .mx import _apart
from .ops import _call, _check, _extent, _meet, _one_device, _ptr, _row_view

PAGES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)
_BF16 = torch.bfloat16


class PageStatus(ops.TableStatus):
    """TableStatus of the page tables and lengths that kv's calls were given."""

    def __init__(self, device):
        super().__init__(device)
        self.address = self.host.data_ptr()
        self._word = ctypes.c_int32.from_address(self.address)

    def poll(self):
        if self._word.value:
            self.host.zero_()
            raise _lib.DitkError("an invalid page table reached the cache kernels (a length outside the table or "
                                 "max_len, or a page that the cache lacks); it was clamped into bounds, so those "
                                 "outputs are not what was meant")


_STATUS = {}


def _status(device):
    st = _STATUS.get(device)
    if st is None:  # (one word for good, also if two threads come here at once)
        st = _STATUS.setdefault(device, PageStatus(device))
    return st


def check_tables(device=None):
    """Wait for `device` (default: the current one) and raise DitkError if a page table or
    length given to these calls since the last report was invalid."""
    device = torch.device(device if device is not None else "cuda")
    if device.index is None:
        device = torch.device(device.type, torch.cuda.current_device())
    _status(device).check()


def _span(pages, heads, ps, hs, size):
    """From the first to the last element of a tensor's (page, head) blocks of `size`; 0 if blocks overlap."""
    if pages > 1 and heads > 1 and ps < hs:
        pages, heads, ps, hs = heads, pages, hs, ps
    if heads > 1:
        if hs < size:
            return 0
        size += (heads - 1) * hs
    if pages > 1:
        if ps < size:
            return 0
        size += (pages - 1) * ps
    return size


def _nearest(delta, stride, count):
    """delta and a multiple of stride, less than `count` of them either way, where that is nearest to 0 on both sides."""
    if count == 1:
        return (delta,)
    i = -delta // stride
    return [delta + j * stride for j in (i, i + 1) if abs(j) < count]


def _meet_blocks(delta, pages, heads, ps, hs, size):
    """Whether two tensors of the same strides, of which _span is not 0, the second `delta` elements behind the first,
    share an element."""
    if pages > 1 and heads > 1 and ps < hs:
        pages, heads, ps, hs = heads, pages, hs, ps
    return any(abs(y) < size for x in _nearest(delta, ps, pages) for y in _nearest(x, hs, heads))


def _blocks_meet(delta, a, b):
    """Whether two tensors' blocks (pages, heads, page stride, head stride, size), of which _span is not 0, the second's
    `delta` behind the first's, share an element.  Exact where their strides are the same, or the larger ones are (what
    lies in between counts as a tensor's own then); else whether their spans meet."""
    levels, sizes = [], []
    for pages, heads, ps, hs, size in (a, b):
        levels.append(sorted(((st, n) for n, st in ((pages, ps), (heads, hs)) if n > 1), reverse=True))
        sizes.append(size)
    same = 0
    while same < len(levels[0]) and levels[0][same] == levels[1][same]:
        same += 1
    sizes = [size + sum((n - 1) * st for st, n in own[same:]) for size, own in zip(sizes, levels)]
    starts = [delta]
    for st, n in levels[0][:same]:
        starts = [y for x in starts for y in _nearest(x, st, n)]
    return any(-sizes[1] < y < sizes[0] for y in starts)


class PagedCache:
    """Keys and values in pages.

    k, v     [pages, kv_heads, page, head_dim] bf16; a page of 16, 32, 64, 128 or 256 slots,
             head_dim 64 or 128.  A (page, head)'s slots are contiguous; the first two strides
             are free (k and v may be halves of one buffer)
    weights  [pages, kv_heads, page] fp32, the attention weight each slot has gathered
             (optional; decode_attn writes it, evict reads it); none of them in a key or value"""

    __slots__ = ("_k", "_v", "_w", "_dims", "_strides", "_bytes")

    def __init__(self, k, v, weights=None):
        strides, ends = [], []
        for t, name in ((k, "k"), (v, "v")):
            if t.__class__ is not torch.Tensor or t.dtype is not _BF16 or not t.is_cuda or t.dim() != 4:
                _check(t, name, _BF16, 4)
            pages, heads, page, d = dims = tuple(t.shape)
            ps, hs, ss, unit = t.stride()
            if page not in PAGES or d not in HEAD_DIMS:
                raise ValueError(f"{name} must be [pages, kv_heads, {PAGES}, {HEAD_DIMS}], got {dims}")
            if pages == 0 or heads == 0:
                raise ValueError(f"{name} has no pages or no heads: {dims}")
            first, span = t.data_ptr(), _span(pages, heads, ps, hs, page * d)
            if unit != 1 or ss != d or (ps | hs) & 7 or first & 15 or not span:
                raise ValueError(f"{name}'s slots must be contiguous within a (page, head), which must not overlap, and "
                                 f"16-byte aligned, got strides {t.stride()}")
            strides += (ps, hs)
            ends.append((first, first + 2 * span))
        if v.shape != k.shape:
            raise ValueError(f"v must be {tuple(k.shape)}, got {tuple(v.shape)}")
        device = k.device
        if v.device != device or (weights is not None and weights.device != device):
            _one_device(device, ("v", v), ("weights", weights))
        if _meet(*ends) and (strides[:2] != strides[2:] or _meet_blocks((ends[1][0] - ends[0][0]) // 2, *dims[:2], ps, hs,
                                                                        page * d)):
            raise ValueError("k and v overlap")
        if weights is not None:
            _check(weights, "weights", torch.float32, 3)
            ps, hs, unit = weights.stride()
            span = _span(pages, heads, ps, hs, page)
            if tuple(weights.shape) != dims[:3] or unit != 1 or not span:
                raise ValueError(f"weights must be {dims[:3]} with unit slot stride, got {tuple(weights.shape)}, strides "
                                 f"{weights.stride()}")
            first = weights.data_ptr()
            for end, st in zip(ends, (strides[:2], strides[2:])):
                if _meet(end, (first, first + 4 * span)) and _blocks_meet(
                        first - end[0], (*dims[:2], 2 * st[0], 2 * st[1], 2 * page * d),
                        (*dims[:2], 4 * ps, 4 * hs, 4 * page)):
                    raise ValueError("weights overlap k or v")
            strides += (ps, hs)
        else:
            span, strides = 0, strides + [0, 0]
        self._bytes = ends[0][1] - ends[0][0], ends[1][1] - ends[1][0], 4 * span
        self._k, self._v, self._w, self._dims, self._strides = k, v, weights, dims, strides
        _status(device)

    @classmethod
    def empty(cls, pages, kv_heads, head_dim, page=64, device="cuda", weights=True):
        """An uninitialised cache (append clears the weights of the slots it fills)."""
        k, v = torch.empty((2, pages, kv_heads, page, head_dim), dtype=_BF16, device=device).unbind(0)
        w = torch.empty((pages, kv_heads, page), dtype=torch.float32, device=device) if weights else None
        return cls(k, v, w)

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    weights = property(lambda self: self._w)
    pages = property(lambda self: self._dims[0])
    kv_heads = property(lambda self: self._dims[1])
    page = property(lambda self: self._dims[2])
    head_dim = property(lambda self: self._dims[3])
    device = property(lambda self: self._k.device)

    def record_stream(self, stream):
        """Mark the cache as in use by `stream` (for steps on a side stream)."""
        for t in (self._k, self._v, self._w):
            if t is not None:
                t.record_stream(stream)

    def _args(self, weights=True):
        """Addresses and strides of keys, values and (unless not wanted) weights."""
        s = self._strides
        w = (self._w.data_ptr(), s[4], s[5]) if weights and self._w is not None else (None, 0, 0)
        return (self._k.data_ptr(), s[0], s[1], self._v.data_ptr(), s[2], s[3], *w)

    def _spans(self):
        """First and last byte of keys, values and weights."""
        k, v, w = self._k.data_ptr(), self._v.data_ptr(), self._w.data_ptr() if self._w is not None else 0
        a, b, c = self._bytes
        return (k, k + a), (v, v + b), (w or k, (w or k) + c)


def _cache_check(cache):
    if not isinstance(cache, PagedCache):
        raise ValueError(f"cache must be a PagedCache, got {type(cache).__name__}")


def _table(t, name, batch, device):
    """(address, row stride, pages of a row) of a page table [batch, pages]."""
    if t.__class__ is not torch.Tensor or t.dtype is not torch.int32 or t.dim() != 2 or t.device != device:
        _check(t, name, torch.int32, 2)
        _one_device(device, (name, t))
    rows, width = t.shape
    st, unit = t.stride()
    if rows != batch or (width > 1 and unit != 1) or (rows > 1 and st < width):
        raise ValueError(f"{name} must be [{batch}, pages] with unit column stride, got {tuple(t.shape)}, strides "
                         f"{t.stride()}")
    return t.data_ptr(), max(st, width), width


def _lengths(t, device):
    if t.__class__ is not torch.Tensor or t.dtype is not torch.int32 or t.dim() != 1 or t.device != device:
        _check(t, "lengths", torch.int32, 1)
        _one_device(device, ("lengths", t))
    if t.shape[0] > 1 and t.stride(0) != 1:
        raise ValueError("lengths must be contiguous")
    return t.shape[0]


def _outside(fn, cache, *spans):
    """Refuse operands (first and last byte) that lie between a cache's first and last byte."""
    own = cache._spans()
    (a, b), (c, d), (e, f) = own
    low, high = min(a, c, e), max(b, d, f)
    for span in spans:
        if span[0] < high and low < span[1] and any(_meet(span, x) for x in own):
            raise ValueError(f"{fn}: an operand lies in the cache")


def append(cache, k, v, table, lengths, segments=None):
    """Writes new keys and values into the slots behind each sequence's last.

    k, v [T, kv_heads * head_dim] bf16 row views: the rows of segment b (ops.Segments; without
    segments one row a sequence) go to slots lengths[b], lengths[b] + 1, ... of sequence b,
    whose pages must be in the table already.  Returns the new lengths, a new int32 tensor;
    `lengths` itself stays.  The slots' weights, if the cache has any, become 0."""
    _cache_check(cache)
    device, (pages, hk, page, d) = cache._k.device, cache._dims
    wide = hk * d
    batch = _lengths(lengths, device)
    T, ldk = _row_view(k, "k", wide, device)
    rows, ldv = _row_view(v, "v", wide, device)
    if rows != T:
        raise ValueError(f"k and v must have the same rows, got {T} and {rows}")
    tp, ldt, width = _table(table, "table", batch, device)
    kp, vp, lp, cu = k.data_ptr(), v.data_ptr(), lengths.data_ptr(), None
    spans = [(kp, kp + 2 * ((T - 1) * ldk + wide) * (T > 0)), (vp, vp + 2 * ((T - 1) * ldv + wide) * (T > 0)),
             (tp, tp + 4 * (batch * ldt - ldt + width)), (lp, lp + 4 * batch)]
    if segments is not None:
        if segments.nseg != batch or segments.total != T:
            raise ValueError(f"segments are {segments.nseg} of {segments.total} rows, lengths {batch} and k {T}")
        if segments.dev.device != device:
            _one_device(device, ("segments", segments.dev))
        cu = segments.dev.data_ptr()
        spans.append((cu, cu + 4 * batch + 4))
    elif T != batch:
        raise ValueError(f"k must have one row for each of the {batch} sequences, got {T} (or pass segments)")
    status = _status(device)
    status.poll()
    new = torch.empty(batch, dtype=torch.int32, device=device)
    _outside("append", cache, *spans)
    _call(device, "ditk_kv_append", kp, ldk, vp, ldv, *cache._args(), pages, page, tp, ldt, width, lp, new.data_ptr(), cu,
          batch, T, hk, d, status.address)
    return new


def decode_attn(q, cache, table, lengths, heads, softmax_scale=None, max_len=None, weights=None, return_lse=False,
                out=None):
    """Attention of one new token of each sequence over the slots its lengths say.

    q [batch, heads * head_dim] bf16 (a row view), heads a multiple of the cache's: query
    head h reads key head h // (heads / kv_heads).  max_len: the longest length there can be
    (default: what the table holds); it sizes the launch.  weights: "set" writes into the
    cache's weights what each slot gets from these queries (the probabilities, summed over
    the query heads of its key head), "add" adds it.  Returns out [batch, heads * head_dim]
    bf16, and with return_lse lse [batch, heads] fp32 (natural log).  A sequence without
    slots gives zeros and -inf.  A sequence's result does not depend on the others.

    The workspace goes by max_len, not by the lengths: beyond 512 slots (head_dim + 2) * 4 bytes
    for each query head and chunk (64 slots, 512 of long caches), and with weights 4 bytes for
    each query head and slot: 64 sequences, 32 heads of 128, max_len 131072 take 0.27 GB, with
    weights 1.35."""
    _cache_check(cache)
    device, (pages, hk, page, d) = cache._k.device, cache._dims
    batch = _lengths(lengths, device)
    heads = int(heads)
    if heads <= 0 or heads % hk:
        raise ValueError(f"heads must be a multiple of the cache's {hk}, got {heads}")
    rows, ldq = _row_view(q, "q", heads * d, device)
    if rows != batch:
        raise ValueError(f"q must have one row for each of the {batch} sequences, got {rows}")
    tp, ldt, width = _table(table, "table", batch, device)
    if weights not in (None, "set", "add"):
        raise ValueError(f"weights must be None, 'set' or 'add', got {weights!r}")
    if weights is not None and cache._w is None:
        raise ValueError("the cache has no weights")
    most = width * page
    if max_len is not None:
        if max_len < 0:
            raise ValueError(f"max_len must not be negative, got {max_len}")
        most = min(most, int(max_len))
    scale = 1.0 / math.sqrt(d) if softmax_scale is None else float(softmax_scale)
    if not 1e-30 <= scale <= 1e30:  # (scores are scaled in fp32)
        raise ValueError(f"softmax_scale must be in 1e-30..1e30, got {scale}")
    if out is None:
        out, ldo = torch.empty((batch, heads * d), dtype=_BF16, device=device), heads * d
    else:
        rows, ldo = _row_view(out, "out", heads * d, device)
        if rows != batch:
            raise ValueError(f"out must have one row for each of the {batch} sequences, got {rows}")
        _outside("decode_attn", cache, _extent(out))
        _apart("decode_attn", (out,), (q, table, lengths))
    if weights is not None:
        _outside("decode_attn", cache, _extent(q), _extent(table), _extent(lengths))
    status = _status(device)
    status.poll()
    lse = torch.empty((batch, heads), dtype=torch.float32, device=device) if return_lse else None
    # (up to 512 slots without weights take one launch and no workspace)
    size = _lib.load().ditk_kv_attn_workspace(batch, heads, d, most, weights is not None) if weights or most > 512 else 0
    space = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _call(device, "ditk_kv_attn", q.data_ptr(), ldq, *cache._args(weights is not None), int(weights == "add"), pages, page,
          tp, ldt, width, lengths.data_ptr(), most, out.data_ptr(), ldo, _ptr(lse), _ptr(space), size, batch, heads, hk, d,
          scale, status.address)
    return (out, lse) if return_lse else out


def evict(cache, table, lengths, out_table, keep, recent=0, max_len=None):
    """Cuts each sequence to `keep` slots by the attention weight they gathered.

    Of each (sequence, key head) the last `recent` slots stay and of the others those with the
    largest weights, `keep` in all (ties: the lowest slot; a NaN weight counts as -inf, the
    lowest).  A sequence of at most `keep` slots keeps them all.  What stays is copied, with
    its weights, in its order into the first slots of the pages of `out_table`, which must be
    other pages than the table's; those may be freed, or go on being read by who shares them.
    (Slots of a page that the cache lacks have the lowest weight; one that has to stay becomes
    zeros, with weight 0, besides being reported.)
    max_len: the longest length there can be (default: what the table holds).  Returns the new
    lengths, a new int32 tensor."""
    _cache_check(cache)
    device, (pages, hk, page, d) = cache._k.device, cache._dims
    if cache._w is None:
        raise ValueError("the cache has no weights")
    batch = _lengths(lengths, device)
    keep, recent = int(keep), int(recent)
    if keep <= 0 or not 0 <= recent <= keep:
        raise ValueError(f"keep must be positive and recent at most keep, got {keep} and {recent}")
    tp, ldt, width = _table(table, "table", batch, device)
    op, ldo, out_width = _table(out_table, "out_table", batch, device)
    _apart("evict", (out_table,), (table,))
    most = width * page
    if max_len is not None:
        if max_len < 0:
            raise ValueError(f"max_len must not be negative, got {max_len}")
        most = min(most, int(max_len))
    if out_width * page < min(keep, most):
        raise ValueError(f"out_table holds {out_width * page} slots, {min(keep, most)} stay")
    _outside("evict", cache, _extent(table), _extent(out_table), _extent(lengths))
    keep = max(min(keep, most), 1)
    recent = min(recent, keep)
    status = _status(device)
    status.poll()
    new = torch.empty(batch, dtype=torch.int32, device=device)
    size = _lib.load().ditk_kv_evict_workspace(batch, hk, most, keep)
    space = torch.empty(size, dtype=torch.uint8, device=device)
    _call(device, "ditk_kv_evict", *cache._args(), pages, page, tp, ldt, width, _ptr(lengths), most, op, ldo, out_width,
          _ptr(new), keep, recent, _ptr(space), size, batch, hk, d, status.address)
    return new
