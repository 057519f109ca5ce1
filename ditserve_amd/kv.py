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
that are only read may be shared.  The reference has no counterpart: its models attend over
whole videos.
"""
import math

import torch

from . import _lib, ops
from .mx import _apart
from .ops import _call, _check, _one_device, _ptr, _rows

PAGES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)
_BF16 = torch.bfloat16


class PageStatus(ops.TableStatus):
    """TableStatus of the page tables and lengths that kv's calls were given."""

    def poll(self):
        if self.host.item() != 0:
            self.host.zero_()
            raise _lib.DitkError("an invalid page table reached the cache kernels (a length outside the table or "
                                 "max_len, or a page that the cache lacks); it was clamped into bounds, so those "
                                 "outputs are not what was meant")


_STATUS = {}


def _status(device):
    st = _STATUS.get(device)
    if st is None:
        st = _STATUS[device] = PageStatus(device)
    return st


def check_tables(device=None):
    """Wait for `device` (default: the current one) and raise DitkError if a page table or
    length given to these calls since the last report was invalid."""
    device = torch.device(device if device is not None else "cuda")
    if device.index is None:
        device = torch.device(device.type, torch.cuda.current_device())
    _status(device).check()


class PagedCache:
    """Keys and values in pages.

    k, v     [pages, kv_heads, page, head_dim] bf16; a page of 16, 32, 64, 128 or 256 slots,
             head_dim 64 or 128.  A (page, head)'s slots are contiguous; the first two strides
             are free (k and v may be halves of one buffer)
    weights  [pages, kv_heads, page] fp32, the attention weight each slot has gathered
             (optional; decode_attn writes it, evict reads it)"""

    __slots__ = ("k", "v", "weights")

    def __init__(self, k, v, weights=None):
        for t, name in ((k, "k"), (v, "v")):
            _check(t, name, _BF16, 4)
            pages, heads, page, d = t.shape
            ps, hs, ss, unit = t.stride()
            if page not in PAGES or d not in HEAD_DIMS:
                raise ValueError(f"{name} must be [pages, kv_heads, {PAGES}, {HEAD_DIMS}], got {tuple(t.shape)}")
            if pages == 0 or heads == 0:
                raise ValueError(f"{name} has no pages or no heads: {tuple(t.shape)}")
            if unit != 1 or ss != d or ps % 8 or hs % 8 or t.data_ptr() % 16 or \
                    (pages > 1 and ps < page * d) or (heads > 1 and hs < page * d):
                raise ValueError(f"{name}'s slots must be contiguous within a (page, head) and 16-byte aligned, got "
                                 f"strides {t.stride()}")
        if v.shape != k.shape:
            raise ValueError(f"v must be {tuple(k.shape)}, got {tuple(v.shape)}")
        _one_device(k.device, ("v", v), ("weights", weights))
        if weights is not None:
            _check(weights, "weights", torch.float32, 3)
            ps, hs, unit = weights.stride()
            if weights.shape != k.shape[:3] or unit != 1 or (k.shape[0] > 1 and ps < k.shape[2]) or \
                    (k.shape[1] > 1 and hs < k.shape[2]):
                raise ValueError(f"weights must be {tuple(k.shape[:3])} with unit slot stride, got "
                                 f"{tuple(weights.shape)}, strides {weights.stride()}")
        self.k, self.v, self.weights = k, v, weights
        _status(k.device)

    @classmethod
    def empty(cls, pages, kv_heads, head_dim, page=64, device="cuda", weights=True):
        """An uninitialised cache (append clears the weights of the slots it fills)."""
        k, v = torch.empty((2, pages, kv_heads, page, head_dim), dtype=_BF16, device=device).unbind(0)
        w = torch.empty((pages, kv_heads, page), dtype=torch.float32, device=device) if weights else None
        return cls(k, v, w)

    @property
    def pages(self):
        return self.k.shape[0]

    @property
    def kv_heads(self):
        return self.k.shape[1]

    @property
    def page(self):
        return self.k.shape[2]

    @property
    def head_dim(self):
        return self.k.shape[3]

    @property
    def device(self):
        return self.k.device

    def record_stream(self, stream):
        """Mark the cache as in use by `stream` (for steps on a side stream)."""
        for t in (self.k, self.v, self.weights):
            if t is not None:
                t.record_stream(stream)

    def _kv(self):
        (kp, kh, _, _), (vp, vh, _, _) = self.k.stride(), self.v.stride()
        return self.k.data_ptr(), kp, kh, self.v.data_ptr(), vp, vh

    def _weights(self, used=True):
        if self.weights is None or not used:
            return None, 0, 0
        ps, hs, _ = self.weights.stride()
        return self.weights.data_ptr(), ps, hs


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


def _outside(fn, cache, *tensors):
    """Refuse rows and tables that lie between a cache's first and last byte."""
    spans = []
    for c in (cache.k, cache.v, cache.weights):
        if c is not None:
            (pages, heads, page), (ps, hs) = c.shape[:3], c.stride()[:2]
            first, size = c.data_ptr(), c.element_size()
            spans.append((first, first + ((pages - 1) * ps + (heads - 1) * hs + page * (c.shape[3] if size == 2 else 1)) * size))
    for t in tensors:
        if t is not None:
            first = t.data_ptr()
            rows = t.shape[0]
            last = first + ((rows - 1) * t.stride(0) + (t.shape[1] if t.dim() == 2 else 1)) * t.element_size() if rows else first
            for a, b in spans:
                if first < b and a < last:
                    raise ValueError(f"{fn}: an operand lies in the cache")


def _rows_of(t, name, rows, cols, device):
    if t.__class__ is not torch.Tensor or t.dtype is not _BF16 or t.dim() != 2 or t.device != device:
        _check(t, name, _BF16, 2)
        _one_device(device, (name, t))
    n, wide = t.shape
    if wide != cols or (rows is not None and n != rows):
        raise ValueError(f"{name} must be [{'rows' if rows is None else rows}, {cols}], got {tuple(t.shape)}")
    ld = _rows(t, name)
    if n > 1 and ld < cols:
        raise ValueError(f"{name}'s rows overlap: strides {t.stride()}")
    return ld


def append(cache, k, v, table, lengths, segments=None):
    """Writes new keys and values into the slots behind each sequence's last.

    k, v [T, kv_heads * head_dim] bf16 row views: the rows of segment b (ops.Segments; without
    segments one row a sequence) go to slots lengths[b], lengths[b] + 1, ... of sequence b,
    whose pages must be in the table already.  Returns the new lengths, a new int32 tensor;
    `lengths` itself stays.  The slots' weights, if the cache has any, become 0."""
    _cache_check(cache)
    device, hk, d = cache.k.device, cache.kv_heads, cache.head_dim
    batch = _lengths(lengths, device)
    ldk = _rows_of(k, "k", None, hk * d, device)
    T = k.shape[0]
    ldv = _rows_of(v, "v", T, hk * d, device)
    tp, ldt, width = _table(table, "table", batch, device)
    cu = None
    if segments is not None:
        if segments.nseg != batch or segments.total != T:
            raise ValueError(f"segments are {segments.nseg} of {segments.total} rows, lengths {batch} and k {T}")
        cu = segments.dev
        _one_device(device, ("segments", cu))
    elif T != batch:
        raise ValueError(f"k must have one row for each of the {batch} sequences, got {T} (or pass segments)")
    status = _status(device)
    status.poll()
    new = torch.empty(batch, dtype=torch.int32, device=device)
    _outside("append", cache, k, v, table, lengths, cu)
    _call(device, "ditk_kv_append", _ptr(k), ldk, _ptr(v), ldv, *cache._kv(), *cache._weights(), cache.pages, cache.page,
          tp, ldt, width, _ptr(lengths), _ptr(new), _ptr(cu), batch, T, hk, d, _ptr(status.host))
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
    slots gives zeros and -inf.  A sequence's result does not depend on the others."""
    _cache_check(cache)
    device, hk, d = cache.k.device, cache.kv_heads, cache.head_dim
    batch = _lengths(lengths, device)
    heads = int(heads)
    if heads <= 0 or heads % hk:
        raise ValueError(f"heads must be a multiple of the cache's {hk}, got {heads}")
    ldq = _rows_of(q, "q", batch, heads * d, device)
    tp, ldt, width = _table(table, "table", batch, device)
    if weights not in (None, "set", "add"):
        raise ValueError(f"weights must be None, 'set' or 'add', got {weights!r}")
    if weights is not None and cache.weights is None:
        raise ValueError("the cache has no weights")
    most = width * cache.page
    if max_len is not None:
        if max_len < 0:
            raise ValueError(f"max_len must not be negative, got {max_len}")
        most = min(most, int(max_len))
    scale = 1.0 / math.sqrt(d) if softmax_scale is None else float(softmax_scale)
    if not 0 < scale < math.inf:
        raise ValueError(f"softmax_scale must be positive and finite, got {scale}")
    if out is None:
        out, ldo = torch.empty((batch, heads * d), dtype=_BF16, device=device), heads * d
    else:
        ldo = _rows_of(out, "out", batch, heads * d, device)
        _outside("decode_attn", cache, out)
        _apart("decode_attn", (out,), (q, table, lengths))
    status = _status(device)
    status.poll()
    lse = torch.empty((batch, heads), dtype=torch.float32, device=device) if return_lse else None
    size = _lib.load().ditk_kv_attn_workspace(batch, heads, d, most, weights is not None)
    space = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _call(device, "ditk_kv_attn", _ptr(q), ldq, *cache._kv(), *cache._weights(weights is not None), int(weights == "add"),
          cache.pages, cache.page, tp, ldt, width, _ptr(lengths), most, _ptr(out), ldo, _ptr(lse), _ptr(space), size,
          batch, heads, hk, d, scale, _ptr(status.host))
    return (out, lse) if return_lse else out


def evict(cache, table, lengths, out_table, keep, recent=0, max_len=None):
    """Cuts each sequence to `keep` slots by the attention weight they gathered.

    Of each (sequence, key head) the last `recent` slots stay and of the others those with the
    largest weights, `keep` in all (ties: the lowest slot; a NaN weight counts as -inf, the
    lowest).  A sequence of at most `keep` slots keeps them all.  What stays is copied, with
    its weights, in its order into the first slots of the pages of `out_table`, which must be
    other pages than the table's; those may be freed, or go on being read by who shares them.
    max_len: the longest length there can be (default: what the table holds).  Returns the new
    lengths, a new int32 tensor."""
    _cache_check(cache)
    device, hk, d = cache.k.device, cache.kv_heads, cache.head_dim
    if cache.weights is None:
        raise ValueError("the cache has no weights")
    batch = _lengths(lengths, device)
    keep, recent = int(keep), int(recent)
    if keep <= 0 or not 0 <= recent <= keep:
        raise ValueError(f"keep must be positive and recent at most keep, got {keep} and {recent}")
    tp, ldt, width = _table(table, "table", batch, device)
    op, ldo, out_width = _table(out_table, "out_table", batch, device)
    _apart("evict", (out_table,), (table,))
    most = width * cache.page
    if max_len is not None:
        if max_len < 0:
            raise ValueError(f"max_len must not be negative, got {max_len}")
        most = min(most, int(max_len))
    if out_width * cache.page < min(keep, most):
        raise ValueError(f"out_table holds {out_width * cache.page} slots, {min(keep, most)} stay")
    keep = max(min(keep, most), 1)
    recent = min(recent, keep)
    status = _status(device)
    status.poll()
    new = torch.empty(batch, dtype=torch.int32, device=device)
    size = _lib.load().ditk_kv_evict_workspace(batch, hk, most, keep)
    space = torch.empty(size, dtype=torch.uint8, device=device)
    _call(device, "ditk_kv_evict", *cache._kv(), *cache._weights(), cache.pages, cache.page, tp, ldt, width,
          _ptr(lengths), most, op, ldo, out_width, _ptr(new), keep, recent, _ptr(space), size, batch, hk, d,
          _ptr(status.host))
    return new
