"""Paged caches where tables and lengths are wrong, where pages, heads and weights have strides of their own, and where
sequences are long enough for every size of chunk."""
import math

import pytest
import torch

from tests.kv_reference import DEV, NAN, attend64, check_out, errors32, get, paged

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from ditserve_amd import _lib, kv


def cache_of(lens, hk, d, page, seed, layout="plain", more=()):
    """(cache, table, lengths, table of `more` slots): paged() with weights in wider rows of their own, NaN around them."""
    cache, table, lengths, out_table, _, _ = paged(lens, hk, d, page, seed, layout=layout, more=more)
    wide = torch.full((cache.pages, hk + 1, page + 12), NAN, device=DEV)
    w = wide[:, :hk, 4:4 + page]
    w.copy_(torch.rand(w.shape, generator=torch.Generator().manual_seed(seed)).to(DEV))
    return kv.PagedCache(cache.k, cache.v, w), table, lengths, out_table, wide


def evicted(cache, table, lens, out_table, keep, recent):
    """(keys, values, weights, new lengths) by definition: slots of pages that the cache lacks have the lowest weight and
    are zeros where they stay; what would go to such a page goes nowhere."""
    k, v, w = (t.clone() for t in (cache.k, cache.v, cache.weights))
    table, out_table, page = table.cpu().long(), out_table.cpu().long(), cache.page
    there = lambda p: (p >= 0) & (p < cache.pages)  # noqa: E731
    new = []
    for b, n in enumerate(lens):
        n = min(max(n, 0), table.shape[1] * page)
        m = min(n, keep)
        r = min(recent, m)
        new.append(m)
        i, j = torch.arange(n), torch.arange(m)
        src, dst = table[b, i // page], out_table[b, j // page]
        for h in range(cache.kv_heads):
            old = cache.weights[src.clamp(0, cache.pages - 1).to(DEV), h, (i % page).to(DEV)].cpu()
            old = torch.where(there(src), old, torch.full_like(old, -math.inf))[:n - r]
            stay = torch.cat([torch.sort(old, descending=True, stable=True).indices[:m - r].sort().values, i[n - r:]])
            for to, of in ((k, cache.k), (v, cache.v), (w, cache.weights)):
                x = of[src[stay].clamp(0, cache.pages - 1).to(DEV), h, (stay % page).to(DEV)]
                x[~there(src[stay]).to(DEV)] = 0
                ok = there(dst)
                to[dst[ok].to(DEV), h, (j % page)[ok].to(DEV)] = x[ok.to(DEV)]
    return k, v, w, new


def same(got, want):
    return torch.equal(torch.nan_to_num(got.float(), 77.0), torch.nan_to_num(want.float(), 77.0))


def check_evict(cache, table, lengths, out_table, wide, keep, recent, lens, reported, max_len=None):
    before = wide.clone()
    k, v, w, new = evicted(cache, table, lens, out_table, keep, recent)
    got = kv.evict(cache, table, lengths, out_table, keep, recent, max_len=max_len)
    if reported:
        with pytest.raises(_lib.DitkError):
            kv.check_tables()
    kv.check_tables()
    assert got.tolist() == new
    assert same(cache.k, k) and same(cache.v, v) and same(cache.weights, w)
    hk, page = cache.kv_heads, cache.page
    assert same(wide[:, hk:], before[:, hk:]) and same(wide[:, :, :4], before[:, :, :4])
    assert same(wide[:, :, 4 + page:], before[:, :, 4 + page:])


@pytest.mark.parametrize("n,page", [(200, 16), (40000, 128)])  # one workgroup, parts of a row
@pytest.mark.parametrize("where,keep,recent", [
    ("old", 0.5, 10), ("last", 0.5, 10), ("all", 1.0, 10), ("all", 2.0, 0), ("dropped", 0.25, None), ("last", 0.25, None)])
@pytest.mark.parametrize("bad", [-1, None, 2**31 - 1, -2**31])
def test_evict_reports_bad_pages(n, page, where, keep, recent, bad):
    """A page that the cache lacks, among slots that weights decide on, among the recent ones, where every slot stays, and
    where only recent ones do: reported, its slots zeros where they stay, the other sequence as ever."""
    keep = int(n * keep)
    recent = keep if recent is None else recent
    stay = [min(n, keep), min(90, keep)]
    cache, table, lengths, out_table, wide = cache_of([n, 90], 2, 64, page, 5, more=stay)
    slot = {"old": n // 3, "last": n - 1, "all": n // 2, "dropped": 5}[where]
    table[0, slot // page] = cache.pages if bad is None else bad
    check_evict(cache, table, lengths, out_table, wide, keep, recent, [n, 90], True)


@pytest.mark.parametrize("n,page", [(200, 16), (40000, 128)])
def test_evict_into_bad_pages(n, page):
    """What would go to a page that the cache lacks goes nowhere, and is reported."""
    keep = n // 2
    for bad in (-1, 2**31 - 1):
        cache, table, lengths, out_table, wide = cache_of([n, 90], 2, 64, page, 6, more=[keep, 90])
        out_table[0, 1] = bad
        check_evict(cache, table, lengths, out_table, wide, keep, 16, [n, 90], True)
        cache, table, lengths, out_table, wide = cache_of([n, 90], 2, 64, page, 6, more=[keep, 90])
        out_table[0, 2] = cache.pages
        check_evict(cache, table, lengths, out_table, wide, keep, 16, [n, 90], True)


@pytest.mark.parametrize("n,page", [(190, 16), (40000, 128)])
def test_evict_clamps_lengths(n, page):
    """Lengths outside the table are clamped to it, and to max_len; both are reported."""
    full = -(-n // page) * page
    for given, holds in ((-5, 0), (-2**31, 0), (2**31 - 1, full), (full + 1, full)):
        cache, table, lengths, out_table, wide = cache_of([full, 90], 1, 128, page, 7, more=[n // 2, 90])
        lengths[0] = given
        check_evict(cache, table, lengths, out_table, wide, n // 2, 9, [holds, 90], True)
    cache, table, lengths, out_table, wide = cache_of([full, 90], 1, 128, page, 7, more=[100, 90])
    check_evict(cache, table, lengths, out_table, wide, 100, 9, [150, 90], True, max_len=150)
    cache, table, lengths, out_table, wide = cache_of([n, 90], 1, 128, page, 7, more=[100, 90])
    check_evict(cache, table, lengths, out_table, wide, 100, 9, [n, 90], False, max_len=n)


@pytest.mark.parametrize("layout", ["interleaved", "heads"])
@pytest.mark.parametrize("lens,keep,recent,hk,d,page", [
    ([300, 0, 41, 1], 40, 7, 3, 64, 16), ([5000, 900], 700, 64, 2, 128, 64), ([40000], 3000, 1, 2, 64, 256)])
def test_evict_layouts(layout, lens, keep, recent, hk, d, page):
    """Pages and heads in any order, weights in wider rows."""
    cache, table, lengths, out_table, wide = cache_of(lens, hk, d, page, 8, layout, [min(n, keep) for n in lens])
    check_evict(cache, table, lengths, out_table, wide, keep, recent, lens, False)


def long_cache(lens, hk, d, page, seed):
    """A cache made on the device, its pages in no order."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    total = sum(counts) + 2
    k = torch.randn((total, hk, page, d), generator=g, device=DEV).bfloat16()
    v = (torch.randn((total, hk, page, d), generator=g, device=DEV) + 0.5).bfloat16()
    order = torch.randperm(total, generator=g, device=DEV).int()
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device=DEV)
    for b, c in enumerate(counts):
        at = sum(counts[:b])
        table[b, :c] = order[at:at + c]
    return kv.PagedCache(k, v, torch.zeros((total, hk, page), device=DEV)), table, torch.tensor(lens, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("lens,heads,hk,d,page", [
    ([65536, 65537, 3], 2, 1, 64, 16), ([262144, 262145], 2, 1, 64, 256), ([262145, 1000], 20, 10, 64, 16),
    ([300001], 3, 1, 128, 16), ([600000, 1024], 17, 1, 64, 16), ([540673], 1, 1, 64, 32)])
def test_decode_long(lens, heads, hk, d, page):
    """Around 65536 and 262144 slots, where chunks become longer, and beyond, where a unit's pages are read in several
    parts, with one chunk a unit and with two: against 64 bits, and bitwise what each sequence is alone."""
    cache, table, lengths = long_cache(lens, hk, d, page, sum(lens) + hk)
    q = torch.randn((len(lens), heads * d), generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
    out, lse = kv.decode_attn(q, cache, table, lengths, heads, return_lse=True)
    kv.check_tables()
    weighed, e = kv.decode_attn(q, cache, table, lengths, heads, return_lse=True, weights="set")
    assert torch.equal(weighed, out) and torch.equal(e, lse)
    for b, n in enumerate(lens):
        want, e, p, mass, size = attend64(q[b].view(heads, 1, d), get(cache.k, table[b], n).transpose(0, 1),
                                          get(cache.v, table[b], n).transpose(0, 1))
        score, rel = errors32(d, n, size)
        check_out(out[b].view(heads, d), want[:, 0], mass[:, 0], rel)
        # fp32: the score's loss, half a step an addition of the sum, the logarithm and its product
        assert bool(((lse[b].double() - e[:, 0]).abs() <= score + (n + 4) * 2.0 ** -24 + 2.0 ** -22 * e[:, 0].abs()).all())
        w = p[:, 0].view(hk, heads // hk, n).sum(1).t()
        off = (get(cache.weights, table[b], n).double() - w).abs()
        assert bool((off <= 2 * (2 * rel + 2.0 ** -19 + (heads // hk + 1) * 2.0 ** -24) * w + 2.0 ** -126).all())
        alone, e = kv.decode_attn(q[b:b + 1], cache, table[b:b + 1], lengths[b:b + 1], heads, return_lse=True, max_len=n)
        assert torch.equal(alone[0], out[b]) and torch.equal(e[0], lse[b])


def test_weights_apart():
    """Weights in the buffer of keys and values: refused where they share an element with them, taken where they lie between."""
    pages, hk, page, d = 5, 2, 16, 64
    block = page * d
    for head_first in (False, True):
        # a record of keys, values and weights for each page (or head), then heads (or pages) in it
        n, m = (hk, pages) if head_first else (pages, hk)
        line = 2 * m * block + 2 * m * page
        x = torch.zeros(n * line, dtype=torch.bfloat16, device=DEV)
        f = x.view(torch.float32)
        ps, hs = (block, line) if head_first else (line, block)
        wps, whs = (page, line // 2) if head_first else (line // 2, page)
        k, v = (x.as_strided((pages, hk, page, d), (ps, hs, d, 1), i * m * block) for i in range(2))
        w = lambda off: f.as_strided((pages, hk, page), (wps, whs, 1), off)  # noqa: E731
        first = m * block  # floats up to a record's weights
        assert kv.PagedCache(k, v, w(first)).weights is not None
        for off in (0, 4, first - page, first - 4, first - 1, m * block // 2):
            with pytest.raises(ValueError, match="overlap"):
                kv.PagedCache(k, v, w(off))
    # each head's weights behind its keys and values
    line = 2 * block + 2 * page
    x = torch.zeros(pages * hk * line, dtype=torch.bfloat16, device=DEV)
    f = x.view(torch.float32)
    k, v = (x.as_strided((pages, hk, page, d), (hk * line, line, d, 1), i * block) for i in range(2))
    w = lambda off: f.as_strided((pages, hk, page), (hk * line // 2, line // 2, 1), off)  # noqa: E731
    kv.PagedCache(k, v, w(block))
    for off in (0, block - 1, block // 2):
        with pytest.raises(ValueError, match="overlap"):
            kv.PagedCache(k, v, w(off))
    # another order than theirs
    with pytest.raises(ValueError, match="overlap"):
        kv.PagedCache(k, v, f.as_strided((pages, hk, page), (page, pages * page, 1), 0))
    kv.PagedCache(k, v, torch.zeros((pages, hk, page), device=DEV))
