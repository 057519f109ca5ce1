"""Paged key-value caches: append, decode_attn and evict against their definitions in 64 bits."""
import math

import pytest
import torch

from tests.kv_reference import DEV, NAN, attend64, check_out, errors32, get, paged

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from ditserve_amd import _lib, kv, ops


def queries(batch, heads, d, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((batch, heads * d), generator=g) + 0.1).bfloat16().to(DEV)


def check_decode(q, cache, lens, keys, values, heads, out, lse=None, table=None, before=None, scale=None):
    """Every sequence's output (and lse, and the weights in the cache: `before` them or NaN-free from none) as defined."""
    d, hk = cache.head_dim, cache.kv_heads
    for b, n in enumerate(lens):
        got = out[b].view(heads, d)
        if n == 0:
            assert not got.any() and (lse is None or bool((lse[b] == -math.inf).all()))
            continue
        want, e, p, mass, size = attend64(q[b].view(heads, 1, d), keys[b].transpose(0, 1), values[b].transpose(0, 1),
                                          scale=scale)
        score, rel = errors32(d, n, size)
        check_out(got, want[:, 0], mass[:, 0], rel)
        if lse is not None:
            assert bool(((lse[b].double() - e[:, 0]).abs() <= score + (n + 4) * 2.0 ** -24 + 2.0 ** -22 * e[:, 0].abs()).all())
        if table is not None:
            w = get(cache.weights, table[b], n).double()  # [n, hk]
            s = p[:, 0].view(hk, heads // hk, n).sum(1).t()
            ref = s if before is None else s + before[b].double()
            # the probability's loss, the lse's half step of up to 32 log2 units, half a step an addition
            assert bool(((w - ref).abs() <= (2 * rel + 2.0 ** -19) * s + (heads // hk + 1) * 2.0 ** -24 * ref + 2.0 ** -126).all())


DECODE = [
    ([1], 1, 1, 128, 16), ([500], 12, 2, 128, 16), ([0, 5, 33, 0], 8, 8, 64, 32), ([31, 32, 33, 64, 65], 32, 8, 128, 64),
    ([255, 256, 257, 1000], 40, 8, 128, 128), ([700, 3], 16, 1, 64, 256), ([511, 513, 129, 127], 9, 3, 128, 16),
    ([4097, 1, 300], 7, 1, 128, 64), ([33000, 12000], 4, 2, 128, 32), ([40001], 34, 2, 64, 16), ([300], 17, 1, 128, 32),
    ([0], 4, 4, 128, 16), ([2, 1, 2, 1] * 30, 2, 1, 64, 16), ([3, 0, 600, 1] * 75, 2, 1, 64, 16), ([1] * 599 + [1100], 1, 1, 64, 32),
]


@pytest.mark.parametrize("lens,heads,hk,d,page", DECODE)
@pytest.mark.parametrize("weights", [None, "set", "add"])
def test_decode(lens, heads, hk, d, page, weights):
    cache, table, lengths, keys, values = paged(lens, hk, d, page, sum(lens) + heads, weights=True)
    before = None
    if weights == "add":
        cache.weights.normal_().abs_()
        before = [get(cache.weights, table[b], n) for b, n in enumerate(lens)]
    kept = cache.weights.clone()
    q = queries(len(lens), heads, d, 1)
    out, lse = kv.decode_attn(q, cache, table, lengths, heads, weights=weights, return_lse=True)
    kv.check_tables()
    check_decode(q, cache, lens, keys, values, heads, out, lse, table if weights else None, before)
    # slots that no sequence holds stay
    held = torch.zeros_like(kept, dtype=torch.bool)
    for b, n in enumerate(lens):
        i = torch.arange(n, device=DEV)
        held[table[b].long()[i // page], :, i % page] = weights is not None
    assert torch.equal(cache.weights.view(torch.int32)[~held], kept.view(torch.int32)[~held])


@pytest.mark.parametrize("layout", ["interleaved", "heads"])
@pytest.mark.parametrize("d,page", [(128, 64), (64, 16)])
def test_decode_layouts_and_batches(layout, d, page):
    """Strided caches, q from wider rows, out into wider rows; each sequence bitwise what it is alone."""
    lens, heads, hk = [300, 1, 777, 0, 128], 10, 2
    cache, table, lengths, keys, values = paged(lens, hk, d, page, 7, layout=layout)
    wide = queries(len(lens), heads + 2, d, 2)
    q = wide[:, d:d + heads * d]
    buf = torch.full((len(lens), (heads + 1) * d), 7.0, dtype=torch.bfloat16, device=DEV)
    out = kv.decode_attn(q, cache, table, lengths, heads, softmax_scale=0.3, out=buf[:, :heads * d])
    kv.check_tables()
    check_decode(q, cache, lens, keys, values, heads, out, scale=0.3)
    assert bool((buf[:, heads * d:] == 7).all())
    for b, n in enumerate(lens):
        alone = kv.decode_attn(q[b:b + 1], cache, table[b:b + 1], lengths[b:b + 1], heads, softmax_scale=0.3, max_len=n)
        assert torch.equal(alone[0], out[b])


@pytest.mark.parametrize("batch,heads,hk,d,page", [(72, 16, 8, 64, 16), (100, 40, 2, 128, 64), (300, 8, 8, 64, 32)])
def test_decode_of_many(batch, heads, hk, d, page):
    """More chunks than waves: each sequence bitwise what it is alone; lengths around those of a chunk, of two and of none."""
    some = [1100, 128 * 9, 128 * 9 + 1, 1025, 1024, 64 * 3, 65, 64, 1, 0, 2000, 128 * 14, 128 * 14 + 31, 8192, 8193]
    lens = [some[i % len(some)] if i % 3 == 0 else 1300 + 7 * i % 640 for i in range(batch)]
    cache, table, lengths, keys, values = paged(lens, hk, d, page, batch)
    cache.v[table[3, 0].long(), 0, 5, 7] = math.inf
    q = queries(batch, heads, d, 8)
    out, lse = kv.decode_attn(q, cache, table, lengths, heads, return_lse=True)
    kv.check_tables()
    picked = [i for i in range(batch) if i != 3 and i % 3 == 0][:24] + [1, batch - 2]
    pick = torch.tensor(picked, device=DEV)
    check_decode(q[pick], cache, [lens[i] for i in picked], [keys[i] for i in picked], [values[i] for i in picked], heads,
                 out[pick], lse[pick])
    assert bool((out[3].view(hk, heads // hk, d)[0, :, 7] == math.inf).all()) and int(torch.isfinite(out[3]).sum()) == heads * d - heads // hk
    for b in {3, *picked}:
        alone, e = kv.decode_attn(q[b:b + 1], cache, table[b:b + 1], lengths[b:b + 1], heads, return_lse=True)
        assert torch.equal(alone[0], out[b]) and torch.equal(e[0], lse[b])


def test_decode_infinite_values():
    """An infinite value of a slot that is held is infinite in the output, one of a slot that is not stays out."""
    cache, table, lengths, _, _ = paged([40, 300], 1, 128, 16, 3)
    i = 299 // 16
    cache.v[table[1, i].long(), 0, 299 % 16, 5] = math.inf  # the last slot held
    out = kv.decode_attn(queries(2, 4, 128, 4), cache, table, lengths, 4).float().view(2, 4, 128)
    assert torch.isfinite(out[0]).all() and bool((out[1, :, 5] == math.inf).all())
    assert torch.isfinite(out[1, :, :5]).all() and torch.isfinite(out[1, :, 6:]).all()


def test_decode_reports_bad_tables():
    """Bad pages are absent slots, bad lengths are clamped; both are reported, once."""
    cache, table, lengths, keys, values = paged([200, 100], 2, 128, 16, 5, weights=True)
    q = queries(2, 4, 128, 5)
    for bad in (-1, cache.pages, 2**31 - 1, -2**31):
        t = table.clone()
        t[0, 3] = bad  # slots 48..63
        out = kv.decode_attn(q, cache, t, lengths, 4, weights="set")
        with pytest.raises(_lib.DitkError):
            kv.check_tables()
        kv.check_tables()
        left = torch.cat([torch.arange(48), torch.arange(64, 200)]).to(DEV)
        check_decode(q, cache, [136, 100], [keys[0][left], keys[1]], [values[0][left], values[1]], 4, out)
    for bad, n in ((-5, 0), (2**31 - 1, 208), (-2**31, 0), (209, 208)):
        x = lengths.clone()
        x[0] = bad
        out = kv.decode_attn(q, cache, table, x, 4)
        with pytest.raises(_lib.DitkError):
            kv.check_tables()
        check_decode(q[1:], cache, [100], keys[1:], values[1:], 4, out[1:])
        if n == 0:
            assert not out[0].any()
    out = kv.decode_attn(q, cache, table, lengths, 4, max_len=150)
    with pytest.raises(_lib.DitkError):
        kv.check_tables()
    check_decode(q, cache, [150, 100], [keys[0][:150], keys[1]], [values[0][:150], values[1]], 4, out)


def test_decode_far_pages():
    """Offsets past 2^31 elements and 2^32 bytes: the last pages of a large cache."""
    pages, hk, page, d = 33000, 8, 64, 128
    k, v = torch.empty((2, pages, hk, page, d), dtype=torch.bfloat16, device=DEV).unbind(0)
    cache = kv.PagedCache(k, v)
    n, g = 150, torch.Generator(device=DEV).manual_seed(1)
    table = torch.tensor([[pages - 1, pages - 3, 17]], dtype=torch.int32, device=DEV)
    keys, values = torch.randn((2, n, hk, d), generator=g, device=DEV).bfloat16().unbind(0)
    lengths = kv.append(cache, keys.flatten(1), values.flatten(1), table, torch.zeros(1, dtype=torch.int32, device=DEV),
                        ops.Segments([0, n], DEV))
    q = queries(1, 16, d, 6)
    out = kv.decode_attn(q, cache, table, lengths, 16)
    kv.check_tables()
    check_decode(q, cache, [n], [keys], [values], 16, out)


@pytest.mark.parametrize("before,counts,hk,d,page", [
    ([0], [1], 1, 64, 16), ([5, 0, 63, 64], [1, 1, 1, 1], 8, 128, 64), ([0, 7, 100], [300, 0, 29], 3, 128, 16),
    ([15, 16, 17], [1, 33, 16], 2, 64, 256), ([0] * 1500, [i % 3 for i in range(1500)], 1, 64, 16)])
@pytest.mark.parametrize("layout", ["plain", "interleaved"])
def test_append(before, counts, hk, d, page, layout):
    after = [a + b for a, b in zip(before, counts)]
    cache, table, _, _, _ = paged(after, hk, d, page, 11, layout=layout, weights=True)
    want = [t.clone() for t in (cache.k, cache.v, cache.weights)]
    T = sum(counts)
    both = torch.randn((T, 2 * hk * d + 8), generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    k, v = both[:, :hk * d], both[:, hk * d:2 * hk * d]
    lengths = torch.tensor(before, dtype=torch.int32, device=DEV)
    cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
    new = kv.append(cache, k, v, table, lengths, ops.Segments(cu, DEV))
    kv.check_tables()
    assert new.tolist() == after and lengths.tolist() == before
    seq = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts)).to(DEV)
    slot = torch.arange(T, device=DEV) - torch.tensor(cu, device=DEV)[seq] + lengths[seq]
    at = (table.long()[seq, slot // page], slice(None), slot % page)
    want[0][at], want[1][at], want[2][at] = k.reshape(T, hk, d), v.reshape(T, hk, d), 0.0
    for got, ref in zip((cache.k, cache.v, cache.weights), want):
        assert torch.equal(torch.nan_to_num(got.float(), 99.0), torch.nan_to_num(ref.float(), 99.0))
    if counts == [1] * len(counts):  # the same without segments
        cache.k.zero_()
        assert kv.append(cache, k, v, table, lengths).tolist() == after
        assert torch.equal(get(cache.k, table[0], after[0])[-1], k.reshape(T, hk, d)[0])


def test_tables_without_pages():
    """No columns: nothing is held, written or moved."""
    cache = kv.PagedCache.empty(2, 2, 64, 16, DEV)
    before = cache.k.clone()
    none, zero = torch.empty((3, 0), dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    q = queries(3, 4, 64, 1)
    for weights in (None, "set", "add"):
        out, lse = kv.decode_attn(q, cache, none, zero, 4, weights=weights, return_lse=True)
        assert not out.any() and bool((lse == -math.inf).all())
    assert kv.evict(cache, none, zero, none.clone(), 4).tolist() == [0, 0, 0]
    kv.check_tables()
    assert kv.append(cache, q[:, :128], q[:, 128:], none, zero).tolist() == [0, 0, 0]
    with pytest.raises(_lib.DitkError):
        kv.check_tables()
    assert torch.equal(cache.k.view(torch.int16), before.view(torch.int16))


def test_overlapping_operands_are_refused():
    pages, hk, page, d = 6, 2, 16, 64
    x = torch.zeros((pages, 2 * hk, page, d), dtype=torch.bfloat16, device=DEV)
    w = torch.zeros((pages, hk, page), device=DEV)
    cache = kv.PagedCache(x[:, ::2], x[:, 1::2], w)  # heads of keys and of values in turn
    kv.PagedCache(x[:3, :hk], x[3:, :hk])
    one, block = x[:, :hk], page * d
    for k, v in ((one, one), (one, x[:, 1:1 + hk]), (one[1:], one[:-1]), (x[:, ::2], x[:, :hk]),
                 (one, x.view(-1)[block // 2:].as_strided(one.shape, one.stride()))):
        with pytest.raises(ValueError, match="overlap"):
            kv.PagedCache(k, v)
    for strides in ((block, block), (block, 2 * block), (0, block), (block // 2, 6 * block)):  # pages that overlap heads
        with pytest.raises(ValueError, match="overlap"):
            kv.PagedCache(x.as_strided(one.shape, (*strides, d, 1)), torch.zeros_like(one))
    with pytest.raises(ValueError, match="weights"):
        kv.PagedCache(x[:, ::2], x[:, 1::2], w.as_strided(w.shape, (page, page, 1)))
    # operands that lie in the cache
    inside = x.view(-1).view(torch.int32)
    table, lengths, fine = inside[:8].view(2, 4), inside[:2], torch.zeros((2, 4), dtype=torch.int32, device=DEV)
    n, q = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros((2, hk * d), dtype=torch.bfloat16, device=DEV)
    for bad in ((table, n, fine), (fine, lengths, fine.clone()), (fine, n, table)):
        with pytest.raises(ValueError, match="lies in the cache"):
            kv.evict(cache, *bad, 4)
    for bad in ((x.view(-1)[:2 * hk * d].view(2, hk * d), fine, n), (q, table, n), (q, fine, lengths)):
        with pytest.raises(ValueError, match="lies in the cache"):
            kv.decode_attn(bad[0], cache, *bad[1:], hk, weights="set")
    # a table that is a few columns of one that the cache follows is none
    flat = torch.zeros(4096 + pages * 2 * hk * block, dtype=torch.bfloat16, device=DEV)
    rows, rest = flat[:4096].view(torch.int32).view(2, 1024), flat[4096:].view(x.shape)
    rows[1] = 1
    beside = kv.PagedCache(rest[:, :hk], rest[:, hk:])
    assert kv.append(beside, q, q, rows[:, 1020:], n).tolist() == [1, 1]


def test_append_past_the_table():
    """Rows that no page is there for are not written; the length stops where the table does."""
    cache, table, _, _, _ = paged([40, 30], 2, 64, 16, 12)
    table[0, 1] = cache.pages
    rows = torch.ones((80, 128), dtype=torch.bfloat16, device=DEV)
    kept = cache.k.clone()
    new = kv.append(cache, rows, rows, table, torch.tensor([10, 40], dtype=torch.int32, device=DEV),
                    ops.Segments([0, 60, 80], DEV))
    with pytest.raises(_lib.DitkError):
        kv.check_tables()
    assert new.tolist() == [48, 48]
    written = torch.zeros(cache.pages, 16, dtype=torch.bool)
    for b, slots in ((0, [*range(10, 16), *range(32, 48)]), (1, [])):
        for i in slots:
            written[int(table[b, i // 16]), i % 16] = True
    written = written[:, None, :, None].expand(kept.shape).to(DEV)
    assert bool((cache.k[written] == 1).all())
    # (sequence 1's slots 40.. lie in pages that its table lacks)
    assert torch.equal(torch.nan_to_num(cache.k[~written].float(), 9.0), torch.nan_to_num(kept[~written].float(), 9.0))


def kept_slots(w, n, keep, recent):
    """Slots that stay, ascending, of one (sequence, head): by weight, then by slot."""
    m = min(n, keep)
    r = min(recent, m)
    w = [(-math.inf if math.isnan(x) else x) for x in w[:n].tolist()]
    old = sorted(range(n - r), key=lambda i: (-w[i], i))[:m - r]
    return sorted(old) + list(range(n - r, n))


@pytest.mark.parametrize("lens,keep,recent,hk,d,page", [
    ([1], 1, 0, 1, 64, 16), ([1, 2, 3], 2, 1, 2, 128, 16), ([100, 7, 0, 64], 20, 5, 3, 64, 16),
    ([5000, 300], 1000, 100, 2, 128, 64), ([2000], 1999, 0, 1, 64, 32), ([700, 650], 64, 64, 2, 128, 256),
    ([33, 65, 129], 33, 32, 1, 128, 32), ([70000], 600, 17, 1, 64, 128),
    ([1024], 511, 1, 2, 64, 64), ([1025, 4096], 1024, 0, 1, 64, 16), ([4097, 8192], 3, 1, 1, 64, 32), ([8193], 8192, 100, 1, 64, 64),
    ([32768], 16000, 0, 1, 64, 128), ([32769, 20, 9000], 8193, 8192, 1, 64, 128), ([131073, 50], 40000, 33, 1, 64, 256)])
@pytest.mark.parametrize("kind", ["random", "ties", "steps", "odd"])
def test_evict(lens, keep, recent, hk, d, page, kind):
    stay = [min(n, keep) for n in lens]
    cache, table, lengths, out_table, keys, values = paged(lens, hk, d, page, sum(lens), weights=True, more=stay)
    g = torch.Generator(device=DEV).manual_seed(keep)
    w = torch.randn(cache.weights.shape, generator=g, device=DEV)
    if kind == "ties":
        w = torch.round(w * 2) / 2  # zeros of both signs among them
    elif kind == "steps":  # few values far apart: digits that leave nothing to decide, and ones that do
        w = torch.exp2(torch.randint(-3, 3, w.shape, generator=g, device=DEV).float()) + (torch.rand(w.shape, generator=g, device=DEV) < 0.3) * w.abs()
    elif kind == "odd":
        pick = torch.randint(0, 6, w.shape, generator=g, device=DEV)
        for i, x in enumerate((NAN, math.inf, -math.inf, 1e-42, -0.0)):
            w[pick == i] = x
    cache.weights.copy_(w)
    kept = [t.clone() for t in (cache.k, cache.v, cache.weights)]
    new = kv.evict(cache, table, lengths, out_table, keep, recent)
    kv.check_tables()
    assert new.tolist() == stay and lengths.tolist() == lens
    touched = torch.zeros(cache.pages, page, dtype=torch.bool, device=DEV)
    for b, (n, m) in enumerate(zip(lens, stay)):
        ws = get(kept[2], table[b], n)
        got = [get(t, out_table[b], m) for t in (cache.k, cache.v, cache.weights)]
        for h in range(hk):
            at = torch.tensor(kept_slots(ws[:, h].cpu(), n, keep, recent), dtype=torch.long, device=DEV)
            assert torch.equal(got[0][:, h], keys[b][at, h]) and torch.equal(got[1][:, h], values[b][at, h])
            assert torch.equal(got[2][:, h].view(torch.int32), ws[at, h].view(torch.int32))
        i = torch.arange(m, device=DEV)
        touched[out_table[b].long()[i // page], i % page] = True
    rest = ~touched[:, None].expand(-1, hk, -1)
    for t, ref in zip((cache.k, cache.v, cache.weights), kept):
        assert torch.equal(torch.nan_to_num(t[rest].float(), 9.0), torch.nan_to_num(ref[rest].float(), 9.0))
