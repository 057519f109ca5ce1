"""Causal attention of packed prompts with grouped heads, against its definition in 64 bits."""
import math

import pytest
import torch

from tests.kv_reference import DEV, attend64, check_out, errors32

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from ditserve_amd import attention, ops


def cu_of(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def prompt(lens_q, lens_k, heads, hk, d, seed, fused=False):
    g = torch.Generator().manual_seed(seed)
    tq, tk = sum(lens_q), sum(lens_k)
    q = torch.randn((tq, heads * d), generator=g)
    k, v = torch.randn((tk, hk * d), generator=g), torch.randn((tk, hk * d), generator=g) + 0.5
    if fused:
        x = torch.cat([q, k, v], 1).bfloat16().to(DEV)
        return x.split([heads * d, hk * d, hk * d], 1)
    return [t.bfloat16().to(DEV) for t in (q, k, v)]


def check(q, k, v, lens_q, lens_k, heads, hk, d, out, lse, scale=None):
    cq, ck = cu_of(lens_q), cu_of(lens_k)
    for m, (nq, nk) in enumerate(zip(lens_q, lens_k)):
        rows, keys = slice(cq[m], cq[m + 1]), slice(ck[m], ck[m + 1])
        if nq == 0:
            continue
        seen = torch.arange(nk, device=DEV)[None] <= torch.arange(nq, device=DEV)[:, None] + (nk - nq)
        want, e, _, mass, size = attend64(q[rows].view(nq, heads, d).transpose(0, 1), k[keys].view(nk, hk, d).transpose(0, 1),
                                          v[keys].view(nk, hk, d).transpose(0, 1), seen, scale)
        some = seen.any(1)
        got = out[rows].view(nq, heads, d).transpose(0, 1)
        score, rel = errors32(d, nk, size)
        want, mass = torch.nan_to_num(want), torch.nan_to_num(mass)
        # the probabilities are rounded to bf16 (8 bits) before the second product, each by half a step at most
        check_out(got, want, mass, rel, p_bits=8)
        assert not got[:, ~some].any()
        if lse is not None:
            x, e = lse[:, rows].double(), e
            assert bool((x[:, ~some] == -math.inf).all())
            off = (x - e)[:, some].abs()
            assert bool((off <= score + (nk + 4) * 2.0 ** -24 + 2.0 ** -22 * e[:, some].abs()).all())


CASES = [
    # queries, keys, heads, key heads, head dim
    ([1], [1], 1, 1, 128), ([77], [77], 12, 12, 64), ([63, 64, 65], None, 8, 2, 128), ([127, 128, 129, 0, 255], None, 6, 2, 64),
    ([256, 257, 1], None, 5, 1, 128), ([700, 31, 1290], None, 4, 4, 128), ([2000], None, 16, 8, 64),
    ([1, 1, 1], [1, 100, 5000], 8, 1, 128), ([300, 20], [1301, 20], 7, 1, 64), ([64, 128], [65, 191], 32, 8, 128),
    # queries that see no key: more queries than keys, and no keys
    ([100, 300], [30, 77], 4, 2, 128), ([5, 300, 7], [0, 1, 0], 8, 8, 64), ([0, 0], [0, 9], 2, 1, 128),
    ([513], [256], 3, 3, 64), ([9000], None, 2, 1, 128), ([3000, 2500], None, 24, 8, 64),
    # few queries over many keys, among others
    ([1], [1024], 1, 1, 64), ([1, 16, 3, 32, 33], [5000, 1024, 1023, 4097, 4097], 8, 2, 128), ([128, 0, 7], [1100, 3000, 1600], 5, 5, 64),
    ([10, 300, 2], [9000, 1300, 1025], 12, 1, 128), ([1, 2, 1] * 100, [1024, 3, 1030] * 100, 2, 1, 64), ([3, 70, 0] * 45, None, 4, 2, 64), ([100], [2000], 6, 6, 128), ([18, 1], [1030, 70000], 7, 1, 64),
]


@pytest.mark.parametrize("lens_q,lens_k,heads,hk,d", CASES)
@pytest.mark.parametrize("fused", [False, True])
def test_causal(lens_q, lens_k, heads, hk, d, fused):
    if fused and lens_k is not None and sum(lens_q) != sum(lens_k):
        fused = False
    lens_k = lens_k or lens_q
    q, k, v = prompt(lens_q, lens_k, heads, hk, d, sum(lens_q) + heads, fused)
    seg_q, seg_k = ops.Segments(cu_of(lens_q), DEV), ops.Segments(cu_of(lens_k), DEV)
    out, lse = ops.flash_attn_causal(q, k, v, seg_q, seg_k, heads, hk, d, return_lse=True)
    check(q, k, v, lens_q, lens_k, heads, hk, d, out, lse)


@pytest.mark.parametrize("d", [64, 128])
def test_packed_is_alone(d):
    """Each segment bitwise what it is alone, whatever work items the launches take; with device tables too."""
    lens_q, heads, hk = [1500, 3, 700, 4100, 64, 20, 1], 16, 4
    lens_k = [1500, 40, 700, 4100, 2064, 3020, 1024]
    q, k, v = prompt(lens_q, lens_k, heads, hk, d, 3)
    q[::37] *= 5.0  # maxima that rise late
    k[::53] *= 4.0
    cq, ck = cu_of(lens_q), cu_of(lens_k)
    out, lse = ops.flash_attn_causal(q, k, v, ops.Segments(cq, DEV), ops.Segments(ck, DEV), heads, hk, d, return_lse=True)
    check(q, k, v, lens_q, lens_k, heads, hk, d, out, lse)
    cu = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (cq, ck)]
    same = attention.causal_attn_varlen_func(q.view(-1, heads, d), k.view(-1, hk, d), v.view(-1, hk, d), *cu, 4100, 4100)
    assert torch.equal(same.view(out.shape), out)
    for m in range(len(lens_q)):
        a, b = slice(cq[m], cq[m + 1]), slice(ck[m], ck[m + 1])
        for h in (slice(0, heads), slice(0, heads // hk)):  # all heads, and one group of them
            hs = slice(0, h.stop * d), slice(0, h.stop // (heads // hk) * d)
            one, e = ops.flash_attn_causal(q[a, hs[0]], k[b, hs[1]], v[b, hs[1]], ops.Segments([0, lens_q[m]], DEV),
                                           ops.Segments([0, lens_k[m]], DEV), h.stop, h.stop // (heads // hk), d,
                                           return_lse=True)
            assert torch.equal(one, out[a, hs[0]]) and torch.equal(e, lse[h, a])


def test_masked_keys_may_be_anything():
    """Infinities and NaN in keys that a query does not see, the type's lowest value among scores, rows behind the last
    segment, an output in wider rows."""
    lens, heads, hk, d = [200, 333], 6, 3, 128
    q, k, v = prompt(lens, lens, heads, hk, d, 9)
    for i, x in enumerate((math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).min)):
        k[190 + i] = x          # seen by the first segment's last ten queries only
        k[200 + 300 + i] = x
    wide = torch.full((sum(lens) + 5, (heads + 1) * d), 3.0, dtype=torch.bfloat16, device=DEV)
    seg = ops.Segments(cu_of(lens), DEV)
    out = ops.flash_attn_causal(q, k, v, seg, seg, heads, hk, d, out=wide[:sum(lens), :heads * d], softmax_scale=0.2)
    assert bool((wide[sum(lens):] == 3).all()) and bool((wide[:, heads * d:] == 3).all())
    cut = [190, 300]  # the queries that see none of it
    rows = torch.cat([torch.arange(190), torch.arange(200, 500)]).to(DEV)
    check(q[rows], k[rows], v[rows], cut, cut, heads, hk, d, out[rows], None, 0.2)
    assert torch.isnan(out[190].float()).all() and torch.isnan(out[500].float()).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,hk", [(4, 2), (40, 8)])
def test_values_that_are_not_seen(d, heads, hk):
    """Values that are not finite reach the queries that see them and no others, in items of 128 and 256 queries and in
    segments of few queries over many keys."""
    lens_q, lens_k = [700, 1900, 5, 30], [700, 1900, 2005, 1100]
    q, k, v = prompt(lens_q, lens_k, heads, hk, d, 21)
    cq, ck = cu_of(lens_q), cu_of(lens_k)
    bad = [(0, 300, 1, math.nan), (0, 301, 2, math.inf), (0, 690, 3, -math.inf), (1, 1000, 0, math.inf), (1, 1001, 0, -math.inf),
           (2, 2002, 5, math.nan), (3, 1080, 7, math.inf), (3, 1099, 8, math.nan)]  # (segment, key, dim of the last head, value)
    clean = v.clone()
    for m, key, dim, x in bad:
        v[ck[m] + key, (hk - 1) * d + dim] = x
        clean[ck[m] + key, (hk - 1) * d + dim] = 0.25
    seg_q, seg_k = ops.Segments(cq, DEV), ops.Segments(ck, DEV)
    out, lse = ops.flash_attn_causal(q, k, v, seg_q, seg_k, heads, hk, d, return_lse=True)
    want = torch.zeros(out.shape, device=DEV)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    for m, key, dim, x in bad:
        first = cq[m] + key - (lens_k[m] - lens_q[m])  # the first query that sees the key
        for h in range(heads - heads // hk, heads):
            want[first:cq[m + 1], h * d + dim] += x
            hit[first:cq[m + 1], h * d + dim] = True
    assert torch.equal(torch.isnan(out.float())[hit], torch.isnan(want)[hit])
    assert torch.equal(torch.nan_to_num(out.float())[hit] > 0, torch.nan_to_num(want)[hit] > 0)
    assert bool((out.float().abs()[hit & ~torch.isnan(want)] == math.inf).all())
    # the rest as without them
    ref = ops.flash_attn_causal(q, k, clean, seg_q, seg_k, heads, hk, d)
    good = torch.where(hit, ref, out)
    check(q, k, clean, lens_q, lens_k, heads, hk, d, good, lse)


def test_offsets_past_32_bits():
    """Rows of a buffer past 4 GiB, on both sides."""
    n, heads, hk, d = 700, 2, 1, 128
    wide = torch.empty((n, 3 * (1 << 20)), dtype=torch.bfloat16, device=DEV)
    q, k, v = prompt([n], [n], heads, hk, d, 5)
    x = wide[:, -1024:]
    x[:, :256], x[:, 256:384], x[:, 384:512] = q, k, v
    seg = ops.Segments([0, n], DEV)
    out, lse = ops.flash_attn_causal(x[:, :256], x[:, 256:384], x[:, 384:512], seg, seg, heads, hk, d, return_lse=True,
                                     out=x[:, 512:768])
    check(q, k, v, [n], [n], heads, hk, d, out, lse)


def test_refusals():
    q, k, v = prompt([8], [8], 4, 2, 64, 1)
    seg = ops.Segments([0, 8], DEV)
    good = dict(q=q, k=k, v=v, seg_q=seg, seg_k=seg, heads=4, kv_heads=2, head_dim=64)
    ops.flash_attn_causal(**good)
    for change in (dict(heads=3), dict(kv_heads=0), dict(head_dim=96), dict(q=q.float()), dict(k=q), dict(v=v[:7]),
                   dict(seg_q=ops.Segments([0, 7], DEV)), dict(seg_k=ops.Segments([0, 4, 8], DEV)), dict(q=q.cpu()),
                   dict(q=q.t().contiguous().t()), dict(out=q), dict(out=k[:, :64])):
        with pytest.raises(ValueError):
            ops.flash_attn_causal(**{**good, **change})
    from ditserve_amd import _lib
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises((_lib.DitkError, ValueError)):
            ops.flash_attn_causal(**good, softmax_scale=scale)
