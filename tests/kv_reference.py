"""Paged caches for the tests, and what their operators are by definition, in 64 bits."""
import math

import torch

DEV = "cuda"
NAN = float("nan")


def paged(lens, hk, d, page, seed, spare=3, layout="plain", weights=False, more=()):
    """(cache, table, lengths[, table of `more` slots], keys, values): pages in no order; every slot that no sequence
    holds is NaN, every table entry behind the last -1."""
    from ditserve_amd import kv
    g = torch.Generator().manual_seed(seed)
    counts = [[-(-n // page) for n in part] for part in (lens, more)]
    total = sum(map(sum, counts)) + spare
    if layout == "plain":
        k, v = torch.full((2, total, hk, page, d), NAN, dtype=torch.bfloat16, device=DEV).unbind(0)
    elif layout == "interleaved":  # both in a page, and room behind them
        k, v = torch.full((total, 3, hk, page, d), NAN, dtype=torch.bfloat16, device=DEV)[:, :2].unbind(1)
    else:  # heads first
        k, v = torch.full((2, hk, total, page, d), NAN, dtype=torch.bfloat16, device=DEV).transpose(1, 2).unbind(0)
    w = torch.full((total, hk, page), NAN, device=DEV) if weights else None
    order = torch.randperm(total, generator=g).tolist()
    tables = []
    for part in counts:
        t = torch.full((len(part), max([1, *part])), -1, dtype=torch.int32)
        for b, n in enumerate(part):
            t[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        tables.append(t.to(DEV))
    keys, values = [], []
    for b, n in enumerate(lens):
        kk = torch.randn((n, hk, d), generator=g).bfloat16().to(DEV)
        vv = (torch.randn((n, hk, d), generator=g) + 0.5).bfloat16().to(DEV)
        put(k, tables[0][b], kk)
        put(v, tables[0][b], vv)
        keys.append(kk)
        values.append(vv)
    cache = kv.PagedCache(k, v, w)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return (cache, tables[0], lengths, *tables[1:] * bool(more), keys, values)


def put(pages, row, x, first=0):
    """Rows x [n, heads, ...] into a sequence's slots from `first` on."""
    page = pages.shape[2]
    i = torch.arange(first, first + x.shape[0], device=DEV)
    pages[row.long()[i // page], :, i % page] = x


def get(pages, row, n):
    """[n, heads, ...] of a sequence's first n slots."""
    i = torch.arange(n, device=DEV)
    return pages[row.long()[i // pages.shape[2]], :, i % pages.shape[2]]


def attend64(q, k, v, seen=None, scale=None):
    """(out, lse, p, sum of p |v|, largest sum of |q k| scale) of q [heads, rows, d] over k, v [kv_heads, keys, d], in 64
    bits; seen [rows, keys], or all."""
    g = q.shape[0] // k.shape[0]
    q, k, v = q.double(), k.double().repeat_interleave(g, 0), v.double().repeat_interleave(g, 0)
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    s = q @ k.transpose(1, 2).contiguous() * scale
    if seen is not None:
        s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, 2) if s.shape[2] else torch.full(s.shape[:2], -math.inf, dtype=torch.float64, device=s.device)
    p = torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None])
    size = float((q.abs() @ k.abs().transpose(1, 2).contiguous()).max() * scale) if s.numel() else 0.0
    return p @ v, lse, p, p @ v.abs(), size


def errors32(d, keys, size):
    """What sums in fp32 may lose: (of a score, of a probability relative to it).  A score is a sum of d products, each
    addition half a step of at most `size`; exp2 and its argument's product a step each; the sum of the probabilities
    half a step an addition, and the score's loss again through it."""
    score = (d + 4) * 2.0 ** -24 * size
    return score, 2 * score + (keys + 16) * 2.0 ** -24


def check_out(out, want, mass, rel, p_bits=16):
    """out (bf16) against want: half a step of bf16 for the output, and of sum p |v| what the probabilities are off: `rel`,
    and their own rounding to p_bits bits."""
    off = (out.double() - want).abs()
    most = 2.0 ** -8 * want.abs() + (rel + 2.0 ** -p_bits) * 1.01 * mass + 2.0 ** -133
    assert torch.isfinite(out.float()).all()
    assert bool((off <= most).all()), float((off - most).max())
