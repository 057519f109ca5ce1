"""Attention over prompts and a paged key-value cache, as they are measured: cases, inputs, plain forms and the framework's calls.

A cache holds keys and values [pages, kv_heads, page, head_dim] in bf16, and for each of its slots the attention weight
gathered there (fp32).  Sequence b's slot i is slot i % page of page table[b, i // page]; it holds lengths[b] of them, and
entries of the table behind them are -1.  Query head h reads key head h // (heads / kv_heads).

  prompt  causal attention over packed prompts: query i of a segment sees the keys j <= i + (its keys - its queries)
  append  rows of new keys and values into the slots behind each sequence's last
  decode  attention of one new token of each sequence over its slots; "set": the probabilities, summed over the
          query heads of a key head, become the slots' weights
  evict   of each sequence and key head the `recent` last slots and those with the largest weights, `keep` in all (ties:
          the lowest slot), in their order, into the pages of another table

`own` False: plain torch operations.  `own` True: the calls a user makes of ditserve_amd.ops and ditserve_amd.kv.
"""
import math
import random

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16


def listed():
    return [
        # one short prompt of an encoder with causal attention: launch latency
        dict(name="prompt_77", kind="prompt", tokens=77, segments=1, cut=0, prefix=0, heads=12, kv_heads=12, head_dim=64,
             lse=False),
        # the prompts of eight requests, up to 512 tokens each, packed
        dict(name="prompt_8_ragged", kind="prompt", tokens=2897, segments=8, cut=3, prefix=0, heads=32, kv_heads=8,
             head_dim=128, lse=False),
        # the next part of two long prompts, the keys of their first parts in front
        dict(name="prompt_2x1024_after_6001", kind="prompt", tokens=2048, segments=2, cut=-1, prefix=6001, heads=40,
             kv_heads=8, head_dim=128, lse=True),
        # one long prompt
        dict(name="prompt_16384", kind="prompt", tokens=16384, segments=1, cut=0, prefix=0, heads=32, kv_heads=8,
             head_dim=128, lse=False),
        # one request that just began to generate: launch latency
        dict(name="decode_1x500", kind="decode", batch=1, longest=500, cut=-1, heads=12, kv_heads=2, head_dim=128,
             page=16, weights=False, lse=False),
        # a serving batch in the middle of its answers
        dict(name="decode_64_ragged", kind="decode", batch=64, longest=4096, cut=5, heads=32, kv_heads=8, head_dim=128,
             page=64, weights=False, lse=False),
        # one request over a very long context
        dict(name="decode_1x131072", kind="decode", batch=1, longest=131072, cut=-1, heads=40, kv_heads=8, head_dim=128,
             page=128, weights=False, lse=True),
        # long contexts, the weights kept for the eviction that follows
        dict(name="decode_16x32768_set", kind="decode", batch=16, longest=32768, cut=-1, heads=32, kv_heads=8,
             head_dim=128, page=64, weights=True, lse=False),
        # the new tokens of a serving batch
        dict(name="append_64x1", kind="append", tokens=64, segments=64, cut=-1, before=2048, kv_heads=8, head_dim=128,
             page=64),
        # packed prompts into their pages
        dict(name="append_6_ragged", kind="append", tokens=16384, segments=6, cut=2, before=129, kv_heads=8, head_dim=128,
             page=32),
        # a batch whose caches are cut to a quarter
        dict(name="evict_8x8192", kind="evict", batch=8, longest=8192, cut=-1, keep=2048, recent=256, kv_heads=8,
             head_dim=128, page=64),
        # a very long context cut to an eighth
        dict(name="evict_1x131072", kind="evict", batch=1, longest=131072, cut=-1, keep=16384, recent=1024, kv_heads=8,
             head_dim=128, page=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "decode", "decode", "append", "evict"])
    heads, kv_heads = rng.choice([(32, 8), (40, 8), (12, 12), (12, 2), (28, 4), (16, 1), (8, 8), (9, 3)])
    head_dim, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    top = {c["kind"]: work(c) for c in listed() if c["name"] in
           ("prompt_16384", "decode_16x32768_set", "append_6_ragged", "evict_1x131072")}[kind]
    while True:
        if kind == "prompt":
            tokens = _log(rng, 1, 16384)
            case = dict(kind=kind, tokens=tokens, segments=min(tokens, _log(rng, 1, 32)), cut=rng.randrange(1000),
                        prefix=rng.choice([0, 0, 0, _log(rng, 1, 8192)]), heads=heads, kv_heads=kv_heads,
                        head_dim=head_dim, lse=rng.random() < 0.3)
        elif kind == "decode":
            case = dict(kind=kind, batch=_log(rng, 1, 128), longest=_log(rng, 1, 131072),
                        cut=rng.choice([-1, rng.randrange(1000)]), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                        page=page, weights=rng.random() < 0.3, lse=rng.random() < 0.3)
        elif kind == "append":
            tokens = _log(rng, 1, 16384)
            case = dict(kind=kind, tokens=tokens, segments=min(tokens, _log(rng, 1, 64)), cut=rng.randrange(1000),
                        before=_log(rng, 1, 4096) - 1, kv_heads=kv_heads, head_dim=head_dim, page=page)
        else:
            longest = _log(rng, 16, 131072)
            keep = max(1, int(longest * rng.uniform(0.05, 0.9)))
            case = dict(kind=kind, batch=_log(rng, 1, 16), longest=longest, cut=rng.choice([-1, rng.randrange(1000)]),
                        keep=keep, recent=int(keep * rng.uniform(0, 0.5)), kv_heads=kv_heads, head_dim=head_dim,
                        page=page)
        cost = work(case)
        if kind == "decode" and 4 * case["batch"] * case["longest"] * kv_heads * head_dim > top["bytes"]:
            continue  # the plain form fills every sequence up to the longest
        if cost["bytes"] <= top["bytes"] and cost["flops"] <= top["flops"]:
            return case


def _cut(total, parts, cut):
    """`total` in `parts` lengths: equal ones (cut -1), or ragged by `cut`."""
    if cut < 0:
        return [total * (i + 1) // parts - total * i // parts for i in range(parts)]
    r = random.Random(cut)
    marks = sorted(r.randint(0, total) for _ in range(parts - 1))
    return [b - a for a, b in zip([0] + marks, marks + [total])]


def _lengths(case):
    """Slots of each sequence of a batch: all `longest`, or spread over its logarithm with one at `longest`."""
    n = case["longest"]
    if case["cut"] < 0:
        return [n] * case["batch"]
    r = random.Random(case["cut"])
    return [n] + [int(math.exp(r.uniform(0, math.log(n)))) for _ in range(case["batch"] - 1)]


def work(case):
    d, hk = case["head_dim"], case["kv_heads"]
    if case["kind"] == "prompt":
        lens = _cut(case["tokens"], case["segments"], case["cut"])
        p, h = case["prefix"], case["heads"]
        pairs = sum(n * p + n * (n + 1) // 2 for n in lens)
        keys = case["tokens"] + p * sum(n > 0 for n in lens)
        return {"bytes": 4 * case["tokens"] * h * d + 4 * keys * hk * d + 4 * case["lse"] * case["tokens"] * h,
                "flops": 4 * d * h * pairs}
    if case["kind"] == "append":
        return {"bytes": 8 * case["tokens"] * hk * d, "flops": 0}
    slots = sum(_lengths(case))
    if case["kind"] == "decode":
        h = case["heads"]
        return {"bytes": slots * hk * (4 * d + 4 * case["weights"]) + 4 * case["batch"] * h * d
                + 4 * case["lse"] * case["batch"] * h, "flops": 4 * d * h * slots}
    kept = sum(min(n, case["keep"]) for n in _lengths(case))
    return {"bytes": 4 * slots * hk + kept * hk * (8 * d + 8), "flops": slots * hk}


# ---------------------------------------------------------------------------------------------
# plain forms (32 bits)
# ---------------------------------------------------------------------------------------------

def _attend(q, k, v, mask):
    """(outputs, lse, probabilities) of q [..., rows, d] over k, v [..., keys, d]; mask True where a key is seen."""
    s = q @ k.transpose(-1, -2)
    s = s.mul_(1 / math.sqrt(q.shape[-1])).masked_fill_(~mask, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full((*s.shape[:-1], 1), -math.inf, device=s.device)
    p = torch.exp(s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    del s
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, torch.ones_like(total), total))
    return p @ v, (top + torch.log(total)).squeeze(-1), p


def _prompt_plain(s):
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    out = torch.empty((c["tokens"], h * d), dtype=BF16, device=DEV)
    lse = torch.empty((h, c["tokens"]), device=DEV)
    for (q0, q1), (k0, k1) in zip(zip(s["cu_q"], s["cu_q"][1:]), zip(s["cu_k"], s["cu_k"][1:])):
        nq, nk = q1 - q0, k1 - k0
        if nq == 0:
            continue
        q = s["q"][q0:q1].float().view(nq, hk, h // hk, d).permute(1, 2, 0, 3).reshape(hk, h // hk * nq, d)
        k, v = (s[n][k0:k1].float().view(nk, hk, d).transpose(0, 1).contiguous() for n in ("k", "v"))
        seen = torch.arange(nk, device=DEV)[None] <= torch.arange(nq, device=DEV)[:, None] + (nk - nq)
        o, e, _ = _attend(q, k, v, seen.repeat(h // hk, 1))
        out[q0:q1] = o.view(h, nq, d).transpose(0, 1).reshape(nq, h * d).to(BF16)
        lse[:, q0:q1] = e.reshape(h, nq)
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


def _slots(paged, table, n):
    """[batch, kv_heads, n, ...] of the first n slots of every sequence, from pages."""
    page = paged.shape[2]
    x = paged[table[:, :(n + page - 1) // page].clamp_min(0).long()]
    return x.transpose(1, 2).flatten(2, 3)[:, :, :n]


def _places(table, page, seq, slot):
    """(pages, slots in them) of slot `slot` of sequence `seq`, as index tensors."""
    return table.long()[seq, slot // page], slot % page


def _decode_plain(s):
    c = s["case"]
    b, h, hk, d, n = c["batch"], c["heads"], c["kv_heads"], c["head_dim"], c["longest"]
    k, v = _slots(s["k"], s["table"], n).float(), _slots(s["v"], s["table"], n).float()
    seen = torch.arange(n, device=DEV)[None] < s["lengths"][:, None]
    o, e, p = _attend(s["q"].float().view(b, hk, h // hk, d), k, v, seen[:, None, None])
    out = {"out": o.reshape(b, h * d).to(BF16)}
    if c["lse"]:
        out["lse"] = e.reshape(b, h)
    if c["weights"]:
        seq, slot = seen.nonzero(as_tuple=True)
        pages, places = _places(s["table"], c["page"], seq, slot)
        s["weights"][pages, :, places] = p.sum(2).transpose(1, 2)[seq, slot]
        out["weights"] = s["weights"]
    return out


def _append_plain(s):
    c = s["case"]
    counts = s["cu_dev"][1:] - s["cu_dev"][:-1]
    seq = torch.repeat_interleave(torch.arange(c["segments"], device=DEV), counts, output_size=c["tokens"])
    slot = torch.arange(c["tokens"], device=DEV) - s["cu_dev"][seq] + s["lengths"][seq]
    pages, places = _places(s["table"], c["page"], seq, slot)
    for cache, rows in ((s["k"], s["new_k"]), (s["v"], s["new_v"])):
        cache[pages, :, places] = rows.reshape(c["tokens"], c["kv_heads"], c["head_dim"])
    return {"k": s["k"], "v": s["v"], "lengths": s["lengths"] + counts}


def _evict_plain(s):
    c = s["case"]
    n, keep, hk = c["longest"], c["keep"], c["kv_heads"]
    w = _slots(s["weights"], s["table"], n).clone()
    at, lengths = torch.arange(n, device=DEV), s["lengths"][:, None, None]
    w.masked_fill_(at >= lengths - c["recent"], math.inf)
    w.masked_fill_(at >= lengths, -math.inf)
    order = torch.sort(w, dim=2, descending=True, stable=True).indices[:, :, :keep]
    new = s["lengths"].clamp_max(keep)
    order = order.masked_fill(torch.arange(order.shape[2], device=DEV) >= new[:, None, None], n).sort(2).values
    seq, head, j = (order < n).nonzero(as_tuple=True)
    to_page, to_slot = _places(s["out_table"], c["page"], seq, j)
    from_page, from_slot = _places(s["table"], c["page"], seq, order[seq, head, j])
    for cache in (s["k"], s["v"], s["weights"]):
        cache[to_page, head, to_slot] = cache[from_page, head, from_slot]
    return {"k": s["k"], "v": s["v"], "weights": s["weights"], "lengths": new}


# ---------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------

def _run_own(s):
    from ditserve_amd import kv, ops

    c = s["case"]
    if c["kind"] == "prompt":
        seg_q = ops.Segments(s["cu_q"], DEV, dev=s["cu_q_dev"])
        seg_k = ops.Segments(s["cu_k"], DEV, dev=s["cu_k_dev"])
        out = ops.flash_attn_causal(s["q"], s["k"], s["v"], seg_q, seg_k, c["heads"], c["kv_heads"], c["head_dim"],
                                    return_lse=c["lse"])
        return {"out": out[0], "lse": out[1]} if c["lse"] else {"out": out}
    cache = kv.PagedCache(s["k"], s["v"], s.get("weights"))
    if c["kind"] == "decode":
        out = kv.decode_attn(s["q"], cache, s["table"], s["lengths"], c["heads"], max_len=c["longest"],
                             weights="set" if c["weights"] else None, return_lse=c["lse"])
        out = {"out": out[0], "lse": out[1]} if c["lse"] else {"out": out}
        return {**out, "weights": cache.weights} if c["weights"] else out
    if c["kind"] == "append":
        segments = ops.Segments(s["cu"], DEV, dev=s["cu_dev"])
        lengths = kv.append(cache, s["new_k"], s["new_v"], s["table"], s["lengths"], segments)
        return {"k": cache.k, "v": cache.v, "lengths": lengths}
    lengths = kv.evict(cache, s["table"], s["lengths"], s["out_table"], c["keep"], recent=c["recent"],
                       max_len=c["longest"])
    return {"k": cache.k, "v": cache.v, "weights": cache.weights, "lengths": lengths}


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    return {"prompt": _prompt_plain, "decode": _decode_plain, "append": _append_plain, "evict": _evict_plain}[kind](state)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _keys(g, *shape):
    """Keys: each of a size of its own, and one in a hundred near its head's common direction, which queries like."""
    x = _normal(g, *shape) * torch.exp(0.3 * _normal(g, *shape[:-1], 1))
    return (x + 1.5 * (torch.rand((*shape[:-1], 1), generator=g, device=DEV) < 0.01)).to(BF16)


def _values(g, *shape):
    """Values around a mean of each channel."""
    return (_normal(g, *shape) + 0.5 * _normal(g, shape[-1])).to(BF16)


def _queries(g, *shape):
    return (_normal(g, *shape) + 0.2).to(BF16)


def _tables(case, lens, g, more=()):
    """(page tables of `lens` slots each, tables of `more` slots each, pages in all): pages in no order, a few unused."""
    page = case["page"]
    rows = [[(n + page - 1) // page for n in part] for part in (lens, more) if part]
    total = sum(map(sum, rows)) + 3
    order = torch.randperm(total, generator=g, device=DEV).int()
    out, used = [], 0
    for part in rows:
        wide = max(max(part), 1)
        counts = torch.tensor(part, device=DEV)
        first = torch.cumsum(counts, 0) - counts + used
        at = torch.arange(wide, device=DEV)
        ids = order[(first[:, None] + at).clamp_max(total - 1)]
        out.append(torch.where(at < counts[:, None], ids, -1).int())
        used += sum(part)
    return (*out, total)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    d, hk, kind = case["head_dim"], case["kv_heads"], case["kind"]
    if kind == "prompt":
        h, lens = case["heads"], _cut(case["tokens"], case["segments"], case["cut"])
        for name, counts in (("cu_q", lens), ("cu_k", [n + case["prefix"] * (n > 0) for n in lens])):
            cu = [0]
            for n in counts:
                cu.append(cu[-1] + n)
            s[name], s[name + "_dev"] = cu, torch.tensor(cu, dtype=torch.int32, device=DEV)
        rows = s["cu_k"][-1]
        # one projection's output where every key has its query
        both = torch.empty((rows, (h + 2 * hk) * d), dtype=BF16, device=DEV) if not case["prefix"] else None
        if both is not None:
            s["q"], s["k"], s["v"] = both.split([h * d, hk * d, hk * d], 1)
        else:
            s["q"] = torch.empty((case["tokens"], h * d), dtype=BF16, device=DEV)
            s["k"], s["v"] = torch.empty((2, rows, hk * d), dtype=BF16, device=DEV).unbind(0)
        s["q"].copy_(_queries(g, case["tokens"], h, d).flatten(1))
        s["k"].copy_(_keys(g, rows, hk, d).flatten(1))
        s["v"].copy_(_values(g, rows, hk, d).flatten(1))
        return s
    if kind == "append":
        counts = _cut(case["tokens"], case["segments"], case["cut"])
        r = random.Random(case["cut"])
        before = [case["before"] if case["cut"] < 0 else r.randint(0, case["before"]) for _ in counts]
        s["table"], pages = _tables(case, [a + b for a, b in zip(before, counts)], g)
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        s["cu"], s["cu_dev"] = cu, torch.tensor(cu, dtype=torch.int32, device=DEV)
        s["new_k"], s["new_v"] = _keys(g, case["tokens"], 2, hk, d).flatten(2).unbind(1)
        lens = before
    else:
        lens = _lengths(case)
        if kind == "decode":
            s["q"] = _queries(g, case["batch"], case["heads"], d).flatten(1)
            s["table"], pages = _tables(case, lens, g)
        else:
            s["table"], s["out_table"], pages = _tables(case, lens, g, [min(n, case["keep"]) for n in lens])
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    shape = (pages, hk, case["page"])
    s["k"], s["v"] = _keys(g, *shape, d), _values(g, *shape, d)
    if kind == "evict":
        # sums of probabilities: few large ones, many small ones, and ties where fp32 holds no difference
        w = torch.exp(2 * _normal(g, *shape) - 6)
        s["weights"] = torch.where(w < 0.002, torch.round(w * 4096) / 4096, w)
    elif case.get("weights"):
        s["weights"] = torch.zeros(shape, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------

def _softmax64(q, k, v, hidden):
    """Rows of q over the keys; hidden: how many of the last keys each row does not see, or None."""
    s = torch.mm(q, k.t()) / k.shape[1] ** 0.5
    if hidden is not None:
        s[torch.arange(k.shape[0], device=DEV)[None] >= k.shape[0] - hidden[:, None]] = -math.inf
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    return torch.mm(p, v), lse, p


def _of_pages(paged, table, n):
    """[kv_heads, n, ...] in 64 bits of one sequence's first n slots."""
    page = paged.shape[2]
    parts = paged.index_select(0, table[:-(-n // page)])
    return torch.cat(list(parts.double()), 1)[:, :n]


def exact(case, seed):
    s = prepare(case, seed)
    d, hk = case["head_dim"], case["kv_heads"]
    if case["kind"] == "prompt":
        h = case["heads"]
        out = torch.zeros((case["tokens"], h * d), dtype=torch.float64, device=DEV)
        lse = torch.zeros((h, case["tokens"]), dtype=torch.float64, device=DEV)
        for m in range(case["segments"]):
            rows, keys = slice(*s["cu_q"][m:m + 2]), slice(*s["cu_k"][m:m + 2])
            nq = rows.stop - rows.start
            for i in range(h if nq else 0):
                a, b = slice(i * d, i * d + d), slice(i * hk // h * d, i * hk // h * d + d)
                out[rows, a], lse[i, rows], _ = _softmax64(
                    s["q"][rows, a].double(), s["k"][keys, b].double(), s["v"][keys, b].double(),
                    torch.arange(nq - 1, -1, -1, device=DEV))
        return {"out": out, "lse": lse} if case["lse"] else {"out": out}
    page, lens = case["page"], s["lengths"].tolist()
    if case["kind"] == "decode":
        h, group = case["heads"], case["heads"] // hk
        out = torch.zeros((case["batch"], h, d), dtype=torch.float64, device=DEV)
        lse = torch.full((case["batch"], h), -math.inf, dtype=torch.float64, device=DEV)
        weights = s["weights"].double() if case["weights"] else None
        for b, n in enumerate(lens):
            k, v = _of_pages(s["k"], s["table"][b], n), _of_pages(s["v"], s["table"][b], n)
            for i in range(hk if n else 0):
                mine = slice(i * group, i * group + group)
                q = s["q"][b].double().view(h, d)[mine]
                out[b, mine], lse[b, mine], p = _softmax64(q, k[i], v[i], None)
                if weights is not None:
                    flat = torch.zeros(-(-n // page) * page, dtype=torch.float64, device=DEV)
                    flat[:n] = p.sum(0)
                    whole = n // page
                    weights[s["table"][b, :whole].long(), i] = flat[:whole * page].view(whole, page)
                    if n % page:
                        weights[int(s["table"][b, whole]), i, :n % page] = flat[whole * page:n]
        got = {"out": out.flatten(1)}
        if case["lse"]:
            got["lse"] = lse
        return got if weights is None else {**got, "weights": weights}
    k, v = s["k"].double(), s["v"].double()
    if case["kind"] == "append":
        new_k, new_v = s["new_k"].double().unflatten(1, (hk, d)), s["new_v"].double().unflatten(1, (hk, d))
        table = s["table"].tolist()
        for m in range(case["segments"]):
            done, last = 0, s["cu"][m + 1] - s["cu"][m]
            while done < last:  # page by page
                at = lens[m] + done
                n = min(page - at % page, last - done)
                rows = slice(s["cu"][m] + done, s["cu"][m] + done + n)
                k[table[m][at // page], :, at % page:at % page + n] = new_k[rows].transpose(0, 1)
                v[table[m][at // page], :, at % page:at % page + n] = new_v[rows].transpose(0, 1)
                done += n
        return {"k": k, "v": v, "lengths": None}
    weights = s["weights"].double()
    for b, n in enumerate(lens):
        m = min(n, case["keep"])
        recent = min(case["recent"], m)
        w = _of_pages(s["weights"], s["table"][b], n)
        for i in range(hk):
            # the lowest slots first among equal weights: by weight, then by slot
            old = w[i, :n - recent]
            by_slot = torch.argsort(old, descending=True, stable=True)[:m - recent]
            slots = torch.cat([by_slot.sort().values, torch.arange(n - recent, n, device=DEV)])
            j = torch.arange(m, device=DEV)
            src, dst = s["table"][b].long()[slots // page], s["out_table"][b].long()[j // page]
            for cache in (k, v, weights):
                cache[dst, i, j % page] = cache[src, i, slots % page]
    return {"k": k, "v": v, "weights": weights, "lengths": None}
