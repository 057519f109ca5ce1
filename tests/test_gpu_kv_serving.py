"""Prompts, cache, single tokens and eviction together, as a serving loop runs them: eagerly, captured, on two streams."""
import pytest
import torch

from tests.kv_reference import DEV, attend64, check_out, errors32, get

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from ditserve_amd import kv, ops

HEADS, HK, D, PAGE = 10, 2, 64, 16


class Plain:
    """The same loop on lists of keys, values and weights, the sums in 64 bits."""

    def __init__(self, batch):
        self.k = [torch.empty((0, HK, D), dtype=torch.bfloat16, device=DEV) for _ in range(batch)]
        self.v = [x.clone() for x in self.k]
        self.w = [torch.zeros((0, HK), dtype=torch.float64, device=DEV) for _ in range(batch)]
        self.rel = 0.0  # what the weights may be off by now, relative

    def append(self, b, k, v):
        self.k[b] = torch.cat([self.k[b], k.reshape(-1, HK, D)])
        self.v[b] = torch.cat([self.v[b], v.reshape(-1, HK, D)])
        self.w[b] = torch.cat([self.w[b], torch.zeros((k.shape[0], HK), dtype=torch.float64, device=DEV)])

    def step(self, q, out):
        for b in range(len(self.k)):
            n = self.k[b].shape[0]
            want, _, p, mass, size = attend64(q[b].view(HEADS, 1, D), self.k[b].transpose(0, 1), self.v[b].transpose(0, 1))
            _, rel = errors32(D, n, size)
            check_out(out[b].view(HEADS, D), want[:, 0], mass[:, 0], rel)
            self.w[b] += p[:, 0].view(HK, HEADS // HK, n).sum(1).t()
            self.rel = max(self.rel, 2 * rel + 2.0 ** -19 + (HEADS // HK + 1) * 2.0 ** -24)

    def check(self, cache, table):
        for b, w in enumerate(self.w):
            n = w.shape[0]
            assert torch.equal(get(cache.k, table[b], n), self.k[b]) and torch.equal(get(cache.v, table[b], n), self.v[b])
            assert bool(((get(cache.weights, table[b], n) - w).abs() <= 3 * self.rel * w + 2.0 ** -126).all())

    def evict(self, cache, table, keep, recent):
        """By the cache's own weights (sums in 32 bits decide)."""
        for b in range(len(self.k)):
            n = self.k[b].shape[0]
            w, m = get(cache.weights, table[b], n), min(n, keep)
            r = min(recent, m)
            new = []
            for h in range(HK):
                old = torch.sort(w[:n - r, h], descending=True, stable=True).indices[:m - r].sort().values
                at = torch.cat([old, torch.arange(n - r, n, device=DEV)])
                new.append((self.k[b][at, h], self.v[b][at, h], self.w[b][at, h]))
            self.k[b], self.v[b], self.w[b] = (torch.stack([x[i] for x in new], 1) for i in range(3))


def pages_of(tables, counts, g, total):
    order = torch.randperm(total, generator=g).int()
    out, at = [], 0
    for batch, n in counts:
        out.append(order[at:at + batch * n].view(batch, n).to(DEV))
        at += batch * n
    return out


def rows(n, heads, g):
    return torch.randn((n, heads * D), generator=g).bfloat16().to(DEV)


def test_a_serving_loop():
    g = torch.Generator().manual_seed(1)
    lens = [37, 600, 1, 260]
    cache = kv.PagedCache.empty(400, HK, D, PAGE, DEV)
    cache.weights.fill_(float("nan"))
    table, second = pages_of(None, [(4, 42), (4, 20)], g, 400)
    plain = Plain(4)
    cu = [0, 37, 637, 638, 898]
    seg = ops.Segments(cu, DEV)
    qkv = rows(898, HEADS + 2 * HK, g)
    q, k, v = qkv.split([HEADS * D, HK * D, HK * D], 1)
    out = ops.flash_attn_causal(q, k, v, seg, seg, HEADS, HK, D)
    lengths = kv.append(cache, k, v, table, torch.zeros(4, dtype=torch.int32, device=DEV), seg)
    for b in range(4):
        plain.append(b, k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]])
        # the last prompt token's attention is that of a single token over the cache
        last = cu[b + 1] - 1
        want, _, _, mass, size = attend64(q[last].view(HEADS, 1, D), plain.k[b].transpose(0, 1), plain.v[b].transpose(0, 1))
        check_out(out[last].view(HEADS, D), want[:, 0], mass[:, 0], errors32(D, lens[b], size)[1], p_bits=8)
    for i in range(12):
        if i == 6:
            old = table
            lengths = kv.evict(cache, old, lengths, second, keep=300, recent=20)
            plain.evict(cache, old, 300, 20)
            table = second
        new_k, new_v, q = rows(4, HK, g), rows(4, HK, g), rows(4, HEADS, g)
        lengths = kv.append(cache, new_k, new_v, table, lengths)
        for b in range(4):
            plain.append(b, new_k[b:b + 1], new_v[b:b + 1])
        o = kv.decode_attn(q, cache, table, lengths, HEADS, max_len=660, weights="add")
        plain.step(q, o)
        plain.check(cache, table)
    kv.check_tables()
    assert lengths.tolist() == [49, 306, 13, 272]


def step_of(cache, table, lengths, q, k, v, max_len, out):
    new = kv.append(cache, k, v, table, lengths)
    kv.decode_attn(q, cache, table, new, HEADS, max_len=max_len, weights="add", out=out)
    lengths.copy_(new)


def caches(n, lens, g, total=300):
    """n equal caches with the same filled slots."""
    table, = pages_of(None, [(len(lens), 60)], g, total)
    first = kv.PagedCache.empty(total, HK, D, PAGE, DEV)
    first.weights.zero_()
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    k, v = rows(cu[-1], HK, g), rows(cu[-1], HK, g)
    lengths = kv.append(first, k, v, table, torch.zeros(len(lens), dtype=torch.int32, device=DEV), ops.Segments(cu, DEV))
    all_ = [first] + [kv.PagedCache(first.k.clone(), first.v.clone(), first.weights.clone()) for _ in range(n - 1)]
    return all_, table, lengths


@pytest.mark.parametrize("max_len", [400, 960])  # one launch, and parts with a join
def test_captured_steps(max_len):
    """Two graphs of a step each on a cache of its own, replayed in turn with eager work between: bitwise the eager steps."""
    g = torch.Generator().manual_seed(2)
    (a, b, c), table, lengths = caches(3, [300, 17, 0, 129], g)
    q, k, v = rows(4, HEADS, g), rows(4, HK, g), rows(4, HK, g)
    ins = [[t.clone() for t in (lengths, q, k, v)] for _ in range(3)]
    outs = [torch.empty_like(q) for _ in range(3)]
    graphs = []
    for cache, (n, *x), out in zip((a, b), ins, outs):
        graph = torch.cuda.CUDAGraph()
        saved = [t.clone() for t in (cache.k, cache.v, cache.weights, n)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step_of(cache, table, n, *x, max_len, out)
        torch.cuda.current_stream().wait_stream(s)
        for t, old in zip((cache.k, cache.v, cache.weights, n), saved):
            t.copy_(old)
        with torch.cuda.graph(graph):
            step_of(cache, table, n, *x, max_len, out)
        graphs.append(graph)
    for i in range(5):
        fresh = rows(4, HEADS, g), rows(4, HK, g), rows(4, HK, g)
        for x in ins:
            for t, new in zip(x[1:], fresh):
                t.copy_(new)
        step_of(c, table, ins[2][0], *ins[2][1:], max_len, outs[2])
        junk = torch.randn((1 << 20,), device=DEV).sort()  # work between, in memory of its own
        for graph in graphs:
            graph.replay()
        del junk
        torch.cuda.synchronize()
        for cache, x, out in zip((a, b), ins, outs):
            assert torch.equal(out, outs[2]) and torch.equal(x[0], ins[2][0])
            for t, ref in ((cache.k, c.k), (cache.v, c.v), (cache.weights, c.weights)):
                assert torch.equal(t.view(torch.int16), ref.view(torch.int16))
    kv.check_tables()


def test_captured_prompts_and_eviction():
    g = torch.Generator().manual_seed(3)
    (cache,), table, lengths = caches(1, [500, 40, 3], g)
    cache.weights.copy_(torch.rand(cache.weights.shape, generator=g))
    used = set(table.flatten().tolist())
    free = torch.tensor([p for p in range(300) if p not in used][:90], dtype=torch.int32).view(3, 30).to(DEV)
    segs = ops.Segments([0, 300, 340], DEV), ops.Segments([0, 300, 1640], DEV)  # the second: few queries over many keys
    q, k, v = rows(340, HEADS, g), rows(1640, HK, g), rows(1640, HK, g)

    def work():
        return (*ops.flash_attn_causal(q, k, v, *segs, HEADS, HK, D, return_lse=True),
                kv.evict(cache, table, lengths, free, keep=450, recent=7))
    def clear():
        for t in (cache.k, cache.v, cache.weights):
            t[free.flatten().long()] = 0
    clear()
    want = [t.clone() for t in work()]
    kept = [t.clone() for t in (cache.k, cache.v, cache.weights)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for i in range(4):
        clear()
        got[0].zero_()
        torch.randn((1 << 20,), device=DEV).sort()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip((cache.k, cache.v, cache.weights), kept))


def test_two_streams():
    """Calls of two streams at once, on caches of their own and over one that both read: bitwise the calls in turn."""
    g = torch.Generator().manual_seed(4)
    lens = [900, 33, 512, 700]
    (a, b, shared), table, lengths = caches(3, lens, g)
    q = [rows(4, HEADS, g) for _ in range(2)]
    seg = ops.Segments([0, 200, 340], DEV)
    prompt = [[rows(340, h, g) for h in (HEADS, HK, HK)] for _ in range(2)]

    def work(i, cache):
        o = kv.decode_attn(q[i], cache, table, lengths, HEADS, weights="set")
        r = kv.decode_attn(q[i], shared, table, lengths, HEADS)
        return [o, r, cache.weights.clone(), ops.flash_attn_causal(*prompt[i], seg, seg, HEADS, HK, D)]
    want = [work(i, c) for i, c in enumerate((a, b))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = []
        for i, (s, c) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got.append(work(i, c))
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert all(torch.equal(s.view(torch.int16), t.view(torch.int16)) for s, t in zip(x, y))
