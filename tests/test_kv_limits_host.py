"""Further checks of the paged cache's and the device tables' entry points, before any launch (no GPU)."""
import random

import pytest
import torch

from ditserve_amd import _lib, attention, kv, ops

if not _lib.LIB_PATH.exists():
    pytest.skip("libditk.so not built (run python -m ditserve_amd.build)", allow_module_level=True)

from tests.test_kv_host import APPEND, ATTN, CAUSAL, EVICT, G, refused  # noqa: E402


@pytest.mark.parametrize("scale", [1e-31, 1e31, 1e39, float("inf"), -1.0])
def test_attn_refuses_scales_beyond_fp32(scale):
    """Scores are scaled in fp32: a scale that is no number there, or near its ends, is refused, as for prompts."""
    refused("ditk_kv_attn", tuple({**ATTN, "scale": scale}.values()), "softmax_scale")


@pytest.mark.parametrize("change", [dict(ldq=128), dict(ldo=248), dict(ldq=-256), dict(ldo=-256), dict(ldo=0)])
def test_attn_refuses_rows_that_overlap(change):
    refused("ditk_kv_attn", tuple({**ATTN, **change}.values()), "rows")


@pytest.mark.parametrize("ldo", [0, 128, 248])
def test_causal_refuses_rows_that_overlap(ldo):
    refused("ditk_flash_attn_causal", tuple({**CAUSAL, "ldo": ldo}.values()), "rows of o")


@pytest.mark.parametrize("change", [dict(w=G + 2), dict(w=G, w_hs=-16), dict(w=G, w_ps=-32)])
@pytest.mark.parametrize("name,args", [
    ("ditk_kv_append", APPEND), ("ditk_kv_attn", {**ATTN, "space": G, "size": 1 << 20}), ("ditk_kv_evict", EVICT)])
def test_weights_are_checked(name, args, change):
    refused(name, tuple({**args, **change}.values()), "weights")


def test_blocks_of_two_tensors():
    """Whether keys or values and weights share a byte: never missed, and exact where both have the same order and strides or
    the same stride of pages with contiguous heads."""
    r = random.Random(1)
    seen = [0, 0]  # cases that do not meet, and that do
    for _ in range(1200):
        pages, heads = r.randint(1, 4), r.randint(1, 3)
        sizes = [r.randint(1, 6), r.randint(1, 6)]
        exact = True
        kind = r.randrange(3)
        if kind == 0:  # the same strides, pages or heads outside
            inner, outside = max(sizes) + r.randint(0, 9), r.random() < 0.5
            outer = inner * (heads if outside else pages) + r.randint(0, 20)
            strides = [(outer, inner) if outside else (inner, outer)] * 2
        elif kind == 1:  # the same outer stride, insides contiguous
            outer = sum(sizes) * heads + r.randint(0, 20)
            strides = [(outer, sizes[0]), (outer, sizes[1])]
        else:
            exact = False
            strides = [(sizes[i] * heads + r.randint(0, 5), sizes[i]) for i in range(2)]
        a, b = [(pages, heads, *st, size) for st, size in zip(strides, sizes)]
        if not kv._span(*a) or not kv._span(*b):
            continue
        cells = [{i * ps + j * hs + e for i in range(p) for j in range(h) for e in range(n)} for p, h, ps, hs, n in (a, b)]
        far = max(map(max, cells)) + 2
        for delta in range(-far, far + 1, r.randint(1, 3)):
            want = any(x + delta in cells[0] for x in cells[1])
            got = kv._blocks_meet(delta, a, b)
            assert got or not want, (delta, a, b)
            if exact:
                assert got == want, (delta, a, b)
                seen[want] += 1
    assert min(seen) > 1000


class Table:
    """A device table, as far as the host looks at one."""

    def __init__(self, device, n=3):
        self.device, self.n, self.dtype = torch.device(device), n, torch.int32

    def dim(self):
        return 1

    def numel(self):
        return self.n

    def to(self, dtype):
        return self

    def contiguous(self):
        return self

    def data_ptr(self):
        return 0


def test_tables_on_two_devices_are_refused(monkeypatch):
    """The check of a pair of tables is one launch: both have to be on one device, the rows' own."""
    def launched(*args):
        raise AssertionError("launched")
    for name in ("_call", "table_status"):
        monkeypatch.setattr(ops, name, launched)
    monkeypatch.setattr(ops._lib, "call", launched)
    with pytest.raises(ValueError, match="cu_seqlens"):
        ops.Segments.pair_from_device(Table("cuda:0"), 8, Table("cuda:1"), 8)
    rows = torch.zeros((8, 2, 64), dtype=torch.bfloat16)  # (rows on the host)
    for q, k in (("cuda:0", "cuda:1"), ("cuda:1", "cuda:0"), ("cuda:0", "cuda:0")):
        with pytest.raises(ValueError):
            attention.causal_attn_varlen_func(rows, rows, rows, Table(q), Table(k), 8, 8)


def test_tables_are_checked_on_their_device(monkeypatch):
    """The launch goes to the tables' device, which need not be the current one."""
    seen = []

    class Status:
        host = torch.zeros(1, dtype=torch.int32)

        def poll(self):
            pass

    empty = torch.empty
    monkeypatch.setattr(ops, "table_status", lambda device: Status())
    monkeypatch.setattr(ops, "_call", lambda device, name, *args: seen.append((str(device), name)))
    monkeypatch.setattr(ops.torch, "empty", lambda *a, device=None, **kw: empty(*a, **kw))
    monkeypatch.setattr(ops.torch, "empty_like", lambda t, **kw: empty(t.numel(), dtype=t.dtype))
    ops.Segments.pair_from_device(Table("cuda:1"), 8, Table("cuda:1"), 8)
    ops.Segments.from_device(Table("cuda:1"), 8)
    assert seen == [("cuda:1", "ditk_check_cu_seqlens_pair"), ("cuda:1", "ditk_check_cu_seqlens")]
