"""Refusals of the paged cache's entry points: on the host, before any launch (no GPU)."""
import pytest
import torch

from ditserve_amd import _lib, kv

if not _lib.LIB_PATH.exists():
    pytest.skip("libditk.so not built (run python -m ditserve_amd.build)", allow_module_level=True)

A, B, C, D, E, F, G, H = (0x10000 * i for i in range(1, 9))  # addresses only: nothing is launched


def refused(name, args, word):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1
    assert word in lib.ditk_last_error().decode(), lib.ditk_last_error()


CACHE = dict(k=A, k_ps=2 * 16 * 64, k_hs=16 * 64, v=B, v_ps=2 * 16 * 64, v_hs=16 * 64, w=None, w_ps=32, w_hs=16)
PAGES = dict(pages=8, page=16, table=C, ldt=4, width=4, lengths=D)
APPEND = dict(new_k=E, ldk=128, new_v=F, ldv=128, **CACHE, **PAGES, new=G, cu=None, batch=2, T=2, hk=2, d=64, status=H,
              stream=None)
ATTN = dict(q=E, ldq=256, **CACHE, add=0, **PAGES, max_len=64, o=F, ldo=256, lse=None, space=None, size=0, batch=2, heads=4,
            hk=2, d=64, scale=0.1, status=H, stream=None)
EVICT = dict(**{**CACHE, "w": E}, **PAGES, max_len=64, out_table=F, ldo=2, out_width=2, new=G, keep=32, recent=4, space=A,
             size=1 << 20, batch=2, hk=2, d=64, status=H, stream=None)

COMMON = [
    (dict(batch=-1), "sequences"), (dict(batch=65536), "sequences"), (dict(hk=0), "key head"), (dict(d=96), "head_dim"),
    (dict(page=8), "slots"), (dict(page=48), "slots"), (dict(pages=0), "no pages"), (dict(table=None), "null table"),
    (dict(lengths=None), "null table"), (dict(status=None), "null table"), (dict(ldt=3), "page table"),
    (dict(width=-1), "page table"), (dict(width=2**26, ldt=2**26), "page table"), (dict(k=None), "null cache"),
    (dict(v=None), "null cache"), (dict(k=A + 8), "aligned"), (dict(v_hs=1028), "aligned"), (dict(k_ps=-2048), "aligned")]


@pytest.mark.parametrize("change,word", COMMON + [
    (dict(new_k=None), "rows"), (dict(T=-1), "rows"), (dict(T=3), "3 rows for 2"), (dict(ldk=120), "aligned"),
    (dict(ldv=132), "aligned"), (dict(new_v=F + 2), "aligned"), (dict(new=None), "lengths")])
def test_append_refuses(change, word):
    refused("ditk_kv_append", tuple({**APPEND, **change}.values()), word)


@pytest.mark.parametrize("change,word", COMMON + [
    (dict(heads=5), "query heads"), (dict(heads=0), "query heads"), (dict(q=None), "null"), (dict(o=None), "null"),
    (dict(ldq=252), "aligned"), (dict(o=F + 8), "aligned"), (dict(max_len=-1), "max_len"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(w=G), "workspace"),
    (dict(width=4096, ldt=4096, max_len=65536, space=G, size=64), "workspace"),
    (dict(batch=65535, heads=128, ldq=8192, ldo=8192), "too many")])
def test_attn_refuses(change, word):
    refused("ditk_kv_attn", tuple({**ATTN, **change}.values()), word)


@pytest.mark.parametrize("change,word", COMMON + [
    (dict(w=None), "no weights"), (dict(w_ps=1 << 32), "too far"), (dict(keep=0), "keep"), (dict(recent=-1), "recent"), (dict(recent=33), "recent"),
    (dict(max_len=-1), "max_len"), (dict(out_table=None), "null table"), (dict(out_width=1), "32 stay"),
    (dict(new=None), "null output"), (dict(space=None), "null output"), (dict(space=A + 8), "null output"),
    (dict(size=4 * 2 * 2 * 32 - 4), "workspace"), (dict(width=4096, ldt=4096, max_len=65536, size=1 << 18), "workspace")])
def test_evict_refuses(change, word):
    refused("ditk_kv_evict", tuple({**EVICT, **change}.values()), word)


def test_nothing_to_do():
    """No sequences: no launch."""
    lib = _lib.load()
    none = dict(batch=0, table=None, lengths=None)
    assert lib.ditk_kv_append(*{**APPEND, **none, "T": 0, "new": None}.values()) == 0
    assert lib.ditk_kv_attn(*{**ATTN, **none}.values()) == 0
    assert lib.ditk_kv_evict(*{**EVICT, **none, "new": None}.values()) == 0


def test_workspace_grows_with_what_it_holds():
    size = _lib.load().ditk_kv_attn_workspace
    assert size(4, 8, 128, 64, 0) == 0 and size(0, 8, 128, 1 << 20, 1) == 0
    assert size(4, 8, 128, 1 << 20, 0) < size(4, 8, 128, 1 << 20, 1)
    # a float for each query head and slot, past 32 bits
    assert size(64, 128, 128, 1 << 20, 1) > 64 * 128 * (1 << 20) * 4


def test_cpu_tensors_are_refused():
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="cuda"):
        kv.PagedCache(k, k)
    with pytest.raises(ValueError, match="PagedCache"):
        kv.append(k, k, k, k, k)
    with pytest.raises(ValueError, match="PagedCache"):
        kv.decode_attn(k, k, k, k, 2)
    with pytest.raises(ValueError, match="PagedCache"):
        kv.evict(k, k, k, k, 2)


@pytest.mark.parametrize("pages,heads,ps,hs,size", [
    (1, 1, 0, 0, 8), (4, 1, 8, 3, 8), (4, 1, 7, 0, 8), (1, 3, 0, 16, 8), (3, 2, 16, 8, 8), (3, 2, 8, 24, 8), (3, 2, 8, 16, 8),
    (3, 4, 40, 8, 8), (3, 4, 24, 8, 8), (2, 3, 100, 16, 8), (5, 2, 8, 8, 8), (2, 2, 64, 32, 8)])
def test_overlapping_blocks(pages, heads, ps, hs, size):
    """What is said of the blocks of one cache, and of two, is what counting their elements says."""
    starts = [i * ps + j * hs for i in range(pages) for j in range(heads)]
    cells = [x + i for x in starts for i in range(size)]
    span = kv._span(pages, heads, ps, hs, size)
    if span == 0:
        assert len(set(cells)) < len(cells)
        return
    assert len(set(cells)) == len(cells) and span == max(cells) + 1
    for delta in range(-max(cells) - 2, max(cells) + 3):
        assert kv._meet_blocks(delta, pages, heads, ps, hs, size) == any(x + delta in set(cells) for x in cells), delta


CAUSAL = dict(q=A, ldq=256, k=B, ldk=128, v=G, ldv=128, o=D, ldo=256, lse=None, lse_ld=0, cu_q=E, cu_k=F, nseg=1, Tq=64,
              Tk=64, heads=4, hk=2, d=64, scale=0.1, kinds=3, space=H,
              size=1 << 20, parts=8, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(kinds=0), "kinds"), (dict(kinds=4), "kinds"), (dict(nseg=1 << 22, Tk=2000), "too many"),
    (dict(Tk=2000, space=None), "workspace"), (dict(Tk=2000, space=H + 8), "workspace"), (dict(Tk=2000, parts=0), "workspace"),
    (dict(Tk=2000, size=8 * 2 * 66 * 4 - 1), "workspace"),
    (dict(scale=0.0), "softmax_scale"), (dict(scale=float("inf")), "softmax_scale"), (dict(cu_q=None), "null"),
    (dict(q=None), "null"), (dict(d=96), "head_dim"), (dict(nseg=0), "sizes"), (dict(Tk=-1), "sizes"),
    (dict(Tq=1 << 30), "sizes"), (dict(heads=3), "query heads"), (dict(hk=0), "query heads"), (dict(ldq=252), "leading"),
    (dict(ldv=124), "leading"), (dict(v=None), "null"), (dict(v=G + 2), "misaligned"), (dict(q=A + 8), "misaligned"), (dict(o=D + 8), "misaligned"),
    (dict(ldk=1 << 23), "32-bit"), (dict(ldv=1 << 23), "32-bit"), (dict(ldo=1 << 30), "32-bit"), (dict(Tq=(1 << 30) - 1), "grid")])
def test_causal_refuses(change, word):
    refused("ditk_flash_attn_causal", tuple({**CAUSAL, **change}.values()), word)
