"""Generate the main loop of the one-wave-per-SIMD MX product (mx_gemm.hip:
mx_gemm_l4) as gfx950 assembly, for each of its wave tiles.

The workgroup computes a tile of C^T = W A^T with four waves, one per SIMD, each
owning a wave tile of 16 FI features x 16 FJ tokens: FI x FJ accumulator tiles of
v_mfma_scale_f32_16x16x128_f8f6f4 (256 accumulators, all of the AGPRs, at 128 x
128), handed to the C++ epilogue as they are.  An operand fragment is 8 VGPRs, so
two full operand sets do not fit beside the addresses: the W fragments have two
sets, the token fragments four buffers that a stage's FJ columns take in turn.

  AGPR a[4 (i FJ + j)..]    acc[i][j]: features 16 i + 4 (lane / 16) + e, token 16 j + lane % 16
  VGPR W[p][i]              W fragments, set p = stage % 2
  VGPR X[b]                 token fragments, column j in b = j % NX
  VGPR S[q][..]             scales of 4 stages (a byte each), set q = (stage / 4) % 2
  VGPR 4 addresses          this stage's fragment reads
  SGPR s40..s63             loop state

K advances in 128-k stages through NBUF LDS buffers (A rows, then W rows, 128 bytes
each, 16-byte units XOR-swizzled by row) filled by direct global->LDS DMA.  A stage is
FI x FJ MFMAs of 32 cycles, column by column.  Its token fragments 1 .. FJ - 1 are read
as their buffers come free; then one barrier (this wave's reads of the stage and
its DMA of the next landed), behind which the DMA of stage s + NBUF fills the stage's
own buffer and the next stage's W fragments and first token fragment are read.

The stages of a workgroup's tiles are one stream: behind a tile's last stages the
DMA goes on with the next tile's first, so that its operands are there when the
epilogue ends.  The scales are 16 bytes a row and 4 stages; their DMA comes with every
fourth stage and a tile's first, out of line, to two buffers in turn.

Usage: python gen_mx_gemm.py [dir/any]  (writes mx_l4_<tokens>x<features>_body.inc, its
prologue mx_l4_<tokens>x<features>_start.inc and mx_l4_clobbers.h into that directory, default beside
this file)
"""
import os
import sys

# the generated wave tiles: (feature fragments, token fragments, stage buffers, slot of the
# barrier, slot of W's barrier if it has one of its own)
VARIANTS = [(8, 8, 2, 40, 8), (8, 4, 3, 8, None), (4, 4, 4, 7, None), (4, 2, 4, 4, None)]


def name_of(fi, fj):
    return f"mx_l4_{32 * fj}x{32 * fi}"


def configure(fi, fj, nbuf, bar, wbar):
    global FI, FJ, NBUF, BAR, WBAR, NX, WOFF, BUF, ROWS, ND, WB, XB, SB, AB, LAST_VGPR
    FI, FJ, NBUF, BAR, WBAR = fi, fj, nbuf, bar, wbar
    WOFF = 32 * fj * 128
    ROWS = 32 * (fi + fj)
    BUF = ROWS * 128
    ND = fi + fj
    NX = min(4, fj)                       # token fragment buffers
    WB = 0
    XB = WB + 2 * fi * 8
    SB = XB + NX * 8
    AB = SB + 2 * (fi + fj)      # addresses: x chunk 0, 1, w chunk 0, 1, x and w scales
    LAST_VGPR = AB + 5
    # (NBUF <= 4: the scales have two buffers)
    assert fj % NX == 0 and nbuf <= 4 and nbuf * BUF + 2 * ROWS * 16 <= 160 * 1024


# loop state
S_A, S_W = 40, 42        # the DMA's sources: A and W of the stage it is at
S_SA, S_SW = 44, 46      # and of the scale group
S_S, S_NK1 = 48, 49      # stage, last stage
S_T = 50                 # the stage the DMA is at
S_RD, S_WR = 51, 52      # buffer offsets: of the next stage to read, of the DMA (LDS address of this wave's slice)
S_SCN = 53               # the stage at which the scales are due
S_SCP = 54               # LDS offset of the scale buffer they go to
S_T0 = 55
S_OFF = 56               # buffer offset of the DMA
S_SCR = 57               # LDS offset of the scale buffer to read next
SGPRS = list(range(40, 58))


def acc(i, j):
    return (i * FJ + j) * 4


def wreg(p, i):
    return WB + (p * FI + i) * 8


def xreg(j):
    return XB + (j % NX) * 8


def swreg(q, i):
    return SB + q * (FI + FJ) + i


def sxreg(q, j):
    return SB + q * (FI + FJ) + FI + j


class Gen:
    def __init__(self):
        self.lines, self.label_n, self.tails = [], 0, []

    def __call__(self, s):
        self.lines.append(s)

    def label(self, name):
        self.lines.append(f"{name}:")

    def new_label(self, stem):
        self.label_n += 1
        return f"L_{stem}_{self.label_n}_%="


def wrap(g, reg):
    """Buffer offset reg += BUF, modulo the ring."""
    g(f"s_add_u32 s{reg}, s{reg}, {BUF}")
    g(f"s_cmp_eq_u32 s{reg}, {NBUF * BUF}")
    g(f"s_cselect_b32 s{reg}, 0, s{reg}")


def dma_m0(g, k):
    """DMA instruction k of this wave (FJ of A, then FI of W) into the buffer at S_WR."""
    g(f"s_add_u32 m0, s{S_WR}, {WOFF + (k - FJ) * 4096 if k >= FJ else k * 4096}")


def dma_go(g, k):
    if k < FJ:
        g(f"global_load_lds_dwordx4 %[aoff{k}], s[{S_A}:{S_A + 1}]")
    else:
        g(f"global_load_lds_dwordx4 %[woff{k - FJ}], s[{S_W}:{S_W + 1}]")


def scale_dma(g):
    """The scale group at S_SA / S_SW into the scale buffer at S_SCP."""
    g(f"s_add_u32 m0, %[scm_a], s{S_SCP}")
    g("s_nop 0")
    g(f"global_load_lds_dwordx4 %[saoff], s[{S_SA}:{S_SA + 1}]")
    g(f"s_add_u32 m0, %[scm_w], s{S_SCP}")
    g("s_nop 0")
    g(f"global_load_lds_dwordx4 %[swoff], s[{S_SW}:{S_SW + 1}]")


def advance_dma(g):
    """The DMA to its next stage: S_T + 1 of this tile, or stage 0 of the next one."""
    for a in (S_A, S_W):
        g(f"s_add_u32 s{a}, s{a}, 128")
        g(f"s_addc_u32 s{a + 1}, s{a + 1}, 0")
    g(f"s_add_u32 s{S_T}, s{S_T}, 1")
    nxt, back = g.new_label("tile"), g.new_label("tileback")
    g(f"s_cmp_eq_u32 s{S_T}, %[nk]")
    g(f"s_cbranch_scc1 {nxt}")
    g.label(back)
    g.tails.append(("tile", nxt, back))
    wrap(g, S_OFF)
    g(f"s_add_u32 s{S_WR}, %[ldsw], s{S_OFF}")


def tails(g):
    for kind, at, back in g.tails:
        g.label(at)
        if kind == "tile":
            # the next tile's first stage
            for reg, name in ((S_A, "na"), (S_W, "nw"), (S_SA, "nsa"), (S_SW, "nsw")):
                g(f"s_mov_b32 s{reg}, %[{name}_lo]")
                g(f"s_mov_b32 s{reg + 1}, %[{name}_hi]")
            g(f"s_mov_b32 s{S_SCN}, s{S_T}")
        else:
            scale_dma(g)
            # four stages on, or at the next tile's first (where S_SA is set anew)
            for a in (S_SA, S_SW):
                g(f"s_add_u32 s{a}, s{a}, 16")
                g(f"s_addc_u32 s{a + 1}, s{a + 1}, 0")
            g(f"s_xor_b32 s{S_SCP}, s{S_SCP}, {ROWS * 16}")
            g(f"s_cmp_ge_u32 s{S_T}, %[nk]")
            g(f"s_cselect_b32 s{S_T0}, 0x40000000, 4")   # the next tile's group 0 is its last here
            g(f"s_add_u32 s{S_SCN}, s{S_SCN}, s{S_T0}")
        g(f"s_branch {back}")
    g.tails = []


def addresses(g):
    """Fragment read addresses in the buffer at S_RD."""
    for k, name in enumerate(("rdx0", "rdx1", "rdw0", "rdw1")):
        g(f"v_add_u32 v{AB + k}, s{S_RD}, %[{name}]")


def read_frag(g, kind, idx, p):
    reg = wreg(p, idx) if kind == "w" else xreg(idx)
    a = AB + (2 if kind == "w" else 0)
    return [f"ds_read_b128 v[{reg + 4 * c}:{reg + 4 * c + 3}], v{a + c} offset:{idx * 2048}" for c in range(2)]


def read_scales(q):
    return ([f"ds_read_b32 v{swreg(q, i)}, v{AB + 5} offset:{i * 256}" for i in range(FI)] +
            [f"ds_read_b32 v{sxreg(q, j)}, v{AB + 4} offset:{j * 256}" for j in range(FJ)])


def scale_addresses(g):
    """The scale buffer to read, S_SCR, which then is the other one."""
    g(f"v_add_u32 v{AB + 4}, s{S_SCR}, %[scx]")
    g(f"v_add_u32 v{AB + 5}, s{S_SCR}, %[scw]")
    g(f"s_xor_b32 s{S_SCR}, s{S_SCR}, {ROWS * 16}")


def sel(b):
    lo, hi = b & 1, b >> 1
    return (f" op_sel:[{lo},{lo},0]" if lo else "") + f" op_sel_hi:[{hi},{hi},0]"


def stage(g, s8, first, done, carry):
    """Stage s with s % 8 == s8 (the first of the tile: accumulators from 0).  carry: the LDS
    reads issued behind the barrier of the stage before, in order (x 0, W, scales);
    returns this stage's."""
    p, q, b = s8 % 2, (s8 // 4) % 2, s8 % 4
    n = FI * FJ
    before = {m: [] for m in range(n)}    # slot -> (tag, instruction) ahead of its MFMA
    after = {m: [] for m in range(n)}     # and behind it
    # the first part's reads: token fragments 1 .. FJ - 1, one instruction a slot, each once its
    # buffer's column of the ring (j - NX) is done
    at = 0
    for j in range(1, FJ):
        at = max(at, (j - NX + 1) * FI)
        for ins in read_frag(g, "x", j, p):
            before[at].append((("x", j), ins))
            at += 1
    assert at <= BAR, (at, BAR)
    # the second part's: the next stage's first token fragment and W fragments, evenly, the
    # scales with the first of them
    second = [(("x", 0), ins) for ins in read_frag(g, "x", 0, 1 - p)]
    for i in range(FI):
        second += [(("w", i), ins) for ins in read_frag(g, "w", i, 1 - p)]
    small = [(("s", 0), ins) for ins in read_scales(1 - q)] if b == 3 else []
    room = n - BAR
    for k, x in enumerate(second):
        after[BAR + k * room // len(second)].append(x)
    for k, x in enumerate(small):
        after[BAR + k // 2].insert(0, x)
    # DMA: W from its barrier on, A from the stage's on
    dmas = {}
    for k in range(FJ):
        dmas.setdefault(BAR + k * room // FJ, []).append(k)
    if WBAR is None:
        dmas = {}
        for k in range(ND):
            dmas.setdefault(BAR + k * room // ND, []).append(k)
    else:
        for k in range(FI):
            dmas.setdefault(WBAR + k * (BAR - WBAR) // FI, []).append(FJ + k)

    issued, waited = list(carry), set()

    def need(*tags):
        """Wait until the reads of these fragments have landed, if not yet waited for."""
        tags = [t for t in tags if t not in waited and t in issued]
        if not tags:
            return
        last = max(k for k, t in enumerate(issued) if t in tags)
        g(f"s_waitcnt lgkmcnt({min(15, len(issued) - 1 - last)})")
        waited.update(set(issued[:last + 1]) - set(issued[last + 1:]))

    for m in range(n):
        j, i = m // FI, m % FI
        if m == 0 and carry:
            need(("s", 0), ("x", 0), ("w", 0))
        elif j == 0:
            need(("w", i))
        elif i == 0 and m < BAR:
            need(("x", j))
        if m == WBAR:
            g("s_barrier")                # W of this stage is read by every wave
        if m == BAR:
            g(f"s_waitcnt vmcnt({(NBUF - 2) * ND + (FI if WBAR is not None else 0)}) lgkmcnt(0)")
            g("s_barrier")
            wrap(g, S_RD)
            addresses(g)
            if small:
                scale_addresses(g)
            issued, waited = [], set()
        if m == (BAR if WBAR is None else WBAR):
            due, back = g.new_label("sc"), g.new_label("scback")
            g(f"s_cmp_eq_u32 s{S_T}, s{S_SCN}")
            g(f"s_cbranch_scc1 {due}")
            g.label(back)
            g.tails.append(("sc", due, back))
        for t, ins in before[m]:
            g(ins)
            issued.append(t)
        ks = dmas.get(m, [])
        if ks:
            dma_m0(g, ks[0])
        c = "0" if first else f"a[{acc(i, j)}:{acc(i, j) + 3}]"
        g(f"v_mfma_scale_f32_16x16x128_f8f6f4 a[{acc(i, j)}:{acc(i, j) + 3}], v[{wreg(p, i)}:{wreg(p, i) + 7}], "
          f"v[{xreg(j)}:{xreg(j) + 7}], {c}, v{swreg(q, i)}, v{sxreg(q, j)}{sel(b)}")
        for t, ins in after[m]:
            g(ins)
            issued.append(t)
        for x, k in enumerate(ks):
            if x:
                dma_m0(g, k)
                g("s_nop 0")
            dma_go(g, k)
    advance_dma(g)
    g(f"s_add_u32 s{S_S}, s{S_S}, 1")
    g(f"s_cmp_gt_u32 s{S_S}, s{S_NK1}")
    g(f"s_cbranch_scc1 {done}")
    return issued


def start():
    """The first tile's first NBUF stages and its first scales (group 0)."""
    g = Gen()
    for reg, name in ((S_A, "a"), (S_W, "w"), (S_SA, "sa"), (S_SW, "sw")):
        g(f"s_mov_b32 s{reg}, %[{name}_lo]")
        g(f"s_mov_b32 s{reg + 1}, %[{name}_hi]")
    g(f"s_mov_b32 s{S_SCP}, 0")
    scale_dma(g)                          # group 0, to buffer 0
    for st in range(NBUF):
        g(f"s_add_u32 s{S_WR}, %[ldsw], {st * BUF}")
        for k in range(ND):
            dma_m0(g, k)
            g("s_nop 0")
            dma_go(g, k)
        for a in (S_A, S_W):
            g(f"s_add_u32 s{a}, s{a}, 128")
            g(f"s_addc_u32 s{a + 1}, s{a + 1}, 0")
    g(f"s_waitcnt vmcnt({(NBUF - 1) * ND})")
    g("s_barrier")
    return g.lines


def body():
    """One tile, its first NBUF stages and group 0 of the scales on their way."""
    g = Gen()
    g(f"s_sub_u32 s{S_NK1}, %[nk], 1")
    g(f"s_mov_b32 s{S_S}, 0")
    g(f"s_mov_b32 s{S_RD}, %[buf]")
    g(f"s_mov_b32 s{S_OFF}, %[buf]")      # stage NBUF goes where stage 0 is
    g(f"s_add_u32 s{S_WR}, %[ldsw], s{S_OFF}")
    for reg, name in ((S_A, "a"), (S_W, "w")):
        g(f"s_add_u32 s{reg}, %[{name}_lo], {128 * NBUF}")
        g(f"s_addc_u32 s{reg + 1}, %[{name}_hi], 0")
    for reg, name in ((S_SA, "sa"), (S_SW, "sw")):
        g(f"s_add_u32 s{reg}, %[{name}_lo], 16")
        g(f"s_addc_u32 s{reg + 1}, %[{name}_hi], 0")
    g(f"s_mov_b32 s{S_SCR}, %[scb]")
    g(f"s_xor_b32 s{S_SCP}, s{S_SCR}, {ROWS * 16}")
    g(f"s_mov_b32 s{S_SCN}, 4")
    g(f"s_mov_b32 s{S_T}, {NBUF}")
    # nk == NBUF: the DMA is at the next tile already
    nxt, back = g.new_label("tile"), g.new_label("tileback")
    g(f"s_cmp_eq_u32 s{S_T}, %[nk]")
    g(f"s_cbranch_scc1 {nxt}")
    g.label(back)
    g.tails.append(("tile", nxt, back))
    addresses(g)
    scale_addresses(g)
    for ins in read_scales(0):
        g(ins)
    for ins in read_frag(g, "x", 0, 0):
        g(ins)
    for i in range(FI):
        for ins in read_frag(g, "w", i, 0):
            g(ins)
    g("s_waitcnt lgkmcnt(0)")
    done, loop = g.new_label("done"), g.new_label("loop")
    carry = stage(g, 0, True, done, [])
    g.label(loop)
    for s in range(1, 9):                 # stage 0's reads are those of every stage 8 n
        carry = stage(g, s % 8, False, done, carry)
    g(f"s_branch {loop}")
    tails(g)
    g.label(done)
    g("s_waitcnt lgkmcnt(0)")
    g(f"s_mov_b32 %[buf], s{S_RD}")
    # the next tile's group 0 is where the DMA was last (a last stage may have read on)
    g(f"s_xor_b32 %[scb], s{S_SCP}, {ROWS * 16}")
    for _ in range(3):
        g("s_nop 7")
    return g.lines


def clobbers():
    """The registers of a body and its prologue, by variant."""
    out = ["// Registers the generated mx_gemm_l4 bodies own (gen_mx_gemm.py register map)."]
    for v in VARIANTS:
        configure(*v)
        regs = [f"v{i}" for i in range(LAST_VGPR + 1)] + [f"s{i}" for i in SGPRS]
        rows = [", ".join(f'"{r}"' for r in regs[i:i + 14]) for i in range(0, len(regs), 14)]
        out.append(f"#define DITK_{name_of(FI, FJ).upper()}_CLOBBERS \\\n" + "".join(f"  {r}, \\\n" for r in rows))
    return "\n".join(out) + "\n"


def write(path, title, lines):
    with open(path, "w") as f:
        f.write(f"// Generated by gen_mx_gemm.py -- {title} of mx_gemm_l4<FI = {FI}, FJ = {FJ}>.\n")
        for line in lines:
            f.write(f'"{line}\\n"\n')


def main(argv):
    here = os.path.dirname(os.path.abspath(__file__))
    out = os.path.dirname(os.path.abspath(argv[1])) if len(argv) > 1 else here
    for v in VARIANTS:
        configure(*v)
        write(os.path.join(out, name_of(FI, FJ) + "_body.inc"), "the instruction body", body())
        write(os.path.join(out, name_of(FI, FJ) + "_start.inc"), "the first tile's DMA", start())
    with open(os.path.join(out, "mx_l4_clobbers.h"), "w") as f:
        f.write(clobbers())
    return 0


if __name__ == "__main__":
    sys.exit(main(sys.argv))
