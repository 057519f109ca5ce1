// Products of microscaled (MX) fp8 matrices on the scaled MFMA, with fused epilogues.
//
//   C[m, n] = epilogue( sum over blocks of 32 k: 2^(ea + ew) sum_32 A[m, k] W[n, k]  + bias[n] )
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 128 k of 16 x 16 outputs and applies one
// e8m0 scale per row and 32 k by itself, at twice the bf16 rate per clock (32 cycles
// for 64 Kflop).  As in gemm.hip the MFMA's A operand is a 16-row slice of W and its B
// operand 16 tokens, so a lane owns one token and 4 consecutive features per
// accumulator tile.  A lane of group g = lane / 16 feeds k 16 g .. + 15 and 64 + 16 g ..
// + 15 of the 128, and the scale of block g (k 32 g .. + 31, whichever lanes hold them).
//
// K advances in 128-k stages through LDS, 128 bytes per operand row, filled by direct
// global->LDS DMA with the 16-byte units XOR-swizzled by row: the geometry of
// gemm.hip's 64-k bf16 stages.  The scales of four stages (16 bytes a row) come with
// every fourth stage.
//
// The k order is fixed and nothing is split along k, so an output element is the same
// whatever M is, wherever its row sits and whichever tile computed it.  Few rows go without
// LDS to single waves (mx_gemm_rows).
//
// What the instruction adds: the products of 8 consecutive k over a common exponent E, the largest sum of two
// nonzero factors' exponents, below which it keeps 13 bits and cuts the others off (measured: 1 + 2^-13 is exact
// within 8 k, 1 + 2^-14 is 1); the sums of 8 and the accumulator with 24 bits.  A product loses less than 2^(E - 13).
// Of factors that are normal numbers that is at most 2^-13 of the largest product of the 8; a subnormal factor (below
// 2^-6 of its scale) counts with the exponent -6, so 448 x 2^-9 = 0.875 hides what a product of 4 would.  e4m3 has
// already rounded a factor by up to 2^-4 of it, and by 2^-10 of its scale where it is subnormal; on random data the
// result is off by 1.6e-5 of the sum of the products' magnitudes.  (Its bf16 counterpart adds exactly, at half the
// rate.)
//
// What bounds it, on one MI355X (M x N x K): 65520 x 1536 x 8960 takes 631 us (2.86 PFLOP/s; 654-692 with the gated
// residual), the matrix pipes busy 70% of the cycles at a clock that their power holds at 1.68 GHz.  The k loop
// without an epilogue does 3.0-3.1 PFLOP/s, a loop of these MFMAs on random registers alone 3.3 (4.5 on
// zeros).  At K = 1536 the epilogue counts: 65520 x 1536 x 1536 130 us for 105 without its stores (201 MB), 65520 x
// 8960 x 1536 774 us with a bias, 866 with GELU, 973 with GELU and an MX output; 32760 x 5120 x 5120 582-617 us.
#include <algorithm>
#include <type_traits>

#include "mx_common.h"
#include "mx_l4_clobbers.h"

namespace {

enum MxEpilogue : int { MXE_BIAS = 0, MXE_GELU = 1, MXE_GATE_RES = 2, MXE_RES = 3, MXE_SILU = 5 };
enum MxOut : int { MXO_BF16 = 0, MXO_FP8 = 1 };

struct MxGemmArgs {
  const uint8_t* A;
  int64_t lda;
  const uint8_t* As;
  int64_t ldas;
  const uint8_t* W;
  int64_t ldw;
  const uint8_t* Ws;
  int64_t ldws;
  const float* bias;
  void* C;
  int64_t ldc;
  uint8_t* Cs;
  int64_t ldcs;
  const bf16_t* R;
  int64_t ldr;
  const float* gate;
  int64_t gate_stride;
  const int32_t* cu;
  int nseg, M, N, K;
  int m_begin;  // this launch's rows: m_begin .. M - 1
  int tiles_m, tiles_n, group_m;
  bool stream;  // output stored past the caches
};

// 16 bytes per lane, global -> LDS; the wave's 64 lanes fill 1 KiB from slot0 on
__device__ __forceinline__ void lds_dma(const uint8_t* src, u32x4_t* slot0) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)slot0, 16, 0, 0);
}

template <int S>
__device__ __forceinline__ f32x4_t mfma_mx(i32x8_t w, i32x8_t x, f32x4_t c, uint32_t sw, uint32_t sx) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, 0, S, (int)sw, S, (int)sx);
}

// Row and feature ranges of a workgroup tile.  A tile that would reach past M or N starts
// earlier instead, so that the rows it loads are there; it stores rows from m0 and features
// from n0 on, which no other tile has.
struct MxTile {
  int m0, n0;  // first row and feature of its own
  int mb, nb;  // and of those it computes
};

// Exchanges halves between lanes l and l ^ 8 of each 16: of the first units of two 16-byte
// registers, a (columns c ..) and b (columns c + 64 bytes ..) of 16 tokens by 4 lanes, to whole
// 128-byte lines of 8 tokens by 8 lanes: `a` the tokens 0-7, `b` the tokens 8-15.
__device__ __forceinline__ void to_lines(u32x4_t& a, u32x4_t& b, bool hi) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t give = hi ? a[d] : b[d];
    const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)give, 0x128, 0xF, 0xF, true);  // row_ror:8
    a[d] = hi ? got : a[d];
    b[d] = hi ? b[d] : got;
  }
}

// The epilogue of a wave tile of FJ x 16 tokens and FI x 16 features, acc(i, j) its accumulators,
// (m, n) its first row and feature; bias8 and gate8 give 8 features' bias and gate (gate8 where
// the tile's rows are one segment).  A lane has features 4 g .. + 3 of a token per accumulator;
// permlane16 swaps between the accumulators of features 32 f and 32 f + 16 leave it with 8
// consecutive ones (32 f + 16 (g % 2) + 8 (g / 2) ..), a block of 32 among the four lanes of a
// token.  Everything before the one rounding is in fp32, and nothing goes through LDS, where
// the next tile's operands are arriving.  Stores are whole 128-byte lines: 65520 x 1536 x 1536
// (201 MB out) 171 us with 64-byte segments, 159 with lines, 145 past the caches (stream).
template <int EPI, int OUT, int FI, int FJ, class Acc, class Bias, class Gate>
__device__ __forceinline__ void mx_epilogue(const MxGemmArgs& p, const Acc& acc, const Bias& bias8, const Gate& gate8,
                                            bool one_seg, const MxTile& tile, int m, int n, int lane) {
  static_assert(FI % 4 == 0, "lines of 64 features");
  constexpr bool kRes = EPI == MXE_RES || EPI == MXE_GATE_RES;
  constexpr int NF = FI / 2;
  const int ql = lane & 15, g = lane >> 4;
  const bool hi = lane & 8;
  const int nl = n + (g & 1) * 16 + (g >> 1) * 8;
  // Output and residual go through buffer descriptors at the wave's first row, and a row or column
  // that is not the tile's has an offset past their range, where stores are dropped and loads
  // give 0: no branches, behind which the compiler would wait for every store before it uses a load.
  constexpr uint32_t kOut = 0x80000000u;
  auto uniform = [](const void* q) {
    const uint64_t x = (uint64_t)(uintptr_t)q;
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x);
    const uint64_t hi32 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(x >> 32));
    return reinterpret_cast<void*>((uintptr_t)(lo | hi32 << 32));
  };
  auto desc = [&](const void* base, int64_t row_bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(
        uniform(reinterpret_cast<const char*>(base) + (base != nullptr ? m * row_bytes : 0)), 0, 0x7fffffff,
        0x00020000);
  };
  const uint32_t ldc = (uint32_t)p.ldc * (OUT == MXO_FP8 ? 1 : 2), ldr = (uint32_t)p.ldr * 2, ldcs = (uint32_t)p.ldcs;
  const __amdgpu_buffer_rsrc_t cdesc = desc(p.C, ldc), rdesc = desc(kRes ? p.R : nullptr, ldr),
                               sdesc = desc(OUT == MXO_FP8 ? p.Cs : nullptr, ldcs);
  const int t_lo = tile.m0 - m, t_hi = p.M - m;  // the tile's rows, from m
  auto row_ok = [&](int t) { return t >= t_lo && t < t_hi; };
  auto col_ok = [&](int col) { return col >= tile.n0 && col < p.N; };
  auto store = [&](const u32x4_t& v, int t, int col, int esize) {
    const uint32_t off = row_ok(t) && col_ok(col) ? (uint32_t)t * ldc + (uint32_t)(col * esize) : kOut;
    if (p.stream) __builtin_amdgcn_raw_buffer_store_b128(v, cdesc, off, 0, 2);  // non-temporal
    else __builtin_amdgcn_raw_buffer_store_b128(v, cdesc, off, 0, 0);
  };
  float bias[NF][8], gate[NF][8];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    bias8(nl + f * 32, bias[f]);
    if (EPI == MXE_GATE_RES && one_seg) gate8(nl + f * 32, gate[f]);
  }
  u32x4_t res[kRes ? FJ : 1][kRes ? NF : 1];  // all of them asked for at once: one latency for the tile
  auto load_res = [&](int j) {
    const int t = j * 16 + ql;
#pragma unroll
    for (int f = 0; f < NF; ++f)
      res[j][f] = __builtin_amdgcn_raw_buffer_load_b128(
          rdesc, row_ok(t) && col_ok(nl + f * 32) ? (uint32_t)t * ldr + (uint32_t)(nl + f * 32) * 2 : kOut, 0, 0);
  };
  if (kRes)
#pragma unroll
    for (int j = 0; j < FJ; ++j) load_res(j);
#pragma unroll
  for (int j = 0; j < FJ; ++j) {
    u32x4_t line[NF];
    uint32_t q0[NF][2], scales = 0;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const f32x4_t a = acc(2 * f, j), b = acc(2 * f + 1, j);
      float y[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[e]), __float_as_uint(b[e]), false, false);
        y[e] = __uint_as_float(s[0]) + bias[f][e];
        y[e + 4] = __uint_as_float(s[1]) + bias[f][e + 4];
      }
      if (EPI == MXE_GELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = gelu_tanh_f(y[e]);
      } else if (EPI == MXE_SILU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = silu_f(y[e]);
      } else if (kRes) {
        float rv[8];
        unpack8(res[j][f], rv);
        if (EPI == MXE_GATE_RES) {
          if (!one_seg) {
            const int mc = min(m + j * 16 + ql, p.M - 1), nc = min(nl + f * 32, p.N - 8);
            const float* gp = p.gate + (int64_t)find_segment(p.cu, p.nseg, mc) * p.gate_stride + nc;
            const f32x4_t g0 = *reinterpret_cast<const f32x4_t*>(gp), g1 = *reinterpret_cast<const f32x4_t*>(gp + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              gate[f][e] = g0[e];
              gate[f][e + 4] = g1[e];
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = fmaf(y[e], gate[f][e], rv[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] += rv[e];
        }
      }
      if (OUT == MXO_FP8) {
        // N is whole blocks of 32 (checked on the host), tiles start at whole blocks
        scales |= mx_quantise8<MX_FP8, true>(y, q0[f]) << (8 * (f & 3));
        if (f & 1) {
          // lanes g = 0, 1: 16 columns of block f - 1 each, g = 2, 3: of block f
          const auto s0 = __builtin_amdgcn_permlane32_swap(q0[f - 1][0], q0[f][0], false, false);
          const auto s1 = __builtin_amdgcn_permlane32_swap(q0[f - 1][1], q0[f][1], false, false);
          line[f / 2] = u32x4_t{s0[0], s1[0], s0[1], s1[1]};
        }
      } else {
        line[f] = pack8(y);
      }
    }
    const int t = j * 16;
    if (OUT == MXO_FP8) {
      // 64 columns a register; lane g stores the scale of block g of each four
      const int nb = n + (g >> 1) * 32 + (g & 1) * 16;
      if (NF == 4) {
        to_lines(line[0], line[1], hi);
        store(line[0], t + (ql & 7), nb + (hi ? 64 : 0), 1);
        store(line[1], t + 8 + (ql & 7), nb + (hi ? 64 : 0), 1);
      } else {
        store(line[0], t + ql, nb, 1);
      }
      const int col = n + g * 32;
      __builtin_amdgcn_raw_buffer_store_b8((uint8_t)(scales >> (8 * g)), sdesc,
                                           g < NF && row_ok(t + ql) && col_ok(col)
                                               ? (uint32_t)(t + ql) * ldcs + (uint32_t)mx_scale_at(col >> 5)
                                               : kOut,
                                           0, 0);
    } else {
#pragma unroll
      for (int f = 0; f < NF; f += 2) {
        to_lines(line[f], line[f + 1], hi);
        const int col = nl + f * 32 + (hi ? 32 : 0);
        store(line[f], t + (ql & 7), col, 2);
        store(line[f + 1], t + 8 + (ql & 7), col, 2);
      }
    }
  }
}

// 8 consecutive floats, 16-byte aligned
__device__ __forceinline__ void load8(const float* src, float (&out)[8]) {
  const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(src), hi = *reinterpret_cast<const f32x4_t*>(src + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    out[e] = lo[e];
    out[e + 4] = hi[e];
  }
}
__device__ __forceinline__ void zero8(float (&out)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = 0.f;
}

// Whether the rows [m, m + rows) (the same for the wave) are one segment, and which: by scalar
// loads, which do not wait for the vector loads and stores on their way.
__device__ __forceinline__ bool one_segment(const MxGemmArgs& p, int m, int rows, int& seg) {
  auto load = [&](int i) {
    int v;
    asm volatile("s_load_dword %0, %1, 0x0\n s_waitcnt lgkmcnt(0)"
                 : "=s"(v)
                 : "s"(p.cu + __builtin_amdgcn_readfirstlane(i))
                 : "memory");
    return v;
  };
  const int last = min(m + rows, p.M) - 1;
  int lo = 0, hi = p.nseg - 1;
  asm volatile("" : "+s"(hi));  // compared here, not kept as a mask across the k loop
  m = min(m, p.M - 1);
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (load(mid) <= m) lo = mid;
    else hi = mid - 1;
  }
  seg = lo;
  asm volatile("" : "+s"(lo));
  return lo + 1 >= p.nseg || load(lo + 1) > last;
}

// An MX output's padding behind N, by the whole launch: zeros up to a multiple of 128 columns,
// scales 2^0 up to a multiple of 16.
__device__ __forceinline__ void mx_out_padding(const MxGemmArgs& p) {
  const int cols = ((int)mx_cols(p.N) - p.N) / 16, b0 = p.N / 32, sc = (int)mx_scale_bytes(p.N) - b0;
  const int i = threadIdx.x & 31, per = blockDim.x / 32;  // 32 threads a row: at most 6 + 15 stores
  if (cols + sc == 0) return;
  for (int row = p.m_begin + blockIdx.x * per + threadIdx.x / 32; row < p.M; row += gridDim.x * per) {
    if (i < cols)
      *reinterpret_cast<u32x4_t*>(reinterpret_cast<uint8_t*>(p.C) + (int64_t)row * p.ldc + p.N + i * 16) =
          u32x4_t{0, 0, 0, 0};
    if (i >= 16 && i < 16 + sc) p.Cs[(int64_t)row * p.ldcs + mx_scale_at(b0 + i - 16)] = 127;
  }
}

// WM x WN waves of FJ x 16 tokens by FI x 16 features each.
template <int EPI, int OUT, int FI, int FJ, int WM, int WN, int EU>
__global__ __launch_bounds__(WM * WN * 64, EU) void mx_gemm_kernel(MxGemmArgs p) {
  constexpr int GW = WM * WN, WTM = FJ * 16, WTN = FI * 16, GBM = WM * WTM, GBN = WN * WTN;
  constexpr int DA = GBM / 8 / GW, DW = GBN / 8 / GW;  // DMA instructions per wave and stage, 8 rows each
  constexpr int ROWS = GBM + GBN, SG = ROWS / 64;      // scale DMA instructions of a workgroup and four stages
  constexpr int STAGE = ROWS * 8;                      // 16-byte units of a stage
  static_assert(DA >= 1 && DW >= 1 && DA * GW * 8 == GBM && DW * GW * 8 == GBN && ROWS % 64 == 0, "tile");
  __shared__ u32x4_t lds[2 * STAGE + 2 * ROWS];
  u32x4_t* const sc_lds = lds + 2 * STAGE;

  if (OUT == MXO_FP8) mx_out_padding(p);
  const int nb = gridDim.x, b = blockIdx.x;
  const int L = (b & 7) * (nb >> 3) + (b >> 3);
  if (L >= p.tiles_m * p.tiles_n) return;
  const int group = L / (p.group_m * p.tiles_n), first_m = group * p.group_m;
  const int gm = min(p.group_m, p.tiles_m - first_m), pid = L % (p.group_m * p.tiles_n);
  const int m0 = (first_m + pid % gm) * GBM, n0 = pid / gm * GBN;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ql = lane & 15, g = lane >> 4;
  const int a_row0 = (wave % WM) * WTM, w_row0 = (wave / WM) * WTN;

  // DMA instruction d of a wave fills rows 8 (d GW + wave) .. + 7: lane -> row lane / 8,
  // LDS unit lane % 8 <- k unit (lane % 8) ^ ((row >> 1) & 7)
  const uint8_t* asrc[DA];
  const uint8_t* wsrc[DW];
#pragma unroll
  for (int d = 0; d < DA; ++d) {
    const int row = (d * GW + wave) * 8 + lane / 8;
    asrc[d] = p.A + (int64_t)min(m0 + row, p.M - 1) * p.lda + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
  }
#pragma unroll
  for (int d = 0; d < DW; ++d) {
    const int row = (d * GW + wave) * 8 + lane / 8;
    wsrc[d] = p.W + (int64_t)min(n0 + row, p.N - 1) * p.ldw + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
  }
  auto issue = [&](int kt) {
    u32x4_t* s = lds + (kt & 1) * STAGE;
#pragma unroll
    for (int d = 0; d < DA; ++d) lds_dma(asrc[d] + (int64_t)kt * 128, s + (d * GW + wave) * 64);
#pragma unroll
    for (int d = 0; d < DW; ++d) lds_dma(wsrc[d] + (int64_t)kt * 128, s + GBM * 8 + (d * GW + wave) * 64);
    if ((kt & 3) == 0) {
      // the scales of stages kt .. kt + 3: instruction i covers rows 64 i .. + 63 of A then W
      for (int i = wave; i < SG; i += GW) {
        const int row = i * 64 + lane;
        const uint8_t* src = row < GBM ? p.As + (int64_t)min(m0 + row, p.M - 1) * p.ldas
                                       : p.Ws + (int64_t)min(n0 + row - GBM, p.N - 1) * p.ldws;
        lds_dma(src + (kt >> 2) * 16, sc_lds + ((kt >> 2) & 1) * ROWS + i * 64);
      }
    }
  };

  f32x4_t acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int nk = (p.K + 127) / 128;
  // operand units of this lane: row ql of a fragment, 16-byte units g and 4 + g
  int unit[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) unit[c] = ql * 8 + ((c * 4 + g) ^ ((ql >> 1) & 7));
  auto frag = [&](const u32x4_t* rows) {
    const u32x4_t lo = rows[unit[0]], hi = rows[unit[1]];
    return i32x8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };
  uint32_t sw[FI], sx[FJ];
  auto stage = [&](int kt, auto sel) {
    constexpr int S = decltype(sel)::value;
    // stage kt is here for every wave, and the other buffer is read out: this wave's reads of it have landed too (the
    // MFMAs that wait for them are not held before the barrier by anything)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (kt + 1 < nk) issue(kt + 1);
    if (S == 0) {
      const uint32_t* s32 = reinterpret_cast<const uint32_t*>(sc_lds + ((kt >> 2) & 1) * ROWS);
#pragma unroll
      for (int i = 0; i < FI; ++i) sw[i] = s32[(GBM + w_row0 + i * 16 + ql) * 4 + g];
#pragma unroll
      for (int j = 0; j < FJ; ++j) sx[j] = s32[(a_row0 + j * 16 + ql) * 4 + g];
    }
    const u32x4_t* as = lds + (kt & 1) * STAGE + a_row0 * 8;
    const u32x4_t* ws = lds + (kt & 1) * STAGE + (GBM + w_row0) * 8;
    i32x8_t w[FI];
#pragma unroll
    for (int i = 0; i < FI; ++i) w[i] = frag(ws + i * 128);
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      const i32x8_t x = frag(as + j * 128);
#pragma unroll
      for (int i = 0; i < FI; ++i) acc[i][j] = mfma_mx<S>(w[i], x, acc[i][j], sw[i], sx[j]);
    }
  };
  issue(0);
  for (int kt = 0; kt < nk; kt += 4) {
    stage(kt, std::integral_constant<int, 0>{});
    if (kt + 1 < nk) stage(kt + 1, std::integral_constant<int, 1>{});
    if (kt + 2 < nk) stage(kt + 2, std::integral_constant<int, 2>{});
    if (kt + 3 < nk) stage(kt + 3, std::integral_constant<int, 3>{});
  }
  int seg = 0;
  const bool one_seg = EPI != MXE_GATE_RES || one_segment(p, m0 + a_row0, WTM, seg);
  auto bias8 = [&](int n, float (&v)[8]) {
    if (p.bias != nullptr) load8(p.bias + min(n, p.N - 8), v);
    else zero8(v);
  };
  auto gate8 = [&](int n, float (&v)[8]) { load8(p.gate + (int64_t)seg * p.gate_stride + min(n, p.N - 8), v); };
  mx_epilogue<EPI, OUT, FI, FJ>(p, [&](int i, int j) { return acc[i][j]; }, bias8, gate8, one_seg,
                                MxTile{m0, n0, m0, n0}, m0 + a_row0, n0 + w_row0, lane);
}

// One wave per SIMD, K of NBUF stages or more: a workgroup tile as 2 x 2 wave tiles with their accumulators in the
// AGPRs.  The k loop is generated assembly (gen_mx_gemm.py -> mx_l4_*_body.inc); this C++ part
// gives it the per-lane addresses and runs the epilogue on the accumulators.  Persistent:
// XCD x (= blockIdx % 8) owns the tiles [x * per_xcd, (x + 1) * per_xcd), which its workgroups take
// in turn; the operands of a workgroup's tiles are one stream of stages, so the next tile's
// first stages arrive under the epilogue.
template <int FI, int FJ>
struct MxL4 {
  static constexpr int GBM = 32 * FJ, GBN = 32 * FI, ROWS = GBM + GBN;
  static constexpr int NBUF = FJ == 8 ? 2 : FI == 8 ? 3 : 4;  // stage buffers, as generated
  static constexpr int VEC0 = NBUF * ROWS * 128 + 2 * ROWS * 16;  // bias of two tiles, then gates of two
  static constexpr int LDS_BYTES = VEC0 + 4 * 1024;
  static_assert(LDS_BYTES <= 160 * 1024, "LDS");
};
#define DITK_MX_L4_START_OPERANDS                                                                                     \
  [a_lo] "s"(lo32(cur.a)), [a_hi] "s"(hi32(cur.a)), [w_lo] "s"(lo32(cur.w)), [w_hi] "s"(hi32(cur.w)),                 \
      [sa_lo] "s"(lo32(cur.sa)), [sa_hi] "s"(hi32(cur.sa)), [sw_lo] "s"(lo32(cur.sw)), [sw_hi] "s"(hi32(cur.sw)),     \
      [ldsw] "s"(ldsw), [scm_a] "s"(scm_a), [scm_w] "s"(scm_w), [saoff] "v"(lv.saoff), [swoff] "v"(lv.swoff),         \
      [aoff0] "v"(lv.aoff[0]), [aoff1] "v"(lv.aoff[1]), [aoff2] "v"(lv.aoff[2]), [aoff3] "v"(lv.aoff[3]),             \
      [aoff4] "v"(lv.aoff[4]), [aoff5] "v"(lv.aoff[5]), [aoff6] "v"(lv.aoff[6]), [aoff7] "v"(lv.aoff[7]),             \
      [woff0] "v"(lv.woff[0]), [woff1] "v"(lv.woff[1]), [woff2] "v"(lv.woff[2]), [woff3] "v"(lv.woff[3]),             \
      [woff4] "v"(lv.woff[4]), [woff5] "v"(lv.woff[5]), [woff6] "v"(lv.woff[6]), [woff7] "v"(lv.woff[7])
#define DITK_MX_L4_OPERANDS                                                                                           \
  DITK_MX_L4_START_OPERANDS, [na_lo] "s"(lo32(nxt.a)), [na_hi] "s"(hi32(nxt.a)), [nw_lo] "s"(lo32(nxt.w)),            \
      [nw_hi] "s"(hi32(nxt.w)), [nsa_lo] "s"(lo32(nxt.sa)), [nsa_hi] "s"(hi32(nxt.sa)), [nsw_lo] "s"(lo32(nxt.sw)),   \
      [nsw_hi] "s"(hi32(nxt.sw)), [nk] "s"(nk), [rdx0] "v"(lv.rdx[0]), [rdx1] "v"(lv.rdx[1]), [rdw0] "v"(lv.rdw[0]),  \
      [rdw1] "v"(lv.rdw[1]), [scx] "v"(lv.scx), [scw] "v"(lv.scw)

template <int EPI, int OUT, int FI, int FJ>
__global__ __launch_bounds__(256, 1) void mx_gemm_l4(MxGemmArgs p) {
  using G = MxL4<FI, FJ>;
  constexpr int GBM = G::GBM, GBN = G::GBN, ROWS = G::ROWS, WTM = 16 * FJ, WTN = 16 * FI;
  __shared__ u32x4_t lds[G::LDS_BYTES / 16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int a_row0 = (wave & 1) * WTM, w_row0 = (wave >> 1) * WTN;
  auto su = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
  auto lo32 = [&](uint64_t x) { return su((uint32_t)x); };
  auto hi32 = [&](uint64_t x) { return su((uint32_t)(x >> 32)); };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) u32x4_t*)&lds[0];
  const uint32_t sc0 = lds0 + G::NBUF * ROWS * 128;
  // The lane's id anew, so that neither it nor what is computed from it is kept across the k loop,
  // which has no registers to spare: spilled, it would be read back behind all of a tile's stores
  // (which share the loads' counter), every store of the tile waited for.
  auto lane_id = []() {
    int l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n v_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
    return l;
  };
  const int sa_row = (wave % (GBM / 64)) * 64, sw_row = (wave % (GBN / 64)) * 64;
  const uint32_t ldsw = su(lds0 + wave * 1024), scm_a = su(sc0 + sa_row * 16), scm_w = su(sc0 + (GBM + sw_row) * 16);
  const uint32_t nk = su((p.K + 127) / 128);
  struct Lane {
    uint32_t rdx[2], rdw[2], scx, scw, aoff[8], woff[8], saoff, swoff;
  };
  auto lane_values = [&](int lane) {
    const int ql = lane & 15, g = lane >> 4;
    Lane v;
    // fragment reads: row ql of a 16-row fragment, 16-byte units g and 4 + g of its 128 k,
    // stored at unit ^ ((row >> 1) & 7) of the 128-byte LDS row
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t part = (uint32_t)(ql * 128 + (((c * 4 + g) ^ ((ql >> 1) & 7)) * 16));
      v.rdx[c] = lds0 + a_row0 * 128 + part;
      v.rdw[c] = lds0 + (GBM + w_row0) * 128 + part;
    }
    v.scx = sc0 + (a_row0 + ql) * 16 + g * 4;
    v.scw = sc0 + (GBM + w_row0 + ql) * 16 + g * 4;
    // DMA instruction d of this wave fills rows 8 (4 d + wave) .. + 7 (1 KiB): lane l -> row l / 8, LDS
    // unit l % 8 <- k unit (l % 8) ^ ((row >> 1) & 7).  Rows past the matrix (of a matrix of less than a
    // tile's rows) read its last one.
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const int row = (d * 4 + wave) * 8 + lane / 8;
      const uint32_t unit = (uint32_t)(((lane & 7) ^ ((row >> 1) & 7)) * 16);
      v.aoff[d] = d < FJ ? (uint32_t)min(row, p.M - 1) * (uint32_t)p.lda + unit : 0u;
      v.woff[d] = d < FI ? (uint32_t)min(row, p.N - 1) * (uint32_t)p.ldw + unit : 0u;
    }
    // scale DMA: 64 rows of 16 bytes; a wave has one instruction for A and one for W (at 128 rows
    // two waves each fetch the same rows)
    v.saoff = (uint32_t)min(sa_row + lane, p.M - 1) * (uint32_t)p.ldas;
    v.swoff = (uint32_t)min(sw_row + lane, p.N - 1) * (uint32_t)p.ldws;
    return v;
  };

  struct Bases {
    uint64_t a, w, sa, sw;
  };
  auto tile_at = [&](int L) {
    const int group = L / (p.group_m * p.tiles_n), first_m = group * p.group_m;
    const int gm = min(p.group_m, p.tiles_m - first_m), pid = L % (p.group_m * p.tiles_n);
    MxTile t;
    t.m0 = p.m_begin + (first_m + pid % gm) * GBM;
    t.n0 = pid / gm * GBN;
    t.mb = min(t.m0, max(0, p.M - GBM));
    t.nb = min(t.n0, max(0, p.N - GBN));
    return t;
  };
  auto bases = [&](const MxTile& t) {
    return Bases{(uint64_t)(uintptr_t)(p.A + t.mb * p.lda), (uint64_t)(uintptr_t)(p.W + t.nb * p.ldw),
                 (uint64_t)(uintptr_t)(p.As + t.mb * p.ldas), (uint64_t)(uintptr_t)(p.Ws + t.nb * p.ldws)};
  };
  const int nb = gridDim.x, b = blockIdx.x, ntiles = p.tiles_m * p.tiles_n, per_xcd = (ntiles + 7) / 8;
  const int thi = min((b & 7) * per_xcd + per_xcd, ntiles);
  int L = (b & 7) * per_xcd + (b >> 3);
  if (OUT == MXO_FP8) mx_out_padding(p);
  if (L >= thi) return;
  MxTile tile = tile_at(L);
  Bases cur = bases(tile);
  {
  const Lane lv = lane_values(lane_id());
  if constexpr (FI == 8 && FJ == 8)
    asm volatile(
#include "mx_l4_256x256_start.inc"
        : : DITK_MX_L4_START_OPERANDS : DITK_MX_L4_256X256_CLOBBERS "m0", "scc", "memory");
  else if constexpr (FI == 8 && FJ == 4)
    asm volatile(
#include "mx_l4_128x256_start.inc"
        : : DITK_MX_L4_START_OPERANDS : DITK_MX_L4_128X256_CLOBBERS "m0", "scc", "memory");
  else if constexpr (FI == 4 && FJ == 4)
    asm volatile(
#include "mx_l4_128x128_start.inc"
        : : DITK_MX_L4_START_OPERANDS : DITK_MX_L4_128X128_CLOBBERS "m0", "scc", "memory");
  else
    asm volatile(
#include "mx_l4_64x128_start.inc"
        : : DITK_MX_L4_START_OPERANDS : DITK_MX_L4_64X128_CLOBBERS "m0", "scc", "memory");
  }
  uint32_t buf = 0, scb = 0;  // LDS offsets of the next tile's stage 0 and scale group 0
  int par = 0;                // this tile's bias and gate in LDS
  for (;;) {
    // The tile's bias and gate come through LDS, asked for a tile ahead of their use: loaded behind
    // the k loop they would wait for the next tile's DMA.  (The buffers alternate: waves may
    // still be in the last tile's epilogue, but behind the last barrier of the tile before.)
    int seg = 0;
    const bool one_seg = EPI != MXE_GATE_RES || one_segment(p, tile.mb, GBM, seg);
    const int vrow = (wave % (GBN / 64)) * 64;
    auto fetch = [&](const float* src, int at) {
      const uint32_t m0v = su(lds0 + G::VEC0 + at * 1024 + vrow * 4),
                     off = (uint32_t)min(tile.nb + vrow + lane_id(), p.N - 1) * 4;
      asm volatile("s_mov_b32 m0, %0\n s_nop 0\n global_load_lds_dword %1, %2" ::"s"(m0v), "v"(off), "s"(src)
                   : "m0", "memory");
    };
    uint64_t has_bias = (uint64_t)(uintptr_t)p.bias;  // compared where it is used, as lane_id()
    asm volatile("" : "+s"(has_bias));
    if (has_bias) fetch(p.bias, par);
    if (EPI == MXE_GATE_RES && one_seg) fetch(p.gate + (int64_t)seg * p.gate_stride, 2 + par);
    const int Ln = L + (nb >> 3);
    const bool more = Ln < thi;
    const MxTile next = more ? tile_at(Ln) : tile;
    const Bases nxt = bases(next);  // behind the last tile: its own first stages once more, read by nobody
    f32x16_t c[FI * FJ / 4];
    buf = su(buf);
    scb = su(scb);
    const Lane lv = lane_values(lane_id());
    if constexpr (FI == 8 && FJ == 8)
      asm volatile(
#include "mx_l4_256x256_body.inc"
          : [buf] "+&s"(buf), [scb] "+&s"(scb), "=&{a[0:15]}"(c[0]), "=&{a[16:31]}"(c[1]), "=&{a[32:47]}"(c[2]),
            "=&{a[48:63]}"(c[3]), "=&{a[64:79]}"(c[4]), "=&{a[80:95]}"(c[5]), "=&{a[96:111]}"(c[6]),
            "=&{a[112:127]}"(c[7]), "=&{a[128:143]}"(c[8]), "=&{a[144:159]}"(c[9]), "=&{a[160:175]}"(c[10]),
            "=&{a[176:191]}"(c[11]),
            "=&{a[192:207]}"(c[12]), "=&{a[208:223]}"(c[13]), "=&{a[224:239]}"(c[14]), "=&{a[240:255]}"(c[15])
          : DITK_MX_L4_OPERANDS : DITK_MX_L4_256X256_CLOBBERS "m0", "scc", "memory");
    else if constexpr (FI == 8 && FJ == 4)
      asm volatile(
#include "mx_l4_128x256_body.inc"
          : [buf] "+&s"(buf), [scb] "+&s"(scb), "=&{a[0:15]}"(c[0]), "=&{a[16:31]}"(c[1]), "=&{a[32:47]}"(c[2]),
            "=&{a[48:63]}"(c[3]), "=&{a[64:79]}"(c[4]), "=&{a[80:95]}"(c[5]), "=&{a[96:111]}"(c[6]),
            "=&{a[112:127]}"(c[7])
          : DITK_MX_L4_OPERANDS : DITK_MX_L4_128X256_CLOBBERS "m0", "scc", "memory");
    else if constexpr (FI == 4 && FJ == 4)
      asm volatile(
#include "mx_l4_128x128_body.inc"
          : [buf] "+&s"(buf), [scb] "+&s"(scb), "=&{a[0:15]}"(c[0]), "=&{a[16:31]}"(c[1]), "=&{a[32:47]}"(c[2]),
            "=&{a[48:63]}"(c[3])
          : DITK_MX_L4_OPERANDS : DITK_MX_L4_128X128_CLOBBERS "m0", "scc", "memory");
    else
      asm volatile(
#include "mx_l4_64x128_body.inc"
          : [buf] "+&s"(buf), [scb] "+&s"(scb), "=&{a[0:15]}"(c[0]), "=&{a[16:31]}"(c[1])
          : DITK_MX_L4_OPERANDS : DITK_MX_L4_64X128_CLOBBERS "m0", "scc", "memory");
    auto acc = [&](int i, int j) {
      const int r = i * FJ + j;
      const f32x16_t& v = c[r / 4];
      const int e = r % 4 * 4;
      return f32x4_t{v[e], v[e + 1], v[e + 2], v[e + 3]};
    };
    const int lane = lane_id();
    const float* vec = reinterpret_cast<const float*>(reinterpret_cast<const char*>(lds) + G::VEC0) - tile.nb;
    asm volatile("" : "+s"(has_bias));
    auto bias8 = [&](int n, float (&v)[8]) {
      if (has_bias) load8(vec + par * 256 + n, v);
      else zero8(v);
    };
    auto gate8 = [&](int n, float (&v)[8]) { load8(vec + (2 + par) * 256 + n, v); };
    mx_epilogue<EPI, OUT, FI, FJ>(p, acc, bias8, gate8, one_seg, tile, tile.mb + a_row0, tile.nb + w_row0, lane);
    if (!more) break;
    par ^= 1;
    L = Ln;
    tile = next;
    cur = nxt;
  }
  // the DMAs on their way behind the last tile have to land before the LDS is another workgroup's
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// An output of this size or more is stored past the caches: it would not stay there until the
// next kernel reads it, as gemm.hip's.
constexpr int64_t kStreamBytes = 64ll << 20;

// Tile order: groups of m-tiles walked m-fastest, so that the tiles running together share
// operand rows in their XCD's L2.  Groups of 2 to 16 are within 3% of each other, 1 loses up to 12%
// where many n-tiles make a round (65520 x 8960 x 1536) and 32 10-48%.
int mx_group_m(int K, int tiles_n) { return K >= 4096 || tiles_n >= 24 ? 4 : 8; }

template <int EPI, int OUT, int FI, int FJ, int WM, int WN, int EU>
int launch(MxGemmArgs p, hipStream_t stream) {
  constexpr int GBM = WM * FJ * 16, GBN = WN * FI * 16;
  p.tiles_m = (p.M + GBM - 1) / GBM;
  p.tiles_n = (p.N + GBN - 1) / GBN;
  p.group_m = mx_group_m(p.K, p.tiles_n);
  const int64_t blocks = ((int64_t)p.tiles_m * p.tiles_n + 7) / 8 * 8;
  DITK_REQUIRE(blocks * (WM * WN * 64) < (1ll << 32), "ditk_mx_gemm: grid too large");
  mx_gemm_kernel<EPI, OUT, FI, FJ, WM, WN, EU><<<(unsigned)blocks, WM * WN * 64, 0, stream>>>(p);
  return ditk_check_launch("ditk_mx_gemm");
}

template <int EPI, int OUT, int FI, int FJ>
int launch_l4(MxGemmArgs p, hipStream_t stream) {
  constexpr int GBM = MxL4<FI, FJ>::GBM, GBN = MxL4<FI, FJ>::GBN;
  p.tiles_m = (p.M - p.m_begin + GBM - 1) / GBM;
  p.tiles_n = (p.N + GBN - 1) / GBN;
  p.group_m = mx_group_m(p.K, p.tiles_n);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  DITK_REQUIRE(tiles < (1ll << 30), "ditk_mx_gemm: grid too large");
  // one persistent workgroup per CU (a multiple of 8: the same number per XCD)
  const int64_t blocks = std::min<int64_t>((tiles + 7) / 8 * 8, std::max(8, ditk_cu_count() / 8 * 8));
  mx_gemm_l4<EPI, OUT, FI, FJ><<<(unsigned)blocks, 256, 0, stream>>>(p);
  return ditk_check_launch("ditk_mx_gemm");
}

// Few rows: a wave computes 16 FJ tokens by 16 FI features by itself, its operand fragments straight from memory
// into registers, a chunk of 512 k (a dword of scales a row and lane) ahead.  Nothing is shared and
// nothing waits for another wave: a 128-k step costs its loads, 0.17 us, where a stage through LDS costs its
// barrier and its reads, and with the weight from memory 0.48.  The same MFMAs in the same k order:
// bitwise the tiles' results.  (Weights from memory: 16 x 1536 x 1536 8.1 us on tiles, 4.9 here; 16 x 5120 x 1536
// 23.1 and 10.2; 64 x 14336 x 512 60 and 22; 128 x 5120 x 1536 26.3 and 14.7.  Two chunks ahead: 10% less
// at K = 14336 and one wave a CU, up to 40% more elsewhere.)
template <int EPI, int OUT, int FI, int FJ>
__global__ __launch_bounds__(64) void mx_gemm_rows(MxGemmArgs p) {
  constexpr int SETS = 2;
  static_assert(OUT == MXO_BF16 || FI == 2, "an MX block is 32 features");
  constexpr bool kRes = EPI == MXE_RES || EPI == MXE_GATE_RES;
  if (OUT == MXO_FP8 && blockIdx.y == 0) mx_out_padding(p);
  const int lane = threadIdx.x, ql = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * FI), m0 = p.m_begin + blockIdx.y * (16 * FJ);
  const int steps = (p.K + 127) / 128, chunks = (steps + 3) / 4;
  const uint8_t *wp[FI], *xp[FJ], *wsp[FI], *xsp[FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i) {
    const int row = min(n0 + i * 16 + ql, p.N - 1);
    wp[i] = p.W + (int64_t)row * p.ldw + g * 16;
    wsp[i] = p.Ws + (int64_t)row * p.ldws + g * 4;
  }
#pragma unroll
  for (int j = 0; j < FJ; ++j) {
    const int row = min(m0 + j * 16 + ql, p.M - 1);
    xp[j] = p.A + (int64_t)row * p.lda + g * 16;
    xsp[j] = p.As + (int64_t)row * p.ldas + g * 4;
  }
  u32x4_t w[SETS][4][FI][2], x[SETS][4][FJ][2];
  uint32_t sw[SETS][FI], sx[SETS][FJ];
  auto load = [&](int set, int c) {  // (behind the last chunk, and the last 128 k, those once more)
    c = min(c, chunks - 1);
#pragma unroll
    for (int i = 0; i < FI; ++i) sw[set][i] = *reinterpret_cast<const uint32_t*>(wsp[i] + c * 16);
#pragma unroll
    for (int j = 0; j < FJ; ++j) sx[set][j] = *reinterpret_cast<const uint32_t*>(xsp[j] + c * 16);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int64_t k = (int64_t)min(c * 4 + t, steps - 1) * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < FI; ++i) w[set][t][i][h] = *reinterpret_cast<const u32x4_t*>(wp[i] + k + h * 64);
#pragma unroll
        for (int j = 0; j < FJ; ++j) x[set][t][j][h] = *reinterpret_cast<const u32x4_t*>(xp[j] + k + h * 64);
      }
    }
  };
  auto frag = [](const u32x4_t (&v)[2]) {
    return i32x8_t{(int)v[0][0], (int)v[0][1], (int)v[0][2], (int)v[0][3],
                   (int)v[1][0], (int)v[1][1], (int)v[1][2], (int)v[1][3]};
  };
  f32x4_t acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto stage = [&](int set, auto sel) {
    constexpr int S = decltype(sel)::value;
#pragma unroll
    for (int j = 0; j < FJ; ++j)
#pragma unroll
      for (int i = 0; i < FI; ++i)
        acc[i][j] = mfma_mx<S>(frag(w[set][S][i]), frag(x[set][S][j]), acc[i][j], sw[set][i], sx[set][j]);
  };
  auto use = [&](int set, int c) {
    stage(set, std::integral_constant<int, 0>{});
    if (c * 4 + 1 < steps) stage(set, std::integral_constant<int, 1>{});
    if (c * 4 + 2 < steps) stage(set, std::integral_constant<int, 2>{});
    if (c * 4 + 3 < steps) stage(set, std::integral_constant<int, 3>{});
  };
#pragma unroll
  for (int d = 0; d < SETS - 1; ++d) load(d, d);
  for (int c = 0; c < chunks; c += SETS) {
#pragma unroll
    for (int d = 0; d < SETS; ++d) {
      if (c + d >= chunks) break;
      load((d + SETS - 1) % SETS, c + d + SETS - 1);
      use(d, c + d);
    }
  }
  // A lane has features 4 g .. + 3 of each 16 of a token; the MX output's 8 of 32 as in mx_epilogue.
#pragma unroll
  for (int j = 0; j < FJ; ++j) {
    const int m = m0 + j * 16 + ql;
    const bool row = m < p.M;
    const float* gate = nullptr;
    if (EPI == MXE_GATE_RES) gate = p.gate + (int64_t)find_segment(p.cu, p.nseg, min(m, p.M - 1)) * p.gate_stride;
    auto apply = [&](f32x4_t y, int n) {
      if (p.bias != nullptr) y += *reinterpret_cast<const f32x4_t*>(p.bias + n);
      if (EPI == MXE_GELU) {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = gelu_tanh_f(y[e]);
      } else if (EPI == MXE_SILU) {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = silu_f(y[e]);
      } else if (kRes) {
        const u32x2_t r = *reinterpret_cast<const u32x2_t*>(p.R + (int64_t)min(m, p.M - 1) * p.ldr + n);
        const f32x4_t rv{__uint_as_float(r[0] << 16), __uint_as_float(r[0] & 0xffff0000u), __uint_as_float(r[1] << 16),
                         __uint_as_float(r[1] & 0xffff0000u)};
        if (EPI == MXE_GATE_RES) {
          const f32x4_t gv = *reinterpret_cast<const f32x4_t*>(gate + n);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = fmaf(y[e], gv[e], rv[e]);
        } else {
          y += rv;
        }
      }
      return y;
    };
    if (OUT == MXO_BF16) {
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const int n = n0 + i * 16 + g * 4;
        if (n >= p.N) continue;
        const f32x4_t y = apply(acc[i][j], n);
        if (row)
          *reinterpret_cast<u32x2_t*>(reinterpret_cast<bf16_t*>(p.C) + (int64_t)m * p.ldc + n) =
              u32x2_t{pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3])};
      }
    } else {
      const f32x4_t a = apply(acc[0][j], n0 + g * 4), b = apply(acc[FI - 1][j], n0 + 16 + g * 4);
      float y[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[e]), __float_as_uint(b[e]), false, false);
        y[e] = __uint_as_float(s[0]);
        y[e + 4] = __uint_as_float(s[1]);
      }
      uint32_t q[2];
      const uint32_t scale = mx_quantise8<MX_FP8, true>(y, q);
      if (row) {
        *reinterpret_cast<u32x2_t*>(reinterpret_cast<uint8_t*>(p.C) + (int64_t)m * p.ldc + n0 + (g & 1) * 16 +
                                    (g >> 1) * 8) = u32x2_t{q[0], q[1]};
        if (g == 0) p.Cs[(int64_t)m * p.ldcs + mx_scale_at(n0 >> 5)] = (uint8_t)scale;
      }
    }
  }
}

template <int EPI, int OUT, int FI, int FJ>
int launch_rows(MxGemmArgs p, hipStream_t stream) {
  const dim3 grid((unsigned)((p.N + 16 * FI - 1) / (16 * FI)), (unsigned)((p.M - p.m_begin + 16 * FJ - 1) / (16 * FJ)));
  mx_gemm_rows<EPI, OUT, FI, FJ><<<grid, 64, 0, stream>>>(p);
  return ditk_check_launch("ditk_mx_gemm");
}

// The tiles of mx_gemm_l4 (tokens x features) and their measured time in us, start + rounds x (tile +
// stage x K / 128) with a round one tile per CU: least squares over 100 products of 16 to 65520 rows with
// seven weights of the Wan and SD3.5 blocks, operands from memory, 9-11% rms.  The tile it predicts
// fastest is 0.15% slower than the fastest on average.  A stage of 256 x 256 is 1.07 us for
// 64 MFMAs of 32 cycles, 0.85 us at 2.4 GHz; the smaller tiles' are bound by their LDS reads and the issue
// of one wave (64 x 128: 0.36 us for 0.11 of MFMA) but let few rows use more CUs.
struct MxCfg {
  int gbm, gbn;
  float start, tile, stage;
};
constexpr int kCfgs = 4;
constexpr MxCfg kCfg[kCfgs] = {{256, 256, -2.4f, 10.1f, 1.067f}, {128, 256, 0.5f, 4.8f, 0.674f},
                               {128, 128, 2.1f, 1.8f, 0.469f},   {64, 128, 2.5f, 0.55f, 0.358f}};

float cfg_us(int c, int64_t tiles, int K, int cus) {
  const int64_t rounds = (tiles + cus - 1) / cus;
  return kCfg[c].start + (float)rounds * (kCfg[c].tile + kCfg[c].stage * (float)((K - 1) / 128 + 1));
}

// How a product runs: rows [0, rows) on tiles of configuration cfg, the others on `rest` in a second
// launch, where the last round of tiles would leave most CUs idle and the estimate gains by
// kSplitGain: 4096 x 5120 x 5120 120 -> 108 us (20% predicted), but 16384 x 1536 x 8960 188 -> 202 us (6%
// predicted: over several rounds the workgroups drift apart).  Every row is computed the same
// way whichever tile has it.
struct MxPlan {
  int cfg, rows, rest;
  float us;
};
constexpr float kSplitGain = 0.9f;
MxPlan plan_one(int M, int N, int K, int cus) {
  MxPlan best{0, M, 0, 1e30f};
  for (int c = 0; c < kCfgs; ++c) {
    const int64_t tiles = ((int64_t)(M - 1) / kCfg[c].gbm + 1) * ((N - 1) / kCfg[c].gbn + 1);
    const float us = cfg_us(c, tiles, K, cus);
    if (us < best.us) best = MxPlan{c, M, 0, us};
  }
  return best;
}
MxPlan mx_plan(int M, int N, int K) {
  const int cus = std::max(8, ditk_cu_count() / 8 * 8);
  const MxPlan one = plan_one(M, N, K, cus);
  MxPlan best = one;
  for (int c = 0; c < kCfgs; ++c) {
    const int64_t tn = (N - 1) / kCfg[c].gbn + 1, tm = (M - 1) / kCfg[c].gbm + 1;
    const int64_t main_m = tm * tn / cus * cus / tn;  // tile rows of the full rounds
    if (main_m == 0 || main_m >= tm || tm * tn % cus == 0) continue;
    const int rows = (int)main_m * kCfg[c].gbm;
    const MxPlan rest = plan_one(M - rows, N, K, cus);
    const float us = cfg_us(c, main_m * tn, K, cus) + rest.us;
    if (us < best.us && us < kSplitGain * one.us) best = MxPlan{c, rows, rest.cfg, us};
  }
  return best;
}

// The kernels a product can run on (as numbered by ditk_mx_gemm_plan): a configuration of kCfg, or
// mx_gemm_kernel on 256 x 256 or 64 x 128 tiles, for the short K that the l4 kernel's ring of stages
// does not fit into (2 for 256 x 256 tiles, up to 4 for the others) and for row strides that its 32-bit
// offsets do not reach over 256 rows.  (65520 x 8960 x 384: 423 us on mx_gemm_kernel, 327 on the l4 one.)
constexpr int kPlainLarge = kCfgs, kPlainSmall = kCfgs + 1;
// mx_gemm_rows on 16 x 16 (16 x 32 for an MX output) and 32 x 32 outputs a wave.  In us, start + step x K / 128 +
// rounds x (wave + stage x K / 128) with a round one wave a CU (bound by what a CU loads, 27-30 KB a us: a second
// wave takes as long again), from M = 1 .. 256, N = 512 .. 13824, K = 512 .. 14336 with the weights from memory.
// The tiles' estimate gets kCold more for each 128 k: its products found some of their operands in the
// caches.  What the rule chooses there takes 1% longer than the best of the three on average, 12% at worst.
constexpr int kRows16 = kCfgs + 2, kRows32 = kCfgs + 3;
constexpr float kCold = 0.2f;
struct RowsCfg {
  int gbm, gbn;
  float start, step, wave, stage;
};
constexpr RowsCfg kRowsCfg[3] = {{16, 16, 2.1f, 0.02f, 0.55f, 0.132f},
                                 {16, 32, 2.2f, 0.07f, 1.0f, 0.18f},
                                 {32, 32, 2.8f, 0.02f, 0.9f, 0.24f}};
float rows_us(const RowsCfg& c, int M, int N, int K, int cus) {
  const int64_t waves = (int64_t)((M - 1) / c.gbm + 1) * ((N - 1) / c.gbn + 1), rounds = (waves + cus - 1) / cus;
  const float steps = (float)((K - 1) / 128 + 1);
  // (more rounds than this are the tiles' business, and their grid is not checked)
  return rounds > 8 ? 1e30f : c.start + c.step * steps + (float)rounds * (c.wave + c.stage * steps);
}
MxPlan mx_plan_any(int M, int N, int K, int64_t ld, bool mx_out) {
  const int cus = ditk_cu_count();
  const float r16 = rows_us(kRowsCfg[mx_out ? 1 : 0], M, N, K, cus), r32 = rows_us(kRowsCfg[2], M, N, K, cus);
  const float rows = std::min(r16, r32);
  if (rows < 1e30f && rows < mx_plan(M, N, K).us + kCold * (float)((K - 1) / 128 + 1))
    return MxPlan{r16 <= r32 ? kRows16 : kRows32, M, 0, rows};
  const bool l4 = 256 * ld < (1ll << 31), large = ((int64_t)(M - 1) / 256 + 1) * ((N - 1) / 256 + 1) >= 128;
  if (l4 && K > 384) return mx_plan(M, N, K);
  return MxPlan{!large ? kPlainSmall : l4 && K > 128 ? 0 : kPlainLarge, M, 0, 0.f};
}

template <int EPI, int OUT>
int launch_plan(const MxGemmArgs& p, hipStream_t stream) {
  auto part = [&](int tile, int begin, int end) {
    MxGemmArgs q = p;
    q.m_begin = begin;
    q.M = end;
    switch (tile) {
      case 0: return launch_l4<EPI, OUT, 8, 8>(q, stream);
      case 1: return launch_l4<EPI, OUT, 8, 4>(q, stream);
      case 2: return launch_l4<EPI, OUT, 4, 4>(q, stream);
      case 3: return launch_l4<EPI, OUT, 4, 2>(q, stream);
      case kPlainLarge: return launch<EPI, OUT, 4, 8, 2, 4, 1>(q, stream);
      case kRows16: return launch_rows<EPI, OUT, OUT == MXO_FP8 ? 2 : 1, 1>(q, stream);
      case kRows32: return launch_rows<EPI, OUT, 2, 2>(q, stream);
      default: return launch<EPI, OUT, 4, 2, 2, 2, 2>(q, stream);
    }
  };
  const int64_t ld = std::max(std::max(p.lda, p.ldw), std::max(p.ldas, p.ldws));
  const MxPlan plan = mx_plan_any(p.M, p.N, p.K, ld, OUT == MXO_FP8);
  const int rc = part(plan.cfg, 0, plan.rows);
  return rc != 0 || plan.rows == p.M ? rc : part(plan.rest, plan.rows, p.M);
}

}  // namespace

DITK_EXPORT int ditk_mx_gemm(const void* A, int64_t lda, const void* As, int64_t ldas, const void* W, int64_t ldw,
                             const void* Ws, int64_t ldws, const float* bias, void* C, int64_t ldc, void* Cs,
                             int64_t ldcs, int M, int N, int K, int epilogue, int out_kind, const void* R, int64_t ldr,
                             const float* gate, int64_t gate_stride, const int32_t* cu_seqlens, int nseg,
                             hipStream_t stream) {
  // the row tensors may be NULL when there are no rows (an empty tensor's pointer)
  DITK_REQUIRE(W && Ws && (M == 0 || (A && As && C)), "ditk_mx_gemm: null operand");
  DITK_REQUIRE(M >= 0 && N > 0 && K > 0, "ditk_mx_gemm: bad shape M=%d N=%d K=%d", M, N, K);
  DITK_REQUIRE(K % 32 == 0 && N % 8 == 0, "ditk_mx_gemm: K=%d must be a multiple of 32, N=%d of 8", K, N);
  DITK_REQUIRE(M <= kMxMaxRows && K <= kMxMaxCols, "ditk_mx_gemm: too many rows (M=%d) or K=%d too long", M, K);
  DITK_REQUIRE(lda % 16 == 0 && ldw % 16 == 0 && lda >= mx_cols(K) && ldw >= mx_cols(K) && ldas % 16 == 0 &&
                   ldws % 16 == 0 && ldas >= mx_scale_bytes(K) && ldws >= mx_scale_bytes(K),
               "ditk_mx_gemm: operand rows need their padding and 16-byte strides");
  DITK_REQUIRE(((uintptr_t)A % 16) == 0 && ((uintptr_t)As % 16) == 0 && ((uintptr_t)W % 16) == 0 &&
                   ((uintptr_t)Ws % 16) == 0 && ((uintptr_t)C % 16) == 0 && ((uintptr_t)bias % 16) == 0,
               "ditk_mx_gemm: operands must be 16-byte aligned");
  DITK_REQUIRE(out_kind == MXO_BF16 || out_kind == MXO_FP8, "ditk_mx_gemm: unknown output %d", out_kind);
  const bool res = epilogue == MXE_RES || epilogue == MXE_GATE_RES;
  DITK_REQUIRE(epilogue == MXE_BIAS || epilogue == MXE_GELU || epilogue == MXE_SILU || res,
               "ditk_mx_gemm: unknown epilogue %d", epilogue);
  if (out_kind == MXO_BF16) {
    DITK_REQUIRE(ldc % 8 == 0 && ldc >= N, "ditk_mx_gemm: ldc must be a multiple of 8 and >= N");
  } else {
    DITK_REQUIRE(!res, "ditk_mx_gemm: a residual epilogue writes bf16");
    DITK_REQUIRE(N % 32 == 0, "ditk_mx_gemm: N=%d of an MX output must be a multiple of 32", N);
    DITK_REQUIRE((M == 0 || Cs) && ldc % 16 == 0 && ldc >= mx_cols(N) && ldcs % 16 == 0 && ldcs >= mx_scale_bytes(N) &&
                     ((uintptr_t)Cs % 16) == 0,
                 "ditk_mx_gemm: MX output rows need their padding and 16-byte strides");
  }
  DITK_REQUIRE(ldc < (1 << 22) && ldr < (1 << 22) && ldcs < (1 << 22), "ditk_mx_gemm: output row strides too large");
  DITK_REQUIRE(!res || ((R || M == 0) && ldr % 8 == 0 && ldr >= N && ((uintptr_t)R % 16) == 0),
               "ditk_mx_gemm: residual epilogue needs a 16-byte aligned R with ldr %% 8 == 0");
  DITK_REQUIRE(epilogue != MXE_GATE_RES || (gate && cu_seqlens && nseg > 0 && gate_stride % 4 == 0 &&
                                            ((uintptr_t)gate % 16) == 0),
               "ditk_mx_gemm: gated epilogue needs 16-byte aligned gate rows and cu_seqlens");
  if (M == 0) return 0;
  const MxGemmArgs p{(const uint8_t*)A, lda, (const uint8_t*)As, ldas, (const uint8_t*)W, ldw, (const uint8_t*)Ws, ldws,
                     bias, C, ldc, (uint8_t*)Cs, ldcs, (const bf16_t*)R, ldr, gate, gate_stride, cu_seqlens, nseg,
                     M, N, K, 0, 0, 0, 0, (int64_t)M * N * (out_kind == MXO_FP8 ? 1 : 2) >= kStreamBytes};
  const bool mx = out_kind == MXO_FP8;
  switch (epilogue) {
    case MXE_BIAS: return mx ? launch_plan<MXE_BIAS, MXO_FP8>(p, stream) : launch_plan<MXE_BIAS, MXO_BF16>(p, stream);
    case MXE_GELU: return mx ? launch_plan<MXE_GELU, MXO_FP8>(p, stream) : launch_plan<MXE_GELU, MXO_BF16>(p, stream);
    case MXE_SILU: return mx ? launch_plan<MXE_SILU, MXO_FP8>(p, stream) : launch_plan<MXE_SILU, MXO_BF16>(p, stream);
    case MXE_RES: return launch_plan<MXE_RES, MXO_BF16>(p, stream);
    default: return launch_plan<MXE_GATE_RES, MXO_BF16>(p, stream);
  }
}

DITK_EXPORT int ditk_mx_gemm_plan_for(int M, int N, int K, int64_t row_stride, int out_kind, int* plan) {
  DITK_REQUIRE(plan && M > 0 && N > 0 && N % 8 == 0 && K > 0 && K % 32 == 0 && row_stride >= mx_cols(K) &&
                   (out_kind == MXO_BF16 || (out_kind == MXO_FP8 && N % 32 == 0)),
               "ditk_mx_gemm_plan: bad arguments");
  const MxPlan p = mx_plan_any(M, N, K, row_stride, out_kind == MXO_FP8);
  plan[0] = p.cfg;
  plan[1] = p.rows;
  plan[2] = p.rest;
  return 0;
}

DITK_EXPORT int ditk_mx_gemm_plan(int M, int N, int K, int* plan) {
  return ditk_mx_gemm_plan_for(M, N, K, K > 0 ? mx_cols(K) : 0, MXO_BF16, plan);
}
