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
// whatever M is, wherever its row sits and whichever tile computed it.
#include <type_traits>

#include "mx_common.h"

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
  int tiles_m, tiles_n, group_m;
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

// The epilogue of a wave tile of FJ x 16 tokens and FI x 16 features: accumulators to
// row-major order through LDS in fp32 (16 tokens at a time, in space of this wave's
// own), so that the bias, the activation and the residual are added before the
// one rounding, then 8 features of a token per lane.
template <int EPI, int OUT, int FI, int FJ>
__device__ __forceinline__ void mx_epilogue(const MxGemmArgs& p, const f32x4_t (&acc)[FI][FJ], f32x4_t* stage, int m0,
                                            int n0, int lane) {
  constexpr int WTN = FI * 16, CPR = WTN / 8, RPP = 64 / CPR, NPASS = 16 / RPP;
  constexpr int ROW = WTN / 4 + 1;  // 16-byte units of a staged row, one spare: rows start 4 banks apart
  static_assert(16 % RPP == 0, "whole passes");
  const int ql = lane & 15, g = lane >> 4;
  const int c8 = lane % CPR, t0 = lane / CPR;
  const int n = n0 + c8 * 8;
  const int nc = min(n, p.N - 8);
  float bias[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x4_t b4 = p.bias != nullptr ? *reinterpret_cast<const f32x4_t*>(p.bias + nc + 4 * h) : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[4 * h + e] = b4[e];
  }
#pragma unroll
  for (int j = 0; j < FJ; ++j) {
    if (m0 + j * 16 >= p.M) break;  // the same for every lane
#pragma unroll
    for (int i = 0; i < FI; ++i) stage[ql * ROW + i * 4 + g] = acc[i][j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < NPASS; ++r) {
      const int t = r * RPP + t0, m = m0 + j * 16 + t;
      float y[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4_t v = stage[t * ROW + c8 * 2 + h];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[4 * h + e] = v[e] + bias[4 * h + e];
      }
      const bool on = m < p.M && n < p.N;
      const int mc = min(m, p.M - 1);
      if (EPI == MXE_GELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = gelu_tanh_f(y[e]);
      } else if (EPI == MXE_SILU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = silu_f(y[e]);
      } else if (EPI == MXE_RES || EPI == MXE_GATE_RES) {
        float rv[8];
        unpack8(*reinterpret_cast<const u32x4_t*>(p.R + (int64_t)mc * p.ldr + nc), rv);
        if (EPI == MXE_GATE_RES) {
          const float* gp = p.gate + (int64_t)find_segment(p.cu, p.nseg, mc) * p.gate_stride + nc;
          const f32x4_t g0 = *reinterpret_cast<const f32x4_t*>(gp), g1 = *reinterpret_cast<const f32x4_t*>(gp + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[e] = fmaf(y[e], g0[e], rv[e]);
            y[e + 4] = fmaf(y[e + 4], g1[e], rv[e + 4]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] += rv[e];
        }
      }
      if (OUT == MXO_FP8) {
        // N is whole blocks of 32 (checked on the host): a quad is on or off as one.
        // What the tile holds behind N is padding.
        uint32_t q[2];
        uint32_t s = mx_quantise8<MX_FP8>(y, q);
        if (n >= p.N) {
          q[0] = q[1] = 0;
          s = 127;
        }
        if (m < p.M) {
          if (n < (int)mx_cols(p.N))
            *reinterpret_cast<u32x2_t*>(reinterpret_cast<uint8_t*>(p.C) + (int64_t)m * p.ldc + n) = u32x2_t{q[0], q[1]};
          if ((c8 & 3) == 0 && n < (int)mx_scale_bytes(p.N) * 32)
            p.Cs[(int64_t)m * p.ldcs + mx_scale_at(n >> 5)] = (uint8_t)s;
        }
      } else if (on) {
        *reinterpret_cast<u32x4_t*>(reinterpret_cast<bf16_t*>(p.C) + (int64_t)m * p.ldc + n) = pack8(y);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// WM x WN waves of FJ x 16 tokens by FI x 16 features each.
template <int EPI, int OUT, int FI, int FJ, int WM, int WN, int EU>
__global__ __launch_bounds__(WM * WN * 64, EU) void mx_gemm_kernel(MxGemmArgs p) {
  constexpr int GW = WM * WN, WTM = FJ * 16, WTN = FI * 16, GBM = WM * WTM, GBN = WN * WTN;
  constexpr int DA = GBM / 8 / GW, DW = GBN / 8 / GW;  // DMA instructions per wave and stage, 8 rows each
  constexpr int ROWS = GBM + GBN, SG = ROWS / 64;      // scale DMA instructions of a workgroup and four stages
  constexpr int STAGE = ROWS * 8;                      // 16-byte units of a stage
  constexpr int EPI_UNITS = GW * 16 * (WTN / 4 + 1);
  constexpr int UNITS = 2 * STAGE + 2 * ROWS;
  static_assert(DA >= 1 && DW >= 1 && DA * GW * 8 == GBM && DW * GW * 8 == GBN && ROWS % 64 == 0, "tile");
  static_assert(GBN % 128 == 0, "an MX output's column padding lies within the last tile");
  __shared__ u32x4_t lds[UNITS > EPI_UNITS ? UNITS : EPI_UNITS];
  u32x4_t* const sc_lds = lds + 2 * STAGE;

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
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // stage kt is here for every wave; the other buffer is read out
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
  __syncthreads();  // every wave's operand reads are done: the space becomes the staging rows
  if (OUT == MXO_FP8 && n0 + GBN >= p.N) {
    // the scales behind the last tile, up to the row's multiple of 16 (the data's
    // padding, up to a multiple of 128 columns, lies within the tile)
    const int b0 = (n0 + GBN) / 32, nb = (int)mx_scale_bytes(p.N) - b0;
    for (int i = tid; i < GBM * nb; i += GW * 64)
      if (m0 + i / nb < p.M) p.Cs[(int64_t)(m0 + i / nb) * p.ldcs + mx_scale_at(b0 + i % nb)] = 127;
  }
  mx_epilogue<EPI, OUT, FI, FJ>(p, acc, reinterpret_cast<f32x4_t*>(lds) + wave * (16 * (WTN / 4 + 1)), m0 + a_row0,
                                n0 + w_row0, lane);
}

// Tile order: groups of m-tiles walked m-fastest, so the tiles running together share
// operand rows in their XCD's L2.
int mx_group_m(int K, int tiles_n) { return K >= 8192 ? 2 : (tiles_n >= 24 ? 4 : 8); }

template <int EPI, int OUT, int FI, int FJ, int WM, int WN, int EU>
int launch(MxGemmArgs p, hipStream_t stream) {
  constexpr int GBM = WM * FJ * 16, GBN = WN * FI * 16;
  p.tiles_m = (p.M + GBM - 1) / GBM;
  p.tiles_n = (p.N + GBN - 1) / GBN;
  p.group_m = mx_group_m(p.K, p.tiles_n);
  const int64_t blocks = ((int64_t)p.tiles_m * p.tiles_n + 7) / 8 * 8;
  DITK_REQUIRE(blocks < (1ll << 31), "ditk_mx_gemm: grid too large");
  mx_gemm_kernel<EPI, OUT, FI, FJ, WM, WN, EU><<<(unsigned)blocks, WM * WN * 64, 0, stream>>>(p);
  return ditk_check_launch("ditk_mx_gemm");
}

template <int EPI, int OUT>
int launch_tile(const MxGemmArgs& p, hipStream_t stream) {
  if ((int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256) >= 128) return launch<EPI, OUT, 4, 8, 2, 4, 1>(p, stream);
  return launch<EPI, OUT, 4, 2, 2, 2, 2>(p, stream);
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
  DITK_REQUIRE(!res || ((R || M == 0) && ldr % 8 == 0 && ldr >= N && ((uintptr_t)R % 16) == 0),
               "ditk_mx_gemm: residual epilogue needs a 16-byte aligned R with ldr %% 8 == 0");
  DITK_REQUIRE(epilogue != MXE_GATE_RES || (gate && cu_seqlens && nseg > 0 && gate_stride % 4 == 0 &&
                                            ((uintptr_t)gate % 16) == 0),
               "ditk_mx_gemm: gated epilogue needs 16-byte aligned gate rows and cu_seqlens");
  if (M == 0) return 0;
  const MxGemmArgs p{(const uint8_t*)A, lda, (const uint8_t*)As, ldas, (const uint8_t*)W, ldw, (const uint8_t*)Ws, ldws,
                     bias, C, ldc, (uint8_t*)Cs, ldcs, (const bf16_t*)R, ldr, gate, gate_stride, cu_seqlens, nseg,
                     M, N, K, 0, 0, 0};
  const bool mx = out_kind == MXO_FP8;
  switch (epilogue) {
    case MXE_BIAS: return mx ? launch_tile<MXE_BIAS, MXO_FP8>(p, stream) : launch_tile<MXE_BIAS, MXO_BF16>(p, stream);
    case MXE_GELU: return mx ? launch_tile<MXE_GELU, MXO_FP8>(p, stream) : launch_tile<MXE_GELU, MXO_BF16>(p, stream);
    case MXE_SILU: return mx ? launch_tile<MXE_SILU, MXO_FP8>(p, stream) : launch_tile<MXE_SILU, MXO_BF16>(p, stream);
    case MXE_RES: return launch_tile<MXE_RES, MXO_BF16>(p, stream);
    default: return launch_tile<MXE_GATE_RES, MXO_BF16>(p, stream);
  }
}
