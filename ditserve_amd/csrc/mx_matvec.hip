// Products of a few bf16 rows with a 4-bit microscaled (MX) weight, with fused epilogues.
//
//   C[m, n] = epilogue( sum_k x[m, k] v[n, k] 2^e[n, k / 32]  + bias[n] )
//
// Two kernels, bitwise alike, and a rule between them (mv_plan): one for few rows, one of tiles for more.
//
// Bound by streaming the weight once, 4.25 bits a value.  In the first a wave takes 16 features at a
// time: lane (ql = lane % 16, g = lane / 16) loads the 16 bytes of block 4 c + g of weight row
// ql -- 32 weights under one scale -- which the convert instructions turn into bf16,
// exactly (an e2m1 value times a power of two), for four MFMAs of 16 features x 16 tokens x 32
// k.  The MFMAs' k order is a permutation of the row's (MFMA u takes k 32 g + 8 u .. + 7 of each
// lane group), the same for both operands.
//
// A workgroup keeps its rows of x in LDS and goes through many groups of 16 features.  Its
// waves split K in chunks of 512 (a lane's four scales of a chunk are one dword) and join in LDS
// in wave order.  The split depends on K alone: a row's result does not depend on M.
//
// What bounds it: 2 x 1536 x 499712 (408 MB) 85 us, 4.8 TB/s, which is what a copy reaches here.  One
// short matrix takes the launch's 2.6 us, a memory latency for x and the first weights, and its
// own bytes: 1 x 1536 x 9216 4.7 us, 1 x 5120 x 5120 8.7, 1 x 8960 x 1536 7.1.  There the way of the code
// into the instruction cache counts too: with x in registers (its operands exchanged
// between lanes) and four chunks ahead, all unrolled, the large one took 85 us as well but the
// small one 7.9.
#include <algorithm>
#include <type_traits>

#include "mx_common.h"

namespace {

enum MvEpilogue : int { MV_BIAS = 0, MV_GELU = 1, MV_RES = 3, MV_F32 = 4, MV_SILU = 5 };

// 8 e2m1 values (one dword) times the block's scale -> bf16, exactly
__device__ __forceinline__ bf16x8_t fp4_to_bf16(uint32_t w, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// e8m0 byte -> fp32 (255: NaN)
__device__ __forceinline__ float e8m0_to_f32(uint32_t byte) {
  return byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}

// y (4 consecutive features of a row, before the bias) -> the output, from element `at`
template <int EPI>
__device__ __forceinline__ void finish4(f32x4_t y, const f32x4_t& b, const u32x2_t& r, void* Cv, int64_t at) {
  y += b;
  if (EPI == MV_F32) {
    *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(Cv) + at) = y;
    return;
  }
  if (EPI == MV_GELU) {
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = gelu_tanh_f(y[k]);
  } else if (EPI == MV_SILU) {
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = silu_f(y[k]);
  } else if (EPI == MV_RES) {
    y[0] += __uint_as_float(r[0] << 16);
    y[1] += __uint_as_float(r[0] & 0xffff0000u);
    y[2] += __uint_as_float(r[1] << 16);
    y[3] += __uint_as_float(r[1] & 0xffff0000u);
  }
  *reinterpret_cast<u32x2_t*>(reinterpret_cast<bf16_t*>(Cv) + at) = u32x2_t{pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3])};
}

constexpr int kMaxWaves = 16;
constexpr int kLds = 160 * 1024;
constexpr int D = 2;      // chunks of weights a wave has in registers or on their way (3: 0-3% slower, 4: 3-8%)
// Waves a CU is given where there are groups for them: 12 take 5-45% longer on the large matrices, 20 0-7%,
// 24 15-24%.
constexpr int kWavesPerCu = 16;

// A row of x in LDS: whole 128-k steps, 16 units of 16 bytes each, unit 4 u + g of a step holding k
// 32 g + 8 u .. + 7 (the operand of MFMA u and lane group g), XOR-swizzled by (row / 2) % 8, and
// 128 bytes more: the units that the lanes of an operand read together lie in different banks
// (as gemm.hip's operand rows).
__host__ __device__ inline int x_stride(int K) { return (int)mx_cols(K) * 2 + 128; }

// FJ x 16 tokens, of which a workgroup has x_rows
template <int EPI, int FJ>
__global__ __launch_bounds__(64 * kMaxWaves) void mx_matvec_kernel(const bf16_t* __restrict__ x, int64_t ldx,
                                                                   const uint8_t* __restrict__ W, int64_t ldw,
                                                                   const uint8_t* __restrict__ Ws, int64_t ldws,
                                                                   const float* __restrict__ bias, void* Cv,
                                                                   int64_t ldc, int M, int N, int K, const bf16_t* R,
                                                                   int64_t ldr, int x_rows) {
  extern __shared__ u32x4_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int ql = lane & 15, g = lane >> 4;
  auto part = reinterpret_cast<f32x4_t(*)[FJ][64]>(lds);  // [2 waves]: the partial sums of two groups in turn
  char* const xs = reinterpret_cast<char*>(lds + 2 * waves * FJ * 64);
  const int m0 = blockIdx.y * x_rows, rows = min(x_rows, M - m0), groups = (N + 15) / 16, stride = x_stride(K);
  const int blocks = K / 32, steps = (blocks + 3) / 4, chunks = (steps + 3) / 4;  // of 32, 128 and 512 k
  const int each = (chunks + waves - 1) / waves;  // a wave's chunks: wave, wave + waves, ...
  // this thread's output of a group: token ql of 16 ej, features n .. n + 3
  const int ej = threadIdx.x >> 6, m = m0 + ej * 16 + ql;
  const bool has_row = ej < FJ && ej * 16 + ql < rows;
  u32x4_t w[D][4];
  uint32_t s[D];
  f32x4_t b4[D], bcur;
  u32x2_t r2[D], rcur;
  // A chunk's weights (past the row's end its last 128 once more) and, with a group's first, its bias
  // and residual: loads return in order, and asked for later they would wait for the next weights.
  auto load = [&](int set, int group, int i) {
    if (i == 0) {
      const int n = group * 16 + 4 * g;
      const bool mine = has_row && n < N;
      b4[set] = mine && bias != nullptr ? *reinterpret_cast<const f32x4_t*>(bias + n) : f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (EPI == MV_RES)
        r2[set] = mine ? *reinterpret_cast<const u32x2_t*>(R + (int64_t)m * ldr + n) : u32x2_t{0, 0};
    }
    const int row = min(group * 16 + ql, N - 1), chunk = min(wave + i * waves, chunks - 1);
    s[set] = *reinterpret_cast<const uint32_t*>(Ws + (int64_t)row * ldws + chunk * 16 + g * 4);
    const uint8_t* wp = W + (int64_t)row * ldw + g * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      w[set][t] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(wp + min(chunk * 4 + t, steps - 1) * 64));
  };
  f32x4_t acc[FJ];
  const char* xl[FJ];
  int swz[FJ];
#pragma unroll
  for (int j = 0; j < FJ; ++j) {
    const int r = min(j * 16 + ql, rows - 1);
    xl[j] = xs + r * stride;
    swz[j] = (r >> 1) & 7;
  }
  auto use = [&](int set, int chunk) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int c = chunk * 4 + t;
      if (c >= steps) break;  // the same for the wave
      const float scale = e8m0_to_f32((s[set] >> (8 * t)) & 255);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bf16x8_t wf = fp4_to_bf16(w[set][t][u], scale);
#pragma unroll
        for (int j = 0; j < FJ; ++j)
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              wf, *reinterpret_cast<const bf16x8_t*>(xl[j] + c * 256 + (((u * 4 + g) ^ swz[j]) * 16)), acc[j], 0, 0, 0);
      }
    }
  };
  // the waves' sums of a group, joined, and the epilogue
  auto join = [&](int group, int buf) {
    const int n = group * 16 + 4 * g;
#pragma unroll
    for (int j = 0; j < FJ; ++j) part[buf * waves + wave][j][lane] = acc[j];
    // LDS only: the next weights stay on their way
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    if (!has_row || n >= N) return;
    f32x4_t y = part[buf * waves][ej][lane];
    for (int v = 1; v < waves; ++v) y += part[buf * waves + v][ej][lane];
    finish4<EPI>(y, bcur, rcur, Cv, (int64_t)m * ldc + n);
  };

  int group = blockIdx.x, i = 0, buf = 0;
  int lgroup = group, li = 0;  // the next chunk to ask for
  auto load_next = [&](int set) {
    if (lgroup >= groups) return;
    load(set, lgroup, li);
    if (++li == each) {
      li = 0;
      lgroup += gridDim.x;
    }
  };
#pragma unroll
  for (int d = 0; d < D - 1; ++d) load_next(d);
  // x: 512 k of a row per DMA instruction; past K zeros, under which weights count for nothing
  // (in a loop of their own: between the DMAs the compiler would wait for each)
  auto x_unit = [&](int p, bool tail) {
    const int r = p / chunks, c = p % chunks, v = lane ^ ((r >> 1) & 7);  // this lane's unit of the four steps
    const int k = c * 512 + (v >> 4) * 128 + (v & 3) * 32 + ((v >> 2) & 3) * 8;
    char* dst = xs + r * stride + c * 1024;
    if (!tail && k < K)
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(x + (int64_t)(m0 + r) * ldx + k),
          (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
    if (tail && k >= K && c * 4 + (lane >> 4) < steps)
      *reinterpret_cast<u32x4_t*>(dst + lane * 16) = u32x4_t{0, 0, 0, 0};
  };
  for (int p = wave; p < rows * chunks; p += waves) x_unit(p, false);
  if (K % 128 != 0)
    for (int p = wave; p < rows * chunks; p += waves) x_unit(p, true);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int j = 0; j < FJ; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // one chunk from `set`; false behind the last
  auto step = [&](int set) {
    load_next((set + D - 1) % D);
    if (i == 0) {
      bcur = b4[set];
      rcur = r2[set];
    }
    if (wave + i * waves < chunks) use(set, wave + i * waves);
    if (++i == each) {
      join(group, buf);
      buf ^= 1;
#pragma unroll
      for (int j = 0; j < FJ; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      i = 0;
      group += gridDim.x;
    }
    return group < groups;
  };
  for (;;) {
    bool more = true;
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (more) more = step(d);
    if (!more) break;
  }
}

// More rows than LDS holds, or more features than the first kernel streams well: tiles of 16 FJ tokens x 64 FI
// features, both operands through LDS in stages of 128 k (x rows of 256 bytes, weight rows of 64,
// their 16-byte units XOR-swizzled by row) by direct DMA into NBUF stages.  G groups of 4 waves share
// the k: `classes` is the first kernel's number of waves, class c its wave c's chunks, and a
// round is a class for each group, each with stages of its own; the classes' sums are added in
// order.  The same additions in the same order: bitwise the first kernel's results.
//
// 48 x 8960 x 51200 361 us on the first kernel (6 passes over the weight), 80 here; 1 x 5120 x 131072 97 and
// 76 (4.7 TB/s).  A tile's stage takes 0.3 us for the instructions of one wave a SIMD and 0.12 for
// each 16 tokens' LDS reads and MFMAs behind one another; more stages ahead (6, 7) change nothing.  Where tiles
// are few, two groups a tile take 0.6 of that; four 1.2 of what two take.
template <int EPI, int FJ, int FI, int NBUF, int G>
__global__ __launch_bounds__(256 * G) void mx_matvec_wide_kernel(const bf16_t* __restrict__ x, int64_t ldx,
                                                                 const uint8_t* __restrict__ W, int64_t ldw,
                                                                 const uint8_t* __restrict__ Ws, int64_t ldws,
                                                                 const float* __restrict__ bias, void* Cv, int64_t ldc,
                                                                 int M, int N, int K, const bf16_t* R, int64_t ldr,
                                                                 int classes) {
  constexpr int TN = 64 * FI, XU = 16 * FJ * 16, STAGE = XU + TN * 4;  // 16-byte units of a stage
  constexpr int DMAS = FJ + FI;                                        // per wave and stage
  // a group's stages, and the scales of four chunks of 512 k, 16 bytes a row: two stages ahead of the chunk that
  // is read may lie one of 128 k and the beginning of the next
  constexpr int GROUP = NBUF * STAGE + 4 * TN;
  __shared__ u32x4_t lds[G * GROUP];
  __shared__ f32x4_t part[G > 1 ? G - 1 : 1][G > 1 ? FI * FJ : 1][G > 1 ? 256 : 1];
  const int lane = threadIdx.x & 63, ql = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  const int q = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  u32x4_t* const ring = lds + q * GROUP;
  u32x4_t* const sc = ring + NBUF * STAGE;
  const int n0 = blockIdx.x * TN, m0 = blockIdx.y * (16 * FJ);
  const int blocks = K / 32, steps = (blocks + 3) / 4, chunks = (steps + 3) / 4;
  // the 128-k steps of a class; a round takes as many stages as the longest of its G classes
  auto steps_of = [&](int c) {
    if (c >= classes) return 0;
    return ((chunks - 1 - c) / classes + 1) * 4 - ((chunks - 1) % classes == c ? chunks * 4 - steps : 0);
  };
  auto stages_of = [&](int r) {
    int s = steps_of(r * G);
#pragma unroll
    for (int c = 1; c < G; ++c) s = max(s, steps_of(r * G + c));
    return s;
  };
  const int rounds = (classes + G - 1) / G;
  int left = 0;  // stages not yet computed
  for (int r = 0; r < rounds; ++r) left += stages_of(r);
  auto lds_at = [&](const void* at) {
    return (uint32_t)__builtin_amdgcn_readfirstlane(
        (int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)reinterpret_cast<const char*>(at));
  };
  // (as assembly, the waits below its own: for a DMA it sees the compiler would wait at every LDS read)
  auto dma = [&](const void* src, const void* dst) {
    asm volatile("s_mov_b32 m0, %0\n s_nop 0\n global_load_lds_dwordx4 %1, off" ::"s"(lds_at(dst)), "v"(src)
                 : "memory", "m0");
  };
  // DMA instruction d of this wave: x rows 4 (4 d + wave) .. + 3, weight rows 16 (4 d + wave) .. + 15
  const bf16_t* xsrc[FJ];
  int xk[FJ];
#pragma unroll
  for (int d = 0; d < FJ; ++d) {
    const int row = (d * 4 + wave) * 4 + (lane >> 4), v = (lane & 15) ^ (row & 15);
    xsrc[d] = x + (int64_t)min(m0 + row, M - 1) * ldx;
    xk[d] = (v & 3) * 32 + (v >> 2) * 8;  // unit 4 u + g: k 32 g + 8 u
  }
  const uint8_t* wsrc[FI];
#pragma unroll
  for (int d = 0; d < FI; ++d) {
    const int row = (d * 4 + wave) * 16 + (lane >> 2);
    wsrc[d] = W + (int64_t)min(n0 + row, N - 1) * ldw + (((lane & 3) ^ (row >> 2)) & 3) * 16;
  }
  const uint8_t* ssrc = Ws + (int64_t)min(n0 + wave * 16 * FI + (lane & (16 * FI - 1)), N - 1) * ldws;
  const uint8_t* zeros = W + K / 2;  // a weight row's padding behind K, where K % 128 != 0
  // A stage: step i of this group's class of round r.  Behind the class's end its last step is loaded again
  // (and not used): every stage is the same number of DMAs.
  int fr = 0, fi = 0, fn = stages_of(0), fbuf = 0, fchunk = 0;  // the next to load
  auto issue = [&]() {
    if (fr >= rounds) return;
    const int c = min(fr * G + q, classes - 1), chunk = min(c + (fi >> 2) * classes, chunks - 1);
    const int kt = min(chunk * 4 + (fi & 3), steps - 1);
    u32x4_t* st = ring + fbuf * STAGE;
    if ((fi & 3) == 0) {
      if (lane < 16 * FI) dma(ssrc + chunk * 16, sc + (fchunk & 3) * TN + wave * 16 * FI);
      ++fchunk;
    }
#pragma unroll
    for (int d = 0; d < FJ; ++d) {
      const int k = kt * 128 + xk[d];
      dma(k < K ? reinterpret_cast<const void*>(xsrc[d] + k) : zeros, st + (d * 4 + wave) * 64);
    }
#pragma unroll
    for (int d = 0; d < FI; ++d) dma(wsrc[d] + kt * 64, st + XU + (d * 4 + wave) * 64);
    fbuf = fbuf + 1 == NBUF ? 0 : fbuf + 1;
    if (++fi == fn) {
      fi = 0;
      fn = stages_of(++fr);
    }
  };
#pragma unroll
  for (int b = 0; b < NBUF - 1; ++b) issue();
  f32x4_t total[FI][FJ];
  int buf = 0, chunk = -1;
  for (int r = 0; r < rounds; ++r) {
    f32x4_t acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int mine = steps_of(r * G + q), n = stages_of(r);
    for (int s = 0; s < n; ++s, --left) {
      // this stage is here (behind it at most NBUF - 2 stages are on their way), and read by every wave is the
      // one whose buffer is filled next
      if (left >= NBUF - 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NBUF - 2) * DMAS) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const int t = s & 3;
      if (t == 0) ++chunk;
      // every operand is asked for before the next stage's DMAs and the first use: one LDS latency a stage
      const u32x4_t* st = ring + buf * STAGE;
      const uint32_t* s32 = reinterpret_cast<const uint32_t*>(sc + (chunk & 3) * TN);
      u32x4_t w[FI];
      uint32_t s4[FI];
      bf16x8_t xf[4][FJ];
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const int row = (wave * FI + i) * 16 + ql;
        s4[i] = s32[row * 4 + g];
        w[i] = st[XU + row * 4 + ((g ^ (row >> 2)) & 3)];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < FJ; ++j)
          xf[u][j] = __builtin_bit_cast(bf16x8_t, st[(j * 16 + ql) * 16 + ((u * 4 + g) ^ ql)]);
      __builtin_amdgcn_sched_barrier(0);
      issue();
      buf = buf + 1 == NBUF ? 0 : buf + 1;
      if (G > 1 && s >= mine) continue;  // the same for the wave
      float scale[FI];
#pragma unroll
      for (int i = 0; i < FI; ++i) scale[i] = e8m0_to_f32((s4[i] >> (8 * t)) & 255);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < FI; ++i) {
          const bf16x8_t wf = fp4_to_bf16(w[i][u], scale[i]);
#pragma unroll
          for (int j = 0; j < FJ; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[u][j], acc[i][j], 0, 0, 0);
        }
    }
    // the round's classes in order, in group 0 (its next write of `part` lies behind the next stage's barrier)
    if (G > 1) {
      if (q > 0) {
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
          for (int j = 0; j < FJ; ++j) part[q - 1][i * FJ + j][wave * 64 + lane] = acc[i][j];
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (q > 0) continue;
    }
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < FJ; ++j) {
        total[i][j] = r == 0 ? acc[i][j] : total[i][j] + acc[i][j];
#pragma unroll
        for (int c = 1; c < G; ++c)
          if (r * G + c < classes) total[i][j] += part[c - 1][i * FJ + j][wave * 64 + lane];
      }
  }
  if (q > 0) return;
#pragma unroll
  for (int i = 0; i < FI; ++i) {
    const int n = n0 + (wave * FI + i) * 16 + 4 * g;
    if (n >= N) continue;
    const f32x4_t b = bias != nullptr ? *reinterpret_cast<const f32x4_t*>(bias + n) : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      const int m = m0 + j * 16 + ql;
      if (m >= M) continue;
      u32x2_t r{0, 0};
      if (EPI == MV_RES) r = *reinterpret_cast<const u32x2_t*>(R + (int64_t)m * ldr + n);
      finish4<EPI>(total[i][j], b, r, Cv, (int64_t)m * ldc + n);
    }
  }
}

// Which kernel, in us beyond the launch.  The first streams the weight `passes` times, more slowly with fewer than
// some 12 waves on a CU.  Tiles take a time for each 128 k, however few they are: of 64 features and two
// groups up to one tile a CU, beyond that of 128 and one.  (16 x 5120 x 9216 18.5 us on the first kernel and
// 16.7 on tiles, x 5120 12.6 and 16.4; 48 x 8960 x 5120 44 and 33, 48 x 5120 x 5120 18.6 and 22; 1 x 1536 x 499712
// 81 and 88, 1 x 5120 x 131072 97 and 76; wrong by 8% at 64 x 5120 x 5120, 28 and 26.)
enum MvKernel : int { MV_STREAM = 0, MV_TILES64 = 1, MV_TILES128 = 2 };
struct MvPlan {
  MvKernel kernel;
  int fj;      // 16-token fragments of a workgroup
  int passes;  // over the weight, each of `rows` tokens but the last
  int rows;
  int waves;  // of the first kernel's workgroups: the classes of k
  int lds, per_cu;
};

int mv_plan(int M, int N, int K, MvPlan& p) {
  // waves: a chunk of 512 k each up to kMaxWaves, beyond that as even a share as there is
  const int chunks = (K - 1) / 512 + 1, each = (chunks + kMaxWaves - 1) / kMaxWaves, waves = (chunks + each - 1) / each;
  DITK_REQUIRE(K <= kLds / 2, "ditk_mx_matvec: K=%d too long", K);
  // the rows of x that fit in LDS, up to 16 (or 32); more rows in as many even passes over the weight
  auto fit = [&](int fj) { return std::min(16 * fj, (kLds - 2 * waves * fj * 1024) / x_stride(K)); };
  DITK_REQUIRE(fit(1) > 0, "ditk_mx_matvec: K=%d too long", K);
  const int fj = waves > 1 && fit(2) > 0 && (M - 1) / fit(2) < (M - 1) / fit(1) ? 2 : 1;
  const int passes = (M - 1) / fit(fj) + 1;
  DITK_REQUIRE(passes <= 65535, "ditk_mx_matvec: too many rows");  // and no more tiles
  const int x_rows = (M + passes - 1) / passes, lds = 2 * waves * fj * 1024 + x_rows * x_stride(K);
  const int per_cu = std::max(1, std::min(kWavesPerCu / waves, kLds / lds));
  const int steps = (K + 127) / 128, tall = (M + 63) / 64, wj = ((M + tall - 1) / tall + 15) / 16;
  const bool narrow = (int64_t)((N - 1) / 64 + 1) * tall <= ditk_cu_count();
  const float weight = (float)N / 68000.f;  // 128 k of the weight at 4.6 TB/s
  const float first = 3.f + (float)steps * weight * (float)passes * std::max(1.f, 12.f / (float)(per_cu * waves));
  const float tiles = narrow ? 4.5f + (float)steps * (0.22f + 0.065f * (float)wj)
                             : 3.2f + (float)steps * std::max(0.3f + 0.12f * (float)wj, weight * 1.05f * (float)tall);
  if (tiles < first) p = MvPlan{narrow ? MV_TILES64 : MV_TILES128, wj, tall, 16 * wj, waves, 0, 0};
  else p = MvPlan{MV_STREAM, fj, passes, x_rows, waves, lds, per_cu};
  return 0;
}

template <int EPI>
int launch(const void* x, int64_t ldx, const void* W, int64_t ldw, const void* Ws, int64_t ldws, const float* bias,
           void* C, int64_t ldc, int M, int N, int K, const void* R, int64_t ldr, hipStream_t stream) {
  MvPlan p;
  if (int rc = mv_plan(M, N, K, p)) return rc;
  if (p.kernel != MV_STREAM) {
    const bool narrow = p.kernel == MV_TILES64;
    const dim3 grid((unsigned)(narrow ? (N - 1) / 64 + 1 : (N - 1) / 128 + 1), (unsigned)p.passes);
    using Kernel = decltype(&mx_matvec_wide_kernel<EPI, 1, 1, 4, 2>);
    const Kernel tiles64[] = {mx_matvec_wide_kernel<EPI, 1, 1, 4, 2>, mx_matvec_wide_kernel<EPI, 2, 1, 4, 2>,
                              mx_matvec_wide_kernel<EPI, 3, 1, 3, 2>, mx_matvec_wide_kernel<EPI, 4, 1, 3, 2>};
    const Kernel tiles128[] = {mx_matvec_wide_kernel<EPI, 1, 2, 4, 1>, mx_matvec_wide_kernel<EPI, 2, 2, 4, 1>,
                               mx_matvec_wide_kernel<EPI, 3, 2, 3, 1>, mx_matvec_wide_kernel<EPI, 4, 2, 3, 1>};
    const Kernel kern = (narrow ? tiles64 : tiles128)[p.fj - 1];
    kern<<<grid, narrow ? 512 : 256, 0, stream>>>((const bf16_t*)x, ldx, (const uint8_t*)W, ldw, (const uint8_t*)Ws,
                                                  ldws, bias, C, ldc, M, N, K, (const bf16_t*)R, ldr, p.waves);
    return ditk_check_launch("ditk_mx_matvec");
  }
  const int groups = (N - 1) / 16 + 1;
  const dim3 grid((unsigned)std::min(groups, std::max(1, ditk_cu_count() * p.per_cu / p.passes)), (unsigned)p.passes);
  auto kern = p.fj == 1 ? mx_matvec_kernel<EPI, 1> : mx_matvec_kernel<EPI, 2>;
  kern<<<grid, 64 * p.waves, p.lds, stream>>>((const bf16_t*)x, ldx, (const uint8_t*)W, ldw, (const uint8_t*)Ws, ldws,
                                              bias, C, ldc, M, N, K, (const bf16_t*)R, ldr, p.rows);
  return ditk_check_launch("ditk_mx_matvec");
}

}  // namespace

DITK_EXPORT int ditk_mx_matvec(const void* x, int64_t ldx, const void* W, int64_t ldw, const void* Ws, int64_t ldws,
                               const float* bias, void* C, int64_t ldc, int M, int N, int K, int epilogue,
                               const void* R, int64_t ldr, hipStream_t stream) {
  DITK_REQUIRE(W && Ws && (M == 0 || (x && C)), "ditk_mx_matvec: null operand");
  DITK_REQUIRE(M >= 0 && N > 0 && K > 0, "ditk_mx_matvec: bad shape M=%d N=%d K=%d", M, N, K);
  DITK_REQUIRE(K % 32 == 0 && N % 8 == 0, "ditk_mx_matvec: K=%d must be a multiple of 32, N=%d of 8", K, N);
  DITK_REQUIRE(ldx % 8 == 0 && ldx >= K && ldw % 16 == 0 && ldw >= mx_cols(K) / 2 && ldws % 16 == 0 &&
                   ldws >= mx_scale_bytes(K),
               "ditk_mx_matvec: operand rows need their padding and 16-byte strides");
  DITK_REQUIRE(((uintptr_t)x % 16) == 0 && ((uintptr_t)W % 16) == 0 && ((uintptr_t)Ws % 16) == 0 &&
                   ((uintptr_t)C % 16) == 0 && ((uintptr_t)bias % 16) == 0,
               "ditk_mx_matvec: operands must be 16-byte aligned");
  DITK_REQUIRE(ldc % 8 == 0 && ldc >= N, "ditk_mx_matvec: ldc must be a multiple of 8 and >= N");
  DITK_REQUIRE(epilogue != MV_RES || ((R || M == 0) && ldr % 8 == 0 && ldr >= N && ((uintptr_t)R % 16) == 0),
               "ditk_mx_matvec: residual epilogue needs a 16-byte aligned R with ldr %% 8 == 0");
  if (M == 0) return 0;
  switch (epilogue) {
    case MV_BIAS: return launch<MV_BIAS>(x, ldx, W, ldw, Ws, ldws, bias, C, ldc, M, N, K, R, ldr, stream);
    case MV_GELU: return launch<MV_GELU>(x, ldx, W, ldw, Ws, ldws, bias, C, ldc, M, N, K, R, ldr, stream);
    case MV_RES: return launch<MV_RES>(x, ldx, W, ldw, Ws, ldws, bias, C, ldc, M, N, K, R, ldr, stream);
    case MV_F32: return launch<MV_F32>(x, ldx, W, ldw, Ws, ldws, bias, C, ldc, M, N, K, R, ldr, stream);
    case MV_SILU: return launch<MV_SILU>(x, ldx, W, ldw, Ws, ldws, bias, C, ldc, M, N, K, R, ldr, stream);
    default: ditk_set_error("ditk_mx_matvec: unknown epilogue %d", epilogue); return 1;
  }
}

DITK_EXPORT int ditk_mx_matvec_plan(int M, int N, int K, int* plan) {
  DITK_REQUIRE(plan && M > 0 && N > 0 && N % 8 == 0 && K > 0 && K % 32 == 0, "ditk_mx_matvec_plan: bad arguments");
  MvPlan p;
  if (int rc = mv_plan(M, N, K, p)) return rc;
  plan[0] = p.kernel;
  plan[1] = p.fj;
  plan[2] = p.passes;
  return 0;
}
