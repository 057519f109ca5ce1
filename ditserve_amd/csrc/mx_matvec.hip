// Products of a few bf16 rows with a 4-bit microscaled (MX) weight, with fused epilogues.
//
//   C[m, n] = epilogue( sum_k x[m, k] v[n, k] 2^e[n, k / 32]  + bias[n] )
//
// Bound by streaming the weight once, 4.25 bits a value.  A wave takes
// 16 features at a time: lane (ql = lane % 16, g = lane / 16) loads the 16 bytes of block 4 c + g
// of weight row ql -- 32 weights under one scale -- which the convert instructions turn
// into bf16, exactly (an e2m1 value times a power of two), for four MFMAs of 16 features x
// 16 tokens x 32 k.  The MFMAs' k order is a permutation of the row's (MFMA t takes k 32 g
// + 8 t .. + 7 of each lane group), the same for both operands.
//
// The four waves of a workgroup share its features and split K; they join in LDS in a
// fixed order, which depends on K alone: a row's result does not depend on M.
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

template <int EPI, int FJ>
__global__ __launch_bounds__(256) void mx_matvec_kernel(const bf16_t* __restrict__ x, int64_t ldx,
                                                        const uint8_t* __restrict__ W, int64_t ldw,
                                                        const uint8_t* __restrict__ Ws, int64_t ldws,
                                                        const float* __restrict__ bias, void* Cv, int64_t ldc, int M,
                                                        int N, int K, const bf16_t* R, int64_t ldr) {
  __shared__ f32x4_t part[3][FJ][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ql = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (16 * FJ);
  const int blocks = K / 32, steps = (blocks + 3) / 4;  // 128-k steps
  const int row = min(n0 + ql, N - 1);
  const uint8_t* wp = W + (int64_t)row * ldw + g * 16;
  const uint8_t* sp = Ws + (int64_t)row * ldws + g * 4;
  const bf16_t* xp[FJ];
#pragma unroll
  for (int j = 0; j < FJ; ++j) xp[j] = x + (int64_t)min(m0 + j * 16 + ql, M - 1) * ldx + g * 32;
  f32x4_t acc[FJ];
#pragma unroll
  for (int j = 0; j < FJ; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int c = wave; c < steps; c += 4) {
    const u32x4_t w = *reinterpret_cast<const u32x4_t*>(wp + (int64_t)c * 64);
    const float s = e8m0_to_f32(sp[(c >> 2) * 16 + (c & 3)]);
    const bool on = c * 4 + g < blocks;  // else padding: zeros, past the end of x
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const bf16x8_t wf = fp4_to_bf16(w[t], s);
#pragma unroll
      for (int j = 0; j < FJ; ++j) {
        const u32x4_t xr = on ? *reinterpret_cast<const u32x4_t*>(xp[j] + (int64_t)c * 128 + t * 8) : u32x4_t{0, 0, 0, 0};
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, __builtin_bit_cast(bf16x8_t, xr), acc[j], 0, 0, 0);
      }
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int j = 0; j < FJ; ++j) part[wave - 1][j][lane] = acc[j];
  }
  __syncthreads();
  if (wave > 0) return;
  // this lane: token ql of each 16, features n .. n + 3
  const int n = n0 + 4 * g;
  if (n >= N) return;
  const f32x4_t b4 = bias != nullptr ? *reinterpret_cast<const f32x4_t*>(bias + n) : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < FJ; ++j) {
    const int m = m0 + j * 16 + ql;
    if (m >= M) continue;
    f32x4_t y = ((acc[j] + part[0][j][lane]) + (part[1][j][lane] + part[2][j][lane])) + b4;
    if (EPI == MV_F32) {
      *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(Cv) + (int64_t)m * ldc + n) = y;
      continue;
    }
    if (EPI == MV_GELU) {
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = gelu_tanh_f(y[e]);
    } else if (EPI == MV_SILU) {
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = silu_f(y[e]);
    } else if (EPI == MV_RES) {
      const u32x2_t r = *reinterpret_cast<const u32x2_t*>(R + (int64_t)m * ldr + n);
      y[0] += __uint_as_float(r[0] << 16);
      y[1] += __uint_as_float(r[0] & 0xffff0000u);
      y[2] += __uint_as_float(r[1] << 16);
      y[3] += __uint_as_float(r[1] & 0xffff0000u);
    }
    *reinterpret_cast<u32x2_t*>(reinterpret_cast<bf16_t*>(Cv) + (int64_t)m * ldc + n) =
        u32x2_t{pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3])};
  }
}

template <int EPI>
int launch(const void* x, int64_t ldx, const void* W, int64_t ldw, const void* Ws, int64_t ldws, const float* bias,
           void* C, int64_t ldc, int M, int N, int K, const void* R, int64_t ldr, hipStream_t stream) {
  const int fj = M <= 16 ? 1 : M <= 32 ? 2 : 4;
  const dim3 grid((unsigned)((N + 15) / 16), (unsigned)((M + 16 * fj - 1) / (16 * fj)));
  auto kern = fj == 1 ? mx_matvec_kernel<EPI, 1> : fj == 2 ? mx_matvec_kernel<EPI, 2> : mx_matvec_kernel<EPI, 4>;
  kern<<<grid, 256, 0, stream>>>((const bf16_t*)x, ldx, (const uint8_t*)W, ldw, (const uint8_t*)Ws, ldws, bias, C, ldc,
                                 M, N, K, (const bf16_t*)R, ldr);
  return ditk_check_launch("ditk_mx_matvec");
}

}  // namespace

DITK_EXPORT int ditk_mx_matvec(const void* x, int64_t ldx, const void* W, int64_t ldw, const void* Ws, int64_t ldws,
                               const float* bias, void* C, int64_t ldc, int M, int N, int K, int epilogue,
                               const void* R, int64_t ldr, hipStream_t stream) {
  DITK_REQUIRE(W && Ws && (M == 0 || (x && C)), "ditk_mx_matvec: null operand");
  DITK_REQUIRE(M >= 0 && N > 0 && K > 0, "ditk_mx_matvec: bad shape M=%d N=%d K=%d", M, N, K);
  DITK_REQUIRE(K % 32 == 0 && N % 8 == 0, "ditk_mx_matvec: K=%d must be a multiple of 32, N=%d of 8", K, N);
  DITK_REQUIRE(M <= 65535 * 64, "ditk_mx_matvec: too many rows");
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
