// Microscaled (MX) matrices, as every ditk_mx_* entry point reads and writes them.
//
// A block of 32 consecutive columns of a row has one scale 2^e, stored as the byte
// e + 127 (e8m0; 255 = NaN), and its values over that scale in e4m3 (fp8, a byte
// each) or e2m1 (fp4, the even column in the low half of a byte).  The quantiser takes
//   e = max(ceil(log2(amax / vmax)), -126),   vmax = 448 or 6,
// the smallest power of two that no value clips at, and rounds to nearest even.
// Rows are padded with zeros to a multiple of 128 columns (one MFMA of 16 x 16 x
// 128); scales with 2^0 to a multiple of 16 blocks.  Within 16 blocks the scale of
// block 4 s + g is byte 4 g + s: an MFMA lane of group g (= lane / 16) needs block
// g of each 128-column step, so its scales of four steps are one aligned dword, whose
// byte the instruction selects.
#pragma once

#include "ditk_common.h"

enum MxFmt : int { MX_FP8 = 0, MX_FP4 = 1 };

typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8_t;
typedef __attribute__((__vector_size__(2 * sizeof(short)))) short s16x2_t;

// The longest row, and the most rows of a product's output: column and row numbers of whole tiles past the last one
// stay below 2^31.
constexpr int kMxMaxCols = 1 << 30, kMxMaxRows = 0x70000000;

// columns a row of K holds with its padding, and bytes of its scales
__host__ __device__ inline int64_t mx_cols(int64_t K) { return (K + 127) / 128 * 128; }
__host__ __device__ inline int64_t mx_scale_bytes(int64_t K) { return (K + 511) / 512 * 16; }

// largest of three magnitudes; a NaN among them stays (v_max3_f32 would drop it)
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float m;
  asm("v_maximum3_f32 %0, |%1|, |%2|, |%3|" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}

// max over the four lanes l % 16 + 16 g: what permlane32_swap and permlane16_swap exchange
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max(b[0], b[1]);
}

// max over the four lanes of a quad (lanes 4 q .. 4 q + 3): DPP quad permutes
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));  // lanes 1, 0, 3, 2
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));  // lanes 2, 3, 0, 1
}

// Quantises 8 consecutive values per lane, four lanes of which hold one block of 32: a
// quad, or (GROUPS) the lanes l % 16 + 16 g.  Returns the block's scale byte and the values' bytes (fp8: q[0..1], fp4:
// q[0]).  The largest magnitude keeps an infinity or a NaN: such a block gets the scale NaN, and NaN
// values in fp8.
template <int FMT, bool GROUPS = false>
__device__ __forceinline__ uint32_t mx_quantise8(const float (&v)[8], uint32_t (&q)[2]) {
  const float m = max3_abs(max3_abs(max3_abs(v[0], v[1], v[2]), v[3], v[4]), max3_abs(v[5], v[6], v[7]), 0.f);
  uint32_t a = __float_as_uint(m) & 0x7fffffffu;
  a = GROUPS ? group_max(a) : quad_max(a);
  // amax = m 2^x with m in [1, 2): amax <= vmax 2^(x - 8) exactly when m <= 1.75
  // (vmax = 1.75 2^8), amax <= 6 2^(x - 2) when m <= 1.5: a mantissa above that carries into
  // the exponent field when the rest of the way to 2 is added
  constexpr uint32_t kUp = FMT == MX_FP8 ? 0x1fffffu : 0x3fffffu;
  constexpr int kBias = FMT == MX_FP8 ? 8 : 2;
  const int byte = max((int)((a + kUp) >> 23) - kBias, 1);
  const float scale = __uint_as_float((uint32_t)byte << 23);  // 2^e; the conversions divide by it, exactly
  if (FMT == MX_FP8) {
    s16x2_t w0 = {0, 0}, w1 = {0, 0};
    w0 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w0, v[0], v[1], scale, false);
    w0 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w0, v[2], v[3], scale, true);
    w1 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w1, v[4], v[5], scale, false);
    w1 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w1, v[6], v[7], scale, true);
    q[0] = __builtin_bit_cast(uint32_t, w0);
    q[1] = __builtin_bit_cast(uint32_t, w1);
  } else {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
    q[0] = w;
    q[1] = 0;
  }
  if (a >= 0x7f800000u) {
    q[0] = q[1] = FMT == MX_FP8 ? 0x7f7f7f7fu : 0u;
    return 255;
  }
  return (uint32_t)byte;
}

// byte of block b's scale within its row
__device__ __forceinline__ int mx_scale_at(int b) { return (b & ~15) | ((b & 3) << 2) | ((b >> 2) & 3); }

// Stores chunk c (columns 8 c .. 8 c + 7) of a row as the MX matrix's, by a wave whose
// lane is c % 64; chunks past the row's `nchunk` are its padding.
template <int FMT>
__device__ __forceinline__ void mx_store_chunk(const float (&v)[8], int c, int nchunk, uint8_t* __restrict__ data,
                                               uint8_t* __restrict__ scales) {
  uint32_t q[2];
  uint32_t s = mx_quantise8<FMT>(v, q);
  if (c >= nchunk) {
    q[0] = q[1] = 0;
    s = 127;
  }
  if (c * 8 < (int)mx_cols(nchunk * 8)) {
    if (FMT == MX_FP8) *reinterpret_cast<u32x2_t*>(data + (int64_t)c * 8) = u32x2_t{q[0], q[1]};
    else *reinterpret_cast<uint32_t*>(data + (int64_t)c * 4) = q[0];
  }
  if ((c & 3) == 0) scales[mx_scale_at(c >> 2)] = (uint8_t)s;
}
