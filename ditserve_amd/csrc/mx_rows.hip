// Row kernels that write microscaled (MX) matrices: the quantiser, and the row norm
// (RMSNorm or LayerNorm, affine, per-segment modulation) with the residual's addition
// before it and the MX output behind it.
//
// Both move each row once and are HBM-bound.  A wave takes 512 columns at a time, 16
// bytes per lane; 8 columns a lane make a block of 32 one quad, whose largest
// magnitude two DPP permutes give.
#include "mx_common.h"

namespace {

constexpr int kRowsPerBlock = 4;  // 4 waves, one row (or 512 columns of one) each
constexpr int kMaxChunks = 12;    // 16-byte chunks per lane -> D <= 64 * 8 * 12 = 6144

// A grid's first dimension holds less than 2^32 threads (more wrap around, and no error is reported): it takes the
// rows of 2^24 waves at most, `rows` of them, and the second dimension the next.
struct RowGrid {
  dim3 grid;
  int rows;
};
constexpr int kMaxGridY = 65535;
RowGrid row_grid(int T, int waves_per_row) {
  const int most = (1 << 24) / waves_per_row, rows = T < most ? T : most;
  const int waves = rows * waves_per_row;
  return RowGrid{dim3((unsigned)((waves + kRowsPerBlock - 1) / kRowsPerBlock), (unsigned)((T - 1) / rows + 1)), rows};
}

template <int FMT>
__global__ __launch_bounds__(256) void mx_quantise_kernel(const bf16_t* __restrict__ x, int64_t ldx,
                                                          uint8_t* __restrict__ data, int64_t ldd,
                                                          uint8_t* __restrict__ scales, int64_t lds, int T, int rows,
                                                          int per_row, int nchunk) {
  const uint32_t u = blockIdx.x * kRowsPerBlock + (threadIdx.x >> 6), part = u / (uint32_t)per_row;
  const int64_t row = (int64_t)blockIdx.y * rows + part;
  if (part >= (uint32_t)rows || row >= T) return;
  const int c = (int)(u - part * (uint32_t)per_row) * 64 + (threadIdx.x & 63);
  const u32x4_t raw = c < nchunk ? *reinterpret_cast<const u32x4_t*>(x + row * ldx + c * 8) : u32x4_t{0, 0, 0, 0};
  float v[8];
  unpack8(raw, v);
  mx_store_chunk<FMT>(v, c, nchunk, data + row * ldd, scales + row * lds);
}

// s = x (+ r) in fp32, h = s rounded, then the norm of the unrounded s: one wave per
// row, the row in registers.
template <int KIND, int NC>
__global__ __launch_bounds__(256) void mx_norm_kernel(
    const bf16_t* x, int64_t ldx, const bf16_t* r, int64_t ldr, bf16_t* h, int64_t ldh, uint8_t* __restrict__ data,
    int64_t ldd, uint8_t* __restrict__ scales, int64_t lds, int T, int D, const int32_t* __restrict__ cu, int nseg,
    const float* __restrict__ shift, const float* __restrict__ scale, int64_t mod_stride, const float* __restrict__ w,
    const float* __restrict__ b, float eps) {
  // (whole workgroups in the first dimension: its rows are a multiple of theirs, or all)
  const int64_t at = (int64_t)blockIdx.y * (1 << 24) + blockIdx.x * kRowsPerBlock + (threadIdx.x >> 6);
  if (at >= T) return;
  const int row = (int)at;
  const int lane = threadIdx.x & 63;
  const int nchunk = D >> 3;
  const bf16_t* xr = x + (int64_t)row * ldx;
  float v[NC][8];
  u32x4_t raw[NC], rraw[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = i * 64 + lane;
    raw[i] = c < nchunk ? *reinterpret_cast<const u32x4_t*>(xr + c * 8) : u32x4_t{0, 0, 0, 0};
  }
  if (r != nullptr) {
    const bf16_t* rr = r + (int64_t)row * ldr;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = i * 64 + lane;
      rraw[i] = c < nchunk ? *reinterpret_cast<const u32x4_t*>(rr + c * 8) : u32x4_t{0, 0, 0, 0};
    }
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) unpack8(raw[i], v[i]);
  if (r != nullptr) {
    // a lane reads its chunks of x and r before it writes them: h may be either
    bf16_t* hr = h + (int64_t)row * ldh;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = i * 64 + lane;
      float t[8];
      unpack8(rraw[i], t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += t[j];
      if (c < nchunk) *reinterpret_cast<u32x4_t*>(hr + c * 8) = pack8(v[i]);
    }
  }
  float mean = 0.f;
  if (KIND == 0) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[i][j];
    mean = wave_sum<64>(s) / (float)D;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NC; ++i)
    if (i * 64 + lane < nchunk)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = v[i][j] - mean;
        q = fmaf(d, d, q);
      }
  const float rstd = rsqrtf(wave_sum<64>(q) / (float)D + eps);
  const float* sh = nullptr;
  const float* sc = nullptr;
  if (shift != nullptr) {
    const int seg = find_segment(cu, nseg, row);
    sh = shift + (int64_t)seg * mod_stride;
    sc = scale + (int64_t)seg * mod_stride;
  }
  auto load8 = [](const float* p, float (&out)[8]) {
    const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(p);
    const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      out[j] = lo[j];
      out[j + 4] = hi[j];
    }
  };
  uint8_t* dr = data + (int64_t)row * ldd;
  uint8_t* sr = scales + (int64_t)row * lds;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = i * 64 + lane;
    const int cc = min(c, nchunk - 1) * 8;
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = (v[i][j] - mean) * rstd;
    if (w != nullptr) {
      load8(w + cc, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= t[j];
    }
    if (b != nullptr) {
      load8(b + cc, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += t[j];
    }
    if (shift != nullptr) {
      float s8[8];
      load8(sc + cc, s8);
      load8(sh + cc, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * (1.0f + s8[j]) + t[j];
    }
    if (i * 512 < (int)mx_scale_bytes(D) * 32) mx_store_chunk<MX_FP8>(v[i], c, nchunk, dr, sr);
  }
}

int mx_out_check(const char* what, const void* data, int64_t ldd, const void* scales, int64_t lds, int T, int K,
                 int fmt) {
  DITK_REQUIRE(T == 0 || (data && scales), "%s: null MX output", what);
  DITK_REQUIRE(K > 0 && K % 32 == 0, "%s: %d columns are not blocks of 32", what, K);
  DITK_REQUIRE(K <= kMxMaxCols, "%s: %d columns are too long", what, K);
  DITK_REQUIRE(ldd % 16 == 0 && ldd >= mx_cols(K) >> (fmt == MX_FP4) && lds % 16 == 0 && lds >= mx_scale_bytes(K),
               "%s: MX rows need their padding and 16-byte strides", what);
  DITK_REQUIRE(((uintptr_t)data % 16) == 0 && ((uintptr_t)scales % 16) == 0,
               "%s: MX data and scales must be 16-byte aligned", what);
  return 0;
}

}  // namespace

DITK_EXPORT int ditk_mx_quantize(const void* x, int64_t ldx, void* data, int64_t ldd, void* scales, int64_t lds,
                                 int T, int K, int fmt, hipStream_t stream) {
  DITK_REQUIRE(T >= 0 && (T == 0 || x), "ditk_mx_quantize: bad rows");
  DITK_REQUIRE(fmt == MX_FP8 || fmt == MX_FP4, "ditk_mx_quantize: unknown format %d", fmt);
  if (int rc = mx_out_check("ditk_mx_quantize", data, ldd, scales, lds, T, K, fmt)) return rc;
  DITK_REQUIRE(ldx % 8 == 0 && ldx >= K && ((uintptr_t)x % 16) == 0,
               "ditk_mx_quantize: x rows must be 16-byte aligned");
  if (T == 0) return 0;
  const int per_row = (K + 511) / 512;
  const RowGrid g = row_grid(T, per_row);
  DITK_REQUIRE(g.grid.y <= kMaxGridY, "ditk_mx_quantize: too many rows");
  auto kern = fmt == MX_FP8 ? mx_quantise_kernel<MX_FP8> : mx_quantise_kernel<MX_FP4>;
  kern<<<g.grid, 256, 0, stream>>>((const bf16_t*)x, ldx, (uint8_t*)data, ldd, (uint8_t*)scales, lds, T, g.rows,
                                   per_row, K / 8);
  return ditk_check_launch("ditk_mx_quantize");
}

DITK_EXPORT int ditk_mx_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* h, int64_t ldh,
                             void* data, int64_t ldd, void* scales, int64_t lds, int T, int D,
                             const int32_t* cu_seqlens, int nseg, const float* shift, const float* scale,
                             int64_t mod_stride, const float* weight, const float* bias, float eps, int norm_kind,
                             hipStream_t stream) {
  DITK_REQUIRE(T >= 0 && (T == 0 || x), "ditk_mx_norm: bad rows");
  DITK_REQUIRE(D <= 64 * 8 * kMaxChunks, "ditk_mx_norm: D=%d above %d", D, 64 * 8 * kMaxChunks);
  DITK_REQUIRE(norm_kind == 0 || norm_kind == 1, "ditk_mx_norm: unknown norm %d", norm_kind);
  if (int rc = mx_out_check("ditk_mx_norm", data, ldd, scales, lds, T, D, MX_FP8)) return rc;
  DITK_REQUIRE(ldx % 8 == 0 && ldx >= D && ((uintptr_t)x % 16) == 0, "ditk_mx_norm: x rows must be 16-byte aligned");
  DITK_REQUIRE(T == 0 || (residual == nullptr) == (h == nullptr), "ditk_mx_norm: residual and h go together");
  DITK_REQUIRE(residual == nullptr || (ldr % 8 == 0 && ldr >= D && ldh % 8 == 0 && ldh >= D &&
                                       ((uintptr_t)residual % 16) == 0 && ((uintptr_t)h % 16) == 0),
               "ditk_mx_norm: residual and h rows must be 16-byte aligned");
  DITK_REQUIRE((shift == nullptr) == (scale == nullptr), "ditk_mx_norm: shift and scale go together");
  DITK_REQUIRE(shift == nullptr || (cu_seqlens && nseg > 0 && mod_stride % 4 == 0), "ditk_mx_norm: bad modulation");
  DITK_REQUIRE(((uintptr_t)shift % 16) == 0 && ((uintptr_t)scale % 16) == 0 && ((uintptr_t)weight % 16) == 0 &&
                   ((uintptr_t)bias % 16) == 0,
               "ditk_mx_norm: vectors must be 16-byte aligned");
  if (T == 0) return 0;
  const dim3 grid = row_grid(T, 1).grid;
#define DITK_MXN(K, NCV)                                                                                         \
  mx_norm_kernel<K, NCV><<<grid, 256, 0, stream>>>((const bf16_t*)x, ldx, (const bf16_t*)residual, ldr, (bf16_t*)h, \
                                                   ldh, (uint8_t*)data, ldd, (uint8_t*)scales, lds, T, D, cu_seqlens, \
                                                   nseg, shift, scale, mod_stride, weight, bias, eps)
#define DITK_MXN_NC(K)             \
  switch ((D + 511) / 512) {       \
    case 1: DITK_MXN(K, 1); break; \
    case 2: DITK_MXN(K, 2); break; \
    case 3: DITK_MXN(K, 3); break; \
    case 4: DITK_MXN(K, 4); break; \
    case 5: DITK_MXN(K, 5); break; \
    case 6: DITK_MXN(K, 6); break; \
    case 7:                        \
    case 8: DITK_MXN(K, 8); break; \
    case 9:                        \
    case 10: DITK_MXN(K, 10); break; \
    default: DITK_MXN(K, 12); break; \
  }
  if (norm_kind == 0) {
    DITK_MXN_NC(0)
  } else {
    DITK_MXN_NC(1)
  }
#undef DITK_MXN_NC
#undef DITK_MXN
  return ditk_check_launch("ditk_mx_norm");
}
