// Causal attention of packed segments with few queries over many keys (the next tokens of long prompts).
//
// The rows of a key head are its (query, query head) pairs.  A wave takes a chunk of a segment's keys for 16 rows of a key
// head (attn_chunk.h) and leaves its part in a workspace; a second kernel joins them in the chunks' order.
//
// 32 heads over 8 of 128: 16 queries after 8192 keys 25 + 10 us, the latency of a chunk's tiles and of the join's parts;
// 32 segments of 4 after 4000 106 + 10 (4.9 TB/s), memory.
#include "attn_chunk.h"
#include "causal_few.h"

namespace {

struct Args {
  const bf16_t *q, *k, *v;
  int64_t ldq, ldk, ldv;
  bf16_t* o;
  int64_t ldo;
  float* lse;
  int64_t lse_ld;
  const int32_t *cu_q, *cu_k;
  int nseg, kv_heads, group;
  float scale2;
  float* part;  // [parts][kv_heads][HD]: a segment's parts are its rows, each its chunks
  float* ml;    // [parts][kv_heads][2]
  int64_t parts;
};

struct Seg {
  int q0, nq, k0, nk, parts, units;
};
__device__ __forceinline__ Seg seg_of(const Args& a, int m) {
  Seg s;
  s.q0 = a.cu_q[m];
  s.nq = a.cu_q[m + 1] - s.q0;
  s.k0 = a.cu_k[m];
  s.nk = a.cu_k[m + 1] - s.k0;
  s.parts = few_parts(s.nq, s.nk, a.group);
  s.units = s.parts ? s.parts / (s.nq * a.group) * ((s.nq * a.group + 15) / 16) * a.kv_heads : 0;
  return s;
}

// Waves take units in order: a segment's chunks, for each its groups of 16 rows, for each the key heads, whose rows lie
// side by side.
template <int HD>
__global__ __launch_bounds__(256, 2) void causal_few_kernel(Args a) {
  using C = Chunk<HD, true>;
  __shared__ __align__(256) char lds[4 * 32 * HD * 2];
  __shared__ int ends[256], froms[256], sums[2][4];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int col = lane & 15, quad = lane >> 4;
  // units and parts up to and with thread t's segments, [t per, t per + per)
  const int per = (a.nseg + 255) / 256;
  int units = 0, parts = 0;
  for (int i = 0; i < per; ++i)
    if (tid * per + i < a.nseg) {
      const Seg s = seg_of(a, tid * per + i);
      units += s.units;
      parts += s.parts;
    }
  units = wave_scan(units);
  parts = wave_scan(parts);
  if (lane == 63) sums[0][wave] = units, sums[1][wave] = parts;
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    units += sums[0][w];
    parts += sums[1][w];
  }
  ends[tid] = units;
  froms[tid] = parts;
  __syncthreads();
  int end[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) end[i] = ends[i * 64 + lane];
  const int total = __builtin_amdgcn_readlane(end[3], 63);

  for (int u = blockIdx.x * 4 + wave; u < total; u += gridDim.x * 4) {
    int th = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) th += __popcll(__ballot(end[i] <= u));
    int m = th * per, unit = u - (th ? ends[th - 1] : 0), from = th ? froms[th - 1] : 0;
    Seg s = seg_of(a, m);
    while (unit >= s.units && m + 1 < a.nseg) {
      unit -= s.units;
      from += s.parts;
      s = seg_of(a, ++m);
    }
    const int all = s.nq * a.group, groups = (all + 15) / 16, chunk = unit / (groups * a.kv_heads);
    const int rest = unit - chunk * (groups * a.kv_heads), first = rest / a.kv_heads * 16, kvh = rest % a.kv_heads;
    const int rows = min(all - first, 16), nch = s.parts / all, len = few_chunk(s.nq, s.nk, a.group);
    // row r: query r / group, its head r % group; sees the keys below ahead + r / group
    const int ahead = s.nk - s.nq + 1, r0 = first + min(col, rows - 1);
    const int query = r0 / a.group, head = kvh * a.group + r0 - query * a.group;
    const int most = ahead + (first + rows - 1) / a.group;  // keys the last row sees
    const int s0 = min(chunk * len, most), s1 = min(s0 + len, most);
    C x;
    RowsSrc src{a.k + (int64_t)s.k0 * a.ldk + kvh * HD, a.v + (int64_t)s.k0 * a.ldv + kvh * HD, (int)a.ldk, (int)a.ldv,
                s.nk - 1};
    x.run(src, a.q + (int64_t)(s.q0 + query) * a.ldq + (int64_t)head * HD + quad * 8, a.scale2, s0, s1, ahead + query,
          ahead + first / a.group, nullptr, lds + wave * (32 * HD * 2));
    const int64_t at = (int64_t)from + (int64_t)r0 * nch + chunk;
    if (col < rows && at < a.parts) {
      float* pb = a.part + (at * a.kv_heads + kvh) * HD + quad * 4;
#pragma unroll
      for (int j = 0; j < C::ND; ++j) *reinterpret_cast<f32x4_t*>(pb + j * 16) = x.o[j];
      if (quad == 0) *reinterpret_cast<u32x2_t*>(a.ml + (at * a.kv_heads + kvh) * 2) =
          u32x2_t{__float_as_uint(x.m), __float_as_uint(x.l)};
    }
  }
}

// Joins the chunks of 16 rows of a (segment, key head), HD / 4 threads a row.  (A part without a finite score is 0, or NaN
// and stays it.)
template <int HD>
__global__ __launch_bounds__(16 * HD / 4) void causal_few_join_kernel(Args a) {
  constexpr int TPR = HD / 4, THREADS = 16 * TPR;
  __shared__ int sums[THREADS / 64];
  const int tid = threadIdx.x, units = a.nseg * a.kv_heads, first = blockIdx.x / units * 16, unit = blockIdx.x % units;
  const int kvh = unit % a.kv_heads, m = unit / a.kv_heads;
  const Seg s = seg_of(a, m);
  const int all = s.nq * a.group;
  if (s.parts == 0 || first >= all) return;
  int before = 0;
  for (int i = tid; i < m; i += THREADS) before += seg_of(a, i).parts;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) before += __shfl_xor(before, off, 64);
  if ((tid & 63) == 0) sums[tid >> 6] = before;
  __syncthreads();
  int64_t from = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) from += sums[i];
  const int r = first + tid / TPR, d = (tid % TPR) * 4, nch = s.parts / all;
  from += (int64_t)r * nch;
  if (r >= all || from + nch > a.parts) return;
  const float* ml = a.ml + (from * a.kv_heads + kvh) * 2;
  const float* part = a.part + (from * a.kv_heads + kvh) * HD + d;
  float top = -INFINITY;
#pragma unroll 8
  for (int c = 0; c < nch; ++c) top = fmaxf(top, ml[(int64_t)c * a.kv_heads * 2]);
  float l = 0.f;
  f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int c = 0; c < nch; ++c) {
    const u32x2_t e = *reinterpret_cast<const u32x2_t*>(ml + (int64_t)c * a.kv_heads * 2);
    const f32x4_t y = *reinterpret_cast<const f32x4_t*>(part + (int64_t)c * a.kv_heads * HD);
    const float mc = __uint_as_float(e[0]), f = mc == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mc - top);
    l = fmaf(__uint_as_float(e[1]), f, l);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fmaf(y[i], f, x[i]);
  }
  const int q = s.q0 + r / a.group, head = kvh * a.group + r % a.group;
  const float inv = inverse(l);
  *reinterpret_cast<u32x2_t*>(a.o + (int64_t)q * a.ldo + (int64_t)head * HD + d) =
      u32x2_t{pack_bf2(x[0] * inv, x[1] * inv), pack_bf2(x[2] * inv, x[3] * inv)};
  if (d == 0 && a.lse != nullptr) a.lse[(int64_t)head * a.lse_ld + q] = row_lse2(top, l) * 0.6931471805599453f;
}

}  // namespace

int64_t causal_few_workspace(int64_t parts, int kv_heads, int head_dim) { return parts * kv_heads * (head_dim + 2) * 4; }

int causal_few_launch(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* o,
                      int64_t ldo, float* lse, int64_t lse_ld, const int32_t* cu_q, const int32_t* cu_k, int nseg,
                      int heads, int kv_heads, int head_dim, float scale2, void* workspace, int64_t parts,
                      hipStream_t stream) {
  // units, parts and their places count in 32 bits
  const int64_t joins = (int64_t)nseg * kv_heads * (kFewRows / 16);
  DITK_REQUIRE(joins < (1 << 23) && (int64_t)nseg * kv_heads * 16 * kFewChunks < (1ll << 31),
               "ditk_flash_attn_causal: too many segments and heads");
  float* part = (float*)workspace;
  const Args a{(const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v, ldq, ldk, ldv, (bf16_t*)o, ldo, lse, lse_ld, cu_q, cu_k,
               nseg, kv_heads, heads / kv_heads, scale2, part, part + parts * kv_heads * head_dim, parts};
  // (a unit leaves at least one part a key head)
  const int64_t wgs = (parts * kv_heads + 3) / 4, most = 2 * ditk_cu_count();
  auto kern = head_dim == 128 ? causal_few_kernel<128> : causal_few_kernel<64>;
  kern<<<(unsigned)(wgs < most ? wgs : most), 256, 0, stream>>>(a);
  if (int rc = ditk_check_launch("ditk_flash_attn_causal")) return rc;
  auto join = head_dim == 128 ? causal_few_join_kernel<128> : causal_few_join_kernel<64>;
  join<<<(unsigned)joins, 16 * head_dim / 4, 0, stream>>>(a);
  return ditk_check_launch("ditk_flash_attn_causal");
}
