// Attention of one new token of each sequence over its paged keys and values (kv_common.h), split over the
// sequence's slots and joined.
//
// The G query heads of a key head make the columns of one matrix product: a wave takes 32 slots at a time,
//   S^T = K Q^T         (A = 16 slots x 32 dims straight from the pages, B = Q)
//   O^T += V^T P^T      (A = V^T by transposing LDS reads, B = P^T)
// with v_mfma_f32_16x16x32_bf16.  Row m of score tile t is slot 8 (m / 4) + 4 t + m % 4, so that the accumulators of both
// tiles are the 8 consecutive slots a lane of the second product's B operand holds: no shuffles between the two.
// P is taken as the sum of two bf16 numbers (16 bits of it at least), so that only the output is rounded to 8 bits: the
// matrix pipe is idle most of the time anyway.
//
// Scores are in log2 units; m, l and O stay fp32.  A chunk's length goes by the sequence's own length alone, so a
// sequence's result does not depend on what it is batched with.
#include "kv_common.h"

namespace {

constexpr int kMaxChunks = 512, kShortChunks = 8;

// slots of a chunk of a sequence of n, whole 32-slot tiles
__host__ __device__ inline int chunk_slots(int n) {
  if (n <= 1024) return 64;
  if (n <= 8192) return 128;
  if (n <= 65536) return 256;
  if (n <= 512 * kMaxChunks) return 512;
  return (int)(((int64_t)n + kMaxChunks * 128 - 1) / (kMaxChunks * 128) * 128);
}
__host__ __device__ inline int chunks_of(int n) { return n == 0 ? 1 : (n - 1) / chunk_slots(n) + 1; }

// the most chunks of any sequence up to `most` slots
int chunks_bound(int most) {
  int c = chunks_of(most);
  for (int n : {1024, 8192, 65536, 512 * kMaxChunks})
    if (n < most && chunks_of(n) > c) c = chunks_of(n);
  return most > 512 * kMaxChunks ? kMaxChunks : c;
}

struct Args {
  KvPages t;
  KvTensor k, v;
  KvWeights w;
  const bf16_t* q;
  int64_t ldq;
  bf16_t* o;
  int64_t ldo;
  float* lse;     // [batch * heads] natural log, or null
  float* lse2;    // [batch * heads] log2 units, for the weights
  float* part;    // [batch * heads][nchunk][HD]
  float* ml;      // [batch * heads][nchunk][2]
  float* score;   // [batch * heads][ld_score], or null
  int64_t ld_score;
  int heads, group, nchunk, batch, hgroups;  // hgroups: (key head, 16 of its query heads) pairs
  float scale2;   // softmax scale times log2 e
};

template <int HD>
__device__ __forceinline__ int v_swizzle(int row) {
  return HD == 128 ? (row & 3) | ((row >> 3) & 1) << 2 : ((row >> 1) & 1) | ((row >> 3) & 1) << 1;
}

__device__ __forceinline__ float group_maxf(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float group_sumf(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

// What a wave gathers of one chunk: lane (quad, col) holds dims 16 j + 4 quad .. + 3 of query head `col`'s sums of
// p v, its m and its l.
template <int HD, bool SCORES>
struct Chunk {
  static constexpr int NC = HD / 32, ND = HD / 16, CH = HD / 8, RPL = 64 / CH;  // RPL: rows of V a load of the wave covers
  f32x4_t o[ND];
  float m, l;

  // slots [s0, s1) of sequence b (n slots) and key head kvh, for nq query heads from head0 on; vt: 32 HD bf16 of LDS
  __device__ __forceinline__ void run(const Args& a, int b, int n, int s0, int s1, int kvh, int head0, int nq, char* vt) {
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int pl = a.t.page_log2, low = (1 << pl) - 1, last = max(n - 1, 0);
    bf16x8_t q[NC];
    const bf16_t* qr = a.q + b * a.ldq + (int64_t)(head0 + min(col, nq - 1)) * HD + quad * 8;
#pragma unroll
    for (int i = 0; i < NC; ++i) q[i] = *reinterpret_cast<const bf16x8_t*>(qr + i * 32);
#pragma unroll
    for (int j = 0; j < ND; ++j) o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
    int page = 0, first = 0;
    for (int t0 = s0; t0 < s1; t0 += 32) {
      // pages of the next 1024 slots, one a lane
      if (((t0 - s0) & 1023) == 0) {
        first = t0 >> pl;
        const int i = min(first + lane, last >> pl), p = a.t.table[b * a.t.ldt + i];
        page = (unsigned)p < (unsigned)a.t.pages ? p : -1;
        if (page < 0 && (first + lane) << pl < s1) *a.t.status = 1;
      }
      // the tile's two halves of 16 slots lie in one page each; slots past the last read it
      const int g0 = __builtin_amdgcn_readlane(page, (min(t0, last) >> pl) - first);
      const int g1 = __builtin_amdgcn_readlane(page, (min(t0 + 16, last) >> pl) - first);
      const bool ok0 = g0 >= 0, ok1 = g1 >= 0;
      const int p0 = max(g0, 0), p1 = max(g1, 0);
      const bf16_t* kb0 = a.k.p + p0 * a.k.ps + kvh * a.k.hs;
      const bf16_t* kb1 = a.k.p + p1 * a.k.ps + kvh * a.k.hs;
      const bf16_t* vb0 = a.v.p + p0 * a.v.ps + kvh * a.v.hs;
      const bf16_t* vb1 = a.v.p + p1 * a.v.ps + kvh * a.v.hs;
      bf16x8_t k[2][NC];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int slot = min(t0 + 8 * (col >> 2) + 4 * i + (col & 3), last);
        const bf16_t* kr = (col < 8 ? kb0 : kb1) + (int64_t)(slot & low) * HD + quad * 8;
#pragma unroll
        for (int c = 0; c < NC; ++c) k[i][c] = *reinterpret_cast<const bf16x8_t*>(kr + c * 32);
      }
      u32x4_t v[32 / RPL];
#pragma unroll
      for (int i = 0; i < 32 / RPL; ++i) {
        const int row = i * RPL + lane / CH, slot = min(t0 + row, last);
        v[i] = *reinterpret_cast<const u32x4_t*>((i * RPL < 16 ? vb0 : vb1) + (int64_t)(slot & low) * HD + (lane % CH) * 8);
      }
      // values of absent slots may be anything: they count as 0
      const int n0 = ok0 ? min(s1 - t0, 16) : 0, n1 = ok1 ? s1 - t0 - 16 : 0;
      const bool whole = n0 == 16 && n1 >= 16;
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 32 / RPL; ++i) {
          const int row = i * RPL + lane / CH;
          if (i * RPL < 16 ? row >= n0 : row - 16 >= n1) v[i] = u32x4_t{0, 0, 0, 0};
        }
      }
      f32x4_t s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[i][c], q[c], s[i], 0, 0, 0);
      }
      float x[8], top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = s[e >> 2][e & 3] * a.scale2;
        const int row = quad * 8 + e;
        if (!whole && (row < 16 ? row >= n0 : row - 16 >= n1)) x[e] = -INFINITY;
        top = fmaxf(top, x[e]);
      }
      if (SCORES) {
        if (col < nq) {
          float* sr = a.score + ((int64_t)b * a.heads + head0 + col) * a.ld_score + t0 + quad * 8;
          *reinterpret_cast<f32x4_t*>(sr) = f32x4_t{x[0], x[1], x[2], x[3]};
          *reinterpret_cast<f32x4_t*>(sr + 4) = f32x4_t{x[4], x[5], x[6], x[7]};
        }
      }
      const float mn = fmaxf(m, group_maxf(top));
      if (__any(mn > m)) {
        const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l *= al;
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[j][r] *= al;
        m = mn;
      }
      const float base = m == -INFINITY ? 0.f : m;
      bf16x8_t hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = __builtin_amdgcn_exp2f(x[e] - base);
        l += p;
        // hi cut off, so that lo is not negative, and lo not 0 unless p is: an infinite value stays one
        const float cut = __uint_as_float(__float_as_uint(p) & 0xffff0000u);
        hi[e] = __builtin_bit_cast(__bf16, (uint16_t)(__float_as_uint(p) >> 16));
        lo[e] = (__bf16)fmaxf(p - cut, fminf(p, 1.17549435e-38f));
      }
#pragma unroll
      for (int i = 0; i < 32 / RPL; ++i) {
        const int row = i * RPL + lane / CH, ch = lane % CH;
        *reinterpret_cast<u32x4_t*>(vt + row * (HD * 2) + (((ch >> 1) ^ v_swizzle<HD>(row)) * 32) + (ch & 1) * 16) = v[i];
      }
      // lane i of a quad reads 8 bytes of row i / 4 and gets 4 rows of column i
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        s16x4 w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = quad * 8 + 4 * i + (col >> 2);
          const char* p = vt + row * (HD * 2) + ((j ^ v_swizzle<HD>(row)) * 32) + (col & 3) * 8;
          w[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
        }
        union { s16x4 h[2]; bf16x8_t f; } f;
        f.h[0] = w[0];
        f.h[1] = w[1];
        o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.f, hi, o[j], 0, 0, 0);
        o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.f, lo, o[j], 0, 0, 0);
      }
    }
    l = group_sumf(l);
  }
};

// 1 / l, 0 for a row without slots
__device__ __forceinline__ float inverse(float l) { return l > 0.f || l != l ? 1.f / l : 0.f; }
__device__ __forceinline__ void store_lse(const Args& a, int64_t row, float m, float l, bool scores) {
  const float e = l > 0.f || l != l ? m + __builtin_amdgcn_logf(l) : -INFINITY;
  if (a.lse != nullptr) a.lse[row] = e * 0.6931471805599453f;
  if (scores) a.lse2[row] = e;
}

// A wave takes one chunk of one (sequence, key head, 16 query heads) after another; units go round the waves in
// order: a sequence's chunks, and for each its heads, which lie side by side in a page.
template <int HD, bool SCORES>
__global__ __launch_bounds__(256, 3) void kv_attn_kernel(Args a) {
  using C = Chunk<HD, SCORES>;
  __shared__ __align__(16) char lds[4 * 32 * HD * 2];
  __shared__ int sums[4], ends[256], lens[256];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int col = lane & 15, quad = lane >> 4;

  // chunks up to and with thread t's sequences, [t per, t per + per)
  const int per = (a.batch + 255) / 256;
  int incl = 0;
  for (int i = 0; i < per; ++i)
    if (tid * per + i < a.batch) {
      const int n = kv_length(a.t, tid * per + i, blockIdx.x == 0);
      if (i == 0) lens[tid] = n;
      incl += chunks_of(n);
    }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(incl, off, 64);
    if (lane >= off) incl += o;
  }
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  for (int w = 0; w < wave; ++w) incl += sums[w];
  ends[tid] = incl;
  __syncthreads();
  int end[4];  // (every wave keeps all of them)
#pragma unroll
  for (int i = 0; i < 4; ++i) end[i] = ends[i * 64 + lane];
  const int units = __builtin_amdgcn_readlane(end[3], 63) * a.hgroups, groups = (a.group + 15) / 16;

  for (int u = blockIdx.x * 4 + wave; u < units; u += gridDim.x * 4) {
    const int c = u / a.hgroups, hg = u - c * a.hgroups;
    // the thread whose sequences hold chunk c, then the sequence
    int th = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) th += __popcll(__ballot(end[i] <= c));
    int b = th * per, chunk = c - (th ? ends[th - 1] : 0), n = lens[th], nch = chunks_of(n);
    while (chunk >= nch && b + 1 < a.batch) {
      chunk -= nch;
      n = kv_length(a.t, ++b, false);
      nch = chunks_of(n);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    n = __builtin_amdgcn_readfirstlane(n);
    chunk = __builtin_amdgcn_readfirstlane(min(chunk, a.nchunk - 1));
    const int kvh = hg / groups, g0 = (hg - kvh * groups) * 16;
    const int csl = chunk_slots(n), s0 = chunk * csl, s1 = min(n, s0 + csl);
    const int nq = min(a.group - g0, 16), head0 = kvh * a.group + g0;  // query heads of this unit
    C x;
    x.run(a, b, n, s0, s1, kvh, head0, nq, lds + wave * (32 * HD * 2));
    if (col < nq) {
      const int64_t row = (int64_t)b * a.heads + head0 + col;
      if (nch == 1) {
        const float inv = inverse(x.l);
        bf16_t* ob = a.o + b * a.ldo + (int64_t)(head0 + col) * HD + quad * 4;
#pragma unroll
        for (int j = 0; j < C::ND; ++j)
          *reinterpret_cast<u32x2_t*>(ob + j * 16) = u32x2_t{pack_bf2(x.o[j][0] * inv, x.o[j][1] * inv),
                                                            pack_bf2(x.o[j][2] * inv, x.o[j][3] * inv)};
        if (quad == 0) store_lse(a, row, x.m, x.l, SCORES);
      } else {
        float* pb = a.part + (row * a.nchunk + chunk) * HD + quad * 4;
#pragma unroll
        for (int j = 0; j < C::ND; ++j) *reinterpret_cast<f32x4_t*>(pb + j * 16) = x.o[j];
        if (quad == 0) *reinterpret_cast<u32x2_t*>(a.ml + (row * a.nchunk + chunk) * 2) =
            u32x2_t{__float_as_uint(x.m), __float_as_uint(x.l)};
      }
    }
  }
}

// Sequences of up to 8 chunks in one launch: eight waves take a chunk each of a (sequence, key head, 16 query heads) and
// join them through LDS, by the join kernel's operations in its order.
template <int HD, bool SCORES>
__global__ __launch_bounds__(512) void kv_attn_short_kernel(Args a) {
  using C = Chunk<HD, SCORES>;
  constexpr int OP = HD + 4;  // floats of a row of LDS
  __shared__ __align__(16) char lds[8 * 16 * OP * 4];
  __shared__ float stat[2][16][8];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int col = lane & 15, quad = lane >> 4, groups = (a.group + 15) / 16;
  const int b = blockIdx.x / a.hgroups, hg = blockIdx.x - b * a.hgroups;
  const int kvh = hg / groups, g0 = (hg - kvh * groups) * 16;
  const int n = kv_length(a.t, b, hg == 0 && tid == 0), csl = chunk_slots(n), nch = chunks_of(n);
  const int s0 = min(wave * csl, n), s1 = min(n, s0 + csl);
  const int nq = min(a.group - g0, 16), head0 = kvh * a.group + g0;
  C x;
  x.run(a, b, n, s0, s1, kvh, head0, nq, lds + wave * (16 * OP * 4));
  if (quad == 0) {
    stat[0][col][wave] = x.m;
    stat[1][col][wave] = x.l;
  }
  // (a wave's rows lie where its values were, which it has read)
  float* ob = reinterpret_cast<float*>(lds) + (wave * 16 + col) * OP + quad * 4;
#pragma unroll
  for (int j = 0; j < C::ND; ++j) *reinterpret_cast<f32x4_t*>(ob + j * 16) = x.o[j];
  __syncthreads();
  for (int i = tid; i < nq * (HD / 4); i += 512) {
#pragma clang fp contract(off)  // products rounded, then added, as where the join reads them
    const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
    float m[8], f[8], top = -INFINITY;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      m[c] = stat[0][r][c];
      top = fmaxf(top, m[c]);
    }
    float l[8];
    f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      f[c] = m[c] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[c] - top);
      if (nch == 1) f[c] = 1.f;
      l[c] = stat[1][r][c] * f[c];
      const f32x4_t z = *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(lds) + (c * 16 + r) * OP + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += z[e] * f[c];
    }
    // wave_sum's order of eight lanes
    const float lt = ((l[0] + l[4]) + (l[2] + l[6])) + ((l[1] + l[5]) + (l[3] + l[7]));
    const float inv = inverse(lt);
    *reinterpret_cast<u32x2_t*>(a.o + b * a.ldo + (int64_t)(head0 + r) * HD + d) =
        u32x2_t{pack_bf2(y[0] * inv, y[1] * inv), pack_bf2(y[2] * inv, y[3] * inv)};
    if (d == 0) store_lse(a, (int64_t)b * a.heads + head0 + r, top, lt, SCORES);
  }
}

// Joins the chunks of one query head.  HD / 4 threads add up every SUB-th chunk, 16 bytes each, and the SUB sums are
// added in order: the order goes by the row's own chunks alone.  (A part without a finite score is 0, or NaN and stays it.)
template <int HD, bool SCORES>
__global__ __launch_bounds__(256) void kv_join_kernel(Args a) {
  constexpr int TPR = HD / 4, SUB = 256 / TPR;
  __shared__ float f[kMaxChunks];
  __shared__ float red[2][4];
  __shared__ __align__(16) float acc[SUB][HD];
  const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nch = chunks_of(kv_length(a.t, b, false));
  if (nch == 1) return;
  const int64_t row = (int64_t)b * a.heads + head;
  const float* ml = a.ml + row * a.nchunk * 2;
  float mc[kMaxChunks / 256], lc[kMaxChunks / 256], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMaxChunks / 256; ++i) {
    const int c = i * 256 + tid;
    mc[i] = c < nch ? ml[2 * c] : -INFINITY;
    lc[i] = c < nch ? ml[2 * c + 1] : 0.f;
    top = fmaxf(top, mc[i]);
  }
  top = wave_max<64>(top);
  if (lane == 0) red[0][wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float lt = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxChunks / 256; ++i) {
    const float fc = mc[i] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mc[i] - top);
    f[i * 256 + tid] = fc;
    lt += lc[i] * fc;
  }
  lt = wave_sum<64>(lt);
  if (lane == 0) red[1][wave] = lt;
  __syncthreads();
  lt = red[1][0] + red[1][1] + red[1][2] + red[1][3];
  const int sub = tid / TPR, d = (tid % TPR) * 4;
  const float* part = a.part + row * a.nchunk * HD + d;
  f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int c = sub; c < nch; c += SUB) {
    const f32x4_t y = *reinterpret_cast<const f32x4_t*>(part + (int64_t)c * HD);
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] += y[r] * f[c];
  }
  *reinterpret_cast<f32x4_t*>(&acc[sub][d]) = x;
  __syncthreads();
  if (tid < TPR) {
    f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < SUB; ++i) y += *reinterpret_cast<const f32x4_t*>(&acc[i][d]);
    const float inv = inverse(lt);
    *reinterpret_cast<u32x2_t*>(a.o + b * a.ldo + (int64_t)head * HD + d) =
        u32x2_t{pack_bf2(y[0] * inv, y[1] * inv), pack_bf2(y[2] * inv, y[3] * inv)};
    if (tid == 0) store_lse(a, row, top, lt, SCORES);
  }
}

// Weights of a key head's slots: the probabilities summed over its query heads, in their order.  Four slots a thread.
__global__ __launch_bounds__(256) void kv_weights_kernel(Args a, int add) {
  const int b = blockIdx.z, kvh = blockIdx.y, i = (blockIdx.x * 256 + threadIdx.x) * 4;
  const int n = kv_length(a.t, b, false);
  if (i >= n) return;
  bool ok;
  const int p = kv_page(a.t, b, i, ok, false);
  if (!ok) return;
  const int64_t row0 = (int64_t)b * a.heads + (int64_t)kvh * a.group;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int g = 0; g < a.group; ++g) {
    const float e = a.lse2[row0 + g];
    const f32x4_t s = *reinterpret_cast<const f32x4_t*>(a.score + (row0 + g) * a.ld_score + i);
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[r] += e == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s[r] - e);
  }
  float* w = a.w.p + p * a.w.ps + kvh * a.w.hs + (i & ((1 << a.t.page_log2) - 1));
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (i + r < n) w[r] = add ? w[r] + sum[r] : sum[r];
}

// floats of the workspace's parts, each a multiple of 4
struct Space {
  int64_t part, ml, lse2, score, ld_score;
  int64_t floats() const { return part + ml + lse2 + score; }
};
Space space_of(int batch, int heads, int head_dim, int most, bool weights) {
  const int64_t rows = (int64_t)batch * heads, nc = chunks_bound(most);
  Space s{};
  if (nc > kShortChunks) {
    s.part = rows * nc * head_dim;
    s.ml = (rows * nc * 2 + 3) & ~(int64_t)3;
  }
  if (weights) {
    s.lse2 = (rows + 3) & ~(int64_t)3;
    s.ld_score = (most + 31) & ~31;
    s.score = rows * s.ld_score;
  }
  return s;
}

}  // namespace

DITK_EXPORT int64_t ditk_kv_attn_workspace(int batch, int heads, int head_dim, int most, int weights) {
  if (batch <= 0 || heads <= 0 || head_dim <= 0 || most < 0 || most >= (1 << 30)) return 0;
  return space_of(batch, heads, head_dim, most, weights != 0).floats() * 4;
}

DITK_EXPORT int ditk_kv_attn(const void* q, int64_t ldq, const void* k_cache, int64_t k_ps, int64_t k_hs,
                             const void* v_cache, int64_t v_ps, int64_t v_hs, float* weights, int64_t w_ps,
                             int64_t w_hs, int add, int pages, int page, const int32_t* table, int64_t ldt, int width,
                             const int32_t* lengths, int max_len, void* o, int64_t ldo, float* lse, void* workspace,
                             int64_t workspace_bytes, int batch, int heads, int kv_heads, int head_dim,
                             float softmax_scale, int32_t* status, hipStream_t stream) {
  const char* what = "ditk_kv_attn";
  if (int rc = kv_check_pages(what, table, lengths, status, batch, width, ldt, pages, page, kv_heads, head_dim)) return rc;
  if (int rc = kv_check_tensor(what, k_cache, k_ps, k_hs, page, head_dim)) return rc;
  if (int rc = kv_check_tensor(what, v_cache, v_ps, v_hs, page, head_dim)) return rc;
  DITK_REQUIRE(heads > 0 && heads <= 65535 && heads % kv_heads == 0, "%s: %d query heads for %d key heads", what, heads,
               kv_heads);
  DITK_REQUIRE(batch == 0 || (q && o), "%s: null tensor", what);
  DITK_REQUIRE(ldq % 8 == 0 && ldo % 8 == 0 && ((uintptr_t)q % 16) == 0 && ((uintptr_t)o % 16) == 0,
               "%s: rows must be 16-byte aligned", what);
  DITK_REQUIRE(max_len >= 0 && softmax_scale > 0.f, "%s: bad max_len or softmax_scale", what);
  if (batch == 0) return 0;
  const int most = width * page < max_len ? width * page : max_len;
  const Space sp = space_of(batch, heads, head_dim, most, weights != nullptr);
  DITK_REQUIRE(sp.floats() * 4 <= workspace_bytes && (sp.floats() == 0 || workspace) && ((uintptr_t)workspace % 16) == 0,
               "%s: the workspace needs %lld bytes", what, (long long)sp.floats() * 4);
  Args a{};
  a.t = KvPages{table, ldt, lengths, pages, __builtin_ctz((unsigned)page), most, status};
  a.k = KvTensor{(bf16_t*)k_cache, k_ps, k_hs};
  a.v = KvTensor{(bf16_t*)v_cache, v_ps, v_hs};
  a.w = KvWeights{weights, w_ps, w_hs};
  a.q = (const bf16_t*)q;
  a.ldq = ldq;
  a.o = (bf16_t*)o;
  a.ldo = ldo;
  a.lse = lse;
  a.part = (float*)workspace;
  a.ml = a.part + sp.part;
  a.lse2 = a.ml + sp.ml;
  a.score = a.lse2 + sp.lse2;
  a.ld_score = sp.ld_score;
  a.heads = heads;
  a.group = heads / kv_heads;
  a.nchunk = chunks_bound(most);
  a.scale2 = softmax_scale * 1.4426950408889634f;
  a.batch = batch;
  a.hgroups = kv_heads * ((a.group + 15) / 16);
  const int64_t units = (int64_t)batch * a.nchunk * a.hgroups, wgs = (units + 3) / 4;
  DITK_REQUIRE((int64_t)batch * heads < (1 << 22) && units < (1ll << 30), "%s: too many sequences, heads and chunks", what);
  const bool s = weights != nullptr;
  if (a.nchunk <= kShortChunks) {
    auto kern = head_dim == 128 ? (s ? kv_attn_short_kernel<128, true> : kv_attn_short_kernel<128, false>)
                                : (s ? kv_attn_short_kernel<64, true> : kv_attn_short_kernel<64, false>);
    kern<<<(unsigned)(batch * a.hgroups), 512, 0, stream>>>(a);
    if (int rc = ditk_check_launch(what)) return rc;
  } else {
    const int most_wgs = 3 * ditk_cu_count();
    auto kern = head_dim == 128 ? (s ? kv_attn_kernel<128, true> : kv_attn_kernel<128, false>)
                                : (s ? kv_attn_kernel<64, true> : kv_attn_kernel<64, false>);
    kern<<<(unsigned)(wgs < most_wgs ? wgs : most_wgs), 256, 0, stream>>>(a);
    if (int rc = ditk_check_launch(what)) return rc;
    auto join = head_dim == 128 ? (s ? kv_join_kernel<128, true> : kv_join_kernel<128, false>)
                                : (s ? kv_join_kernel<64, true> : kv_join_kernel<64, false>);
    join<<<dim3((unsigned)heads, (unsigned)batch), 256, 0, stream>>>(a);
    if (int rc = ditk_check_launch(what)) return rc;
  }
  if (s && most > 0) {
    kv_weights_kernel<<<dim3((unsigned)((most + 1023) / 1024), (unsigned)kv_heads, (unsigned)batch), 256, 0, stream>>>(a, add);
    if (int rc = ditk_check_launch(what)) return rc;
  }
  return 0;
}
