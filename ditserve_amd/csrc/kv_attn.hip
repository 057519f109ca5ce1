// Attention of one new token of each sequence over its paged keys and values (kv_common.h), split over the
// sequence's slots and joined.
//
// The query heads of a key head, 16 at a time, are the columns of a wave's products (attn_chunk.h).  A chunk's length
// goes by the sequence's own length alone, so a sequence's result does not depend on what it is batched with.
//
// Up to 16 query heads a key head, each slot is read once, and gives 2 operations a byte and query head: memory bounds it.
// 32 heads over 8 of 128, this kernel: 16 sequences of 32768 slots 360 us (5.9 TB/s), 64 of 2000 90 (5.8), one of 131072 (40
// heads) 89 (6.0); where few waves have a unit each, the latency of a chunk's tiles: one of 8192 14 us.  Of more than 16
// heads, every 16 read the slots again, side by side in the list: 16 of 32768 with one key head 51 us for 16 query
// heads (5.2 TB/s), 84 for 32 (3.2 of what there is).
#include "attn_chunk.h"
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
  int* twos;      // whether parts are of two chunks each
  float* score;   // [batch * heads][ld_score], or null
  int64_t ld_score;
  int heads, group, nchunk, batch, hgroups;  // hgroups: (key head, 16 of its query heads) pairs
  float scale2;   // softmax scale times log2 e
};

// Pages of a sequence, 64 of them (1024 slots at least) in a wave's lanes.  ONCE: a long cache's rows go past the caches,
// also where more than 16 query heads read them more than once (16 x 32768 slots 410 -> 397 us, 1 x 131072 105 -> 94, 64 x 2000 112 -> 108; not where scores are written
// beside: 469 -> 475).
template <int HD, bool ONCE>
struct PagedSrc {
  static constexpr bool once = ONCE;
  const Args& a;
  int b, kvh, last;
  int page = 0, first = 0;
  int64_t k0, k1, v0, v1;  // offsets of the halves' first slots
  bool ok0, ok1;
  __device__ __forceinline__ void tile(int t0, int s0, int s1) {
    const int pl = a.t.page_log2, low = (1 << pl) - 1;
    if (((t0 - s0) & 1023) == 0) {
      first = t0 >> pl;
      const int lane = threadIdx.x & 63, i = min(first + lane, last >> pl), p = a.t.table[b * a.t.ldt + i];
      page = (unsigned)p < (unsigned)a.t.pages ? p : -1;
      if (page < 0 && (first + lane) << pl < s1) *a.t.status = 1;
    }
    // a half of 16 slots lies in one page; one behind the last slot stands where the first half does
    const int t1 = t0 + 16 <= last ? t0 + 16 : t0;
    const int g0 = __builtin_amdgcn_readlane(page, (t0 >> pl) - first), g1 = __builtin_amdgcn_readlane(page, (t1 >> pl) - first);
    ok0 = g0 >= 0;
    ok1 = g1 >= 0;
    k0 = max(g0, 0) * a.k.ps + (t0 & low) * HD;
    k1 = max(g1, 0) * a.k.ps + (t1 & low) * HD;
    v0 = max(g0, 0) * a.v.ps + (t0 & low) * HD;
    v1 = max(g1, 0) * a.v.ps + (t1 & low) * HD;
  }
  __device__ __forceinline__ bool ok(int half) const { return half ? ok1 : ok0; }
  __device__ __forceinline__ const bf16_t* k(int half) const { return a.k.p + kvh * a.k.hs + (half ? k1 : k0); }
  __device__ __forceinline__ const bf16_t* v(int half) const { return a.v.p + kvh * a.v.hs + (half ? v1 : v0); }
  __device__ __forceinline__ int k_stride() const { return HD; }
  __device__ __forceinline__ int v_stride() const { return HD; }
};

__device__ __forceinline__ void store_lse(const Args& a, int64_t row, float e, bool scores) {
  if (a.lse != nullptr) a.lse[row] = e * 0.6931471805599453f;
  if (scores) a.lse2[row] = e;
}

// A wave takes one chunk of one (sequence, key head, 16 query heads) after another; units go round the waves in
// order: a sequence's chunks, and for each its heads, which lie side by side in a page.
//
// With two chunks or more a wave, units are two neighbouring chunks and leave one part, joined as the join kernel joins
// the parts of two (the bits are the same): half as much is written and read again (4 KB for 128 slots of 8 query heads,
// 64 KB of keys and values).  32 heads over 8: 64 sequences of 2000 slots 107 -> 96 us, 256 437 -> 402, 16 of 32768 398
// -> 363; with fewer units waves would stand idle (64 ragged ones 51 and 58), and where scores are written nothing is won
// (16 of 32768 470 and 475).
template <int HD, bool SCORES>
__global__ __launch_bounds__(256, 2) void kv_attn_kernel(Args a) {
  using C = Chunk<HD, false>;
  __shared__ __align__(256) char lds[4 * 32 * HD * 2];
  __shared__ int sums[2][4], ends[256], lens[256];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int col = lane & 15, quad = lane >> 4;

  // chunks up to and with thread t's sequences, [t per, t per + per)
  const int per = (a.batch + 255) / 256;
  int incl = 0, pairs = 0;
  for (int i = 0; i < per; ++i)
    if (tid * per + i < a.batch) {
      const int n = kv_length(a.t, tid * per + i, blockIdx.x == 0), nch = chunks_of(n);
      if (i == 0) lens[tid] = n;
      incl += nch;
      pairs += (nch + 1) >> 1;
    }
  incl = wave_scan(incl);
  pairs = wave_scan(pairs);
  if (lane == 63) sums[0][wave] = incl, sums[1][wave] = pairs;
  __syncthreads();
  const int chunks = (sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]);
  const int two = !SCORES && (int64_t)chunks * a.hgroups >= (int64_t)gridDim.x * 4 * 2;  // 1: units of two chunks
  if (two) incl = pairs;
  for (int w = 0; w < wave; ++w) incl += sums[two][w];
  ends[tid] = incl;
  if (blockIdx.x == 0 && tid == 0) *a.twos = two;
  __syncthreads();
  int end[4];  // (every wave keeps all of them)
#pragma unroll
  for (int i = 0; i < 4; ++i) end[i] = ends[i * 64 + lane];
  const int units = __builtin_amdgcn_readlane(end[3], 63) * a.hgroups, groups = (a.group + 15) / 16;

  for (int u = blockIdx.x * 4 + wave; u < units; u += gridDim.x * 4) {
    const int c = u / a.hgroups, hg = u - c * a.hgroups;
    // the thread whose sequences hold unit c, then the sequence
    int th = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) th += __popcll(__ballot(end[i] <= c));
    int b = th * per, part = c - (th ? ends[th - 1] : 0), n = lens[th], nch = chunks_of(n);
    while (part >= (nch + two) >> two && b + 1 < a.batch) {
      part -= (nch + two) >> two;
      n = kv_length(a.t, ++b, false);
      nch = chunks_of(n);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    n = __builtin_amdgcn_readfirstlane(n);
    part = __builtin_amdgcn_readfirstlane(min(part, (a.nchunk - 1) >> two));
    const int kvh = hg / groups, g0 = (hg - kvh * groups) * 16;
    const int csl = chunk_slots(n), s0 = (part << two) * csl, s1 = min(n, s0 + csl), s2 = two ? min(n, s1 + csl) : s1;
    const int nq = min(a.group - g0, 16), head0 = kvh * a.group + g0;  // query heads of this unit
    const int64_t row = (int64_t)b * a.heads + head0 + min(col, nq - 1);
    C x;
    PagedSrc<HD, !SCORES> src{a, b, kvh, max(n - 1, 0)};
    const bf16_t* qr = a.q + b * a.ldq + (int64_t)(head0 + min(col, nq - 1)) * HD + quad * 8;
    if constexpr (SCORES) x.run(src, qr, a.scale2, s0, s1, n, n, col < nq ? a.score + row * a.ld_score : nullptr, lds + wave * (32 * HD * 2));
    else x.run_two(src, qr, a.scale2, s0, s1, s2, n, n, nullptr, lds + wave * (32 * HD * 2));
    if (col < nq) {
      if (nch == 1) {
        const float inv = inverse(x.l);
        bf16_t* ob = a.o + b * a.ldo + (int64_t)(head0 + col) * HD + quad * 4;
#pragma unroll
        for (int j = 0; j < C::ND; ++j)
          *reinterpret_cast<u32x2_t*>(ob + j * 16) = u32x2_t{pack_bf2(x.o[j][0] * inv, x.o[j][1] * inv),
                                                            pack_bf2(x.o[j][2] * inv, x.o[j][3] * inv)};
        if (quad == 0) store_lse(a, row, row_lse2(x.m, x.l), SCORES);
      } else {
        float* pb = a.part + (row * a.nchunk + part) * HD + quad * 4;
#pragma unroll
        for (int j = 0; j < C::ND; ++j) *reinterpret_cast<f32x4_t*>(pb + j * 16) = x.o[j];
        if (quad == 0) *reinterpret_cast<u32x2_t*>(a.ml + (row * a.nchunk + part) * 2) =
            u32x2_t{__float_as_uint(x.m), __float_as_uint(x.l)};
      }
    }
  }
}

// Sequences of up to 8 chunks in one launch: eight waves take a chunk each of a (sequence, key head, 16 query heads) and
// join them through LDS, by the join kernel's operations in its order.  One sequence of 500 slots, 12 heads over 2: 9 us,
// the latency of lengths, pages, two tiles and the join.
template <int HD, bool SCORES>
__global__ __launch_bounds__(512) void kv_attn_short_kernel(Args a) {
  using C = Chunk<HD, false>;
  constexpr int OP = HD + 4;  // floats of a row of LDS
  __shared__ __align__(256) char lds[8 * 16 * OP * 4];
  __shared__ float stat[2][16][8];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int col = lane & 15, quad = lane >> 4, groups = (a.group + 15) / 16;
  const int b = blockIdx.x / a.hgroups, hg = blockIdx.x - b * a.hgroups;
  const int kvh = hg / groups, g0 = (hg - kvh * groups) * 16;
  const int n = kv_length(a.t, b, hg == 0 && tid == 0), csl = chunk_slots(n), nch = chunks_of(n);
  const int s0 = min(wave * csl, n), s1 = min(n, s0 + csl);
  const int nq = min(a.group - g0, 16), head0 = kvh * a.group + g0;
  const int64_t row = (int64_t)b * a.heads + head0 + min(col, nq - 1);
  C x;
  PagedSrc<HD, false> src{a, b, kvh, max(n - 1, 0)};
  x.run(src, a.q + b * a.ldq + (int64_t)(head0 + min(col, nq - 1)) * HD + quad * 8, a.scale2, s0, s1,
                       n, n, SCORES && col < nq ? a.score + row * a.ld_score : nullptr,
                       lds + wave * (16 * OP * 4));
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
    const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
    float top, lt;
    const f32x4_t y = join8<HD>(reinterpret_cast<const float*>(lds), stat, r, d, top, lt);
    const float inv = inverse(lt);
    *reinterpret_cast<u32x2_t*>(a.o + b * a.ldo + (int64_t)(head0 + r) * HD + d) =
        u32x2_t{pack_bf2(y[0] * inv, y[1] * inv), pack_bf2(y[2] * inv, y[3] * inv)};
    if (d == 0) store_lse(a, (int64_t)b * a.heads + head0 + r, row_lse2(top, lt), SCORES);
  }
}

// Joins the parts of one query head: those of two chunks as units of two leave them, or two at a time.  HD / 4 threads add
// up every SUB-th, 16 bytes each, and the SUB sums are added in order: the order goes by the row's own chunks alone.
template <int HD, bool SCORES>
__global__ __launch_bounds__(256) void kv_join_kernel(Args a) {
  constexpr int TPR = HD / 4, SUB = 256 / TPR;
  static_assert(kMaxChunks == 2 * 256, "a pair of chunks a thread");
  __shared__ float f[256], fa[256], fb[256];
  __shared__ float red[2][4];
  __shared__ __align__(16) float acc[SUB][HD];
  const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nch = chunks_of(kv_length(a.t, b, false));
  if (nch == 1) return;
  const int64_t row = (int64_t)b * a.heads + head;
  const float* ml = a.ml + row * a.nchunk * 2;
  const int np = (nch + 1) >> 1, odd = nch & 1;  // pairs; whether the last is one chunk
  // (both places are read before the word that says which counts is there)
  const int last = nch - 1, at0 = min(tid, last), at1 = min(2 * tid, last), at2 = min(2 * tid + 1, last);
  const u32x2_t e0 = *reinterpret_cast<const u32x2_t*>(ml + 2 * at0), e1 = *reinterpret_cast<const u32x2_t*>(ml + 2 * at1),
                e2 = *reinterpret_cast<const u32x2_t*>(ml + 2 * at2);
  const bool two = *a.twos != 0;
  Pair p{-INFINITY, 0.f, 1.f, 0.f};
  if (tid < np) {
    p.m = __uint_as_float(two ? e0[0] : e1[0]);
    p.l = __uint_as_float(two ? e0[1] : e1[1]);
    if (!two && !(odd && tid == np - 1)) p = join_pair(p.m, p.l, __uint_as_float(e2[0]), __uint_as_float(e2[1]));
  }
  fa[tid] = p.fa;
  fb[tid] = p.fb;
  float top = wave_max<64>(p.m);
  if (lane == 0) red[0][wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float fc = p.m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(p.m - top);
  f[tid] = fc;
  float lt = wave_sum<64>(fmaf(p.l, fc, 0.f));  // (a rounded product)
  if (lane == 0) red[1][wave] = lt;
  __syncthreads();
  lt = red[1][0] + red[1][1] + red[1][2] + red[1][3];
  const int sub = tid / TPR, d = (tid % TPR) * 4;
  const float* part = a.part + row * a.nchunk * HD + d;
  f32x4_t x = {0.f, 0.f, 0.f, 0.f};
  if (two) {
#pragma unroll 8
    for (int c = sub; c < np; c += SUB) {
      const f32x4_t y = *reinterpret_cast<const f32x4_t*>(part + (int64_t)c * HD);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = fmaf(y[r], f[c], x[r]);
    }
  } else {
#pragma unroll 4
    for (int c = sub; c < nch >> 1; c += SUB) {
      const f32x4_t ya = *reinterpret_cast<const f32x4_t*>(part + (int64_t)(2 * c) * HD);
      const f32x4_t yb = *reinterpret_cast<const f32x4_t*>(part + (int64_t)(2 * c + 1) * HD);
      const f32x4_t y = join_pair(Pair{0.f, 0.f, fa[c], fb[c]}, ya, yb);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = fmaf(y[r], f[c], x[r]);
    }
    if (odd && (np - 1) % SUB == sub) {
      const f32x4_t y = *reinterpret_cast<const f32x4_t*>(part + (int64_t)last * HD);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = fmaf(y[r], f[np - 1], x[r]);
    }
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
    if (tid == 0) store_lse(a, row, row_lse2(top, lt), SCORES);
  }
}

// Weights of a key head's slots: the probabilities summed over its query heads, in their order.  Four slots a thread.
// Memory: 80 MB of scores and weights of 16 x 32768 slots 17 us (4.7 TB/s).
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

// floats of the workspace's parts, each a multiple of 64 (scores are written in whole lines: 16 bytes off one, 16 x 32768
// slots took 457 us for 443)
struct Space {
  int64_t part, ml, twos, lse2, score, ld_score;
  int64_t floats() const { return part + ml + twos + lse2 + score; }
};
Space space_of(int batch, int heads, int head_dim, int most, bool weights) {
  const int64_t rows = (int64_t)batch * heads, nc = chunks_bound(most);
  Space s{};
  if (nc > kShortChunks) {
    s.part = rows * nc * head_dim;
    s.ml = (rows * nc * 2 + 63) & ~(int64_t)63;
    s.twos = 64;
  }
  if (weights) {
    s.lse2 = (rows + 63) & ~(int64_t)63;
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
  if (int rc = kv_check_tensor(what, k_cache, k_ps, k_hs)) return rc;
  if (int rc = kv_check_tensor(what, v_cache, v_ps, v_hs)) return rc;
  if (int rc = kv_check_weights(what, weights, w_ps, w_hs)) return rc;
  DITK_REQUIRE(heads > 0 && heads <= 65535 && heads % kv_heads == 0, "%s: %d query heads for %d key heads", what, heads,
               kv_heads);
  DITK_REQUIRE(batch == 0 || (q && o), "%s: null tensor", what);
  DITK_REQUIRE(ldq % 8 == 0 && ldo % 8 == 0 && ((uintptr_t)q % 16) == 0 && ((uintptr_t)o % 16) == 0,
               "%s: rows must be 16-byte aligned", what);
  const int64_t row = (int64_t)heads * head_dim;
  DITK_REQUIRE(batch <= 1 || (ldq >= row && ldo >= row), "%s: rows of q or o overlap", what);
  DITK_REQUIRE(max_len >= 0, "%s: bad max_len %d", what, max_len);
  DITK_REQUIRE(softmax_scale >= 1e-30f && softmax_scale <= 1e30f, "%s: softmax_scale must be in 1e-30..1e30", what);
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
  a.twos = (int*)(a.ml + sp.ml);
  a.lse2 = a.ml + sp.ml + sp.twos;
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
    const int most_wgs = 2 * ditk_cu_count();  // (3 a CU, with fewer registers, spill: 1 x 8192 slots 20 us for 18)
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
