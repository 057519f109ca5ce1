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

constexpr int kMinChunk = 256, kMaxChunks = 128;

// slots of a chunk of a sequence of n: at most kMaxChunks of them, whole 32-slot tiles for four waves
__host__ __device__ inline int chunk_slots(int n) {
  const int64_t least = ((int64_t)n + kMaxChunks - 1) / kMaxChunks;
  const int c = (int)((least + 127) / 128 * 128);
  return c < kMinChunk ? kMinChunk : c;
}
__host__ __device__ inline int chunks_of(int n) { return n == 0 ? 1 : (n - 1) / chunk_slots(n) + 1; }

// the most chunks of any sequence up to `most` slots (fewer are possible past a change of the chunk's length)
int chunks_bound(int most) {
  const int c = most / kMinChunk + (most % kMinChunk != 0);
  return c < 1 ? 1 : c > kMaxChunks ? kMaxChunks : c;
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
  int heads, group, nchunk;
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

template <int HD, bool SCORES>
__global__ __launch_bounds__(256) void kv_attn_kernel(Args a) {
  constexpr int NC = HD / 32, ND = HD / 16, CH = HD / 8, RPL = 64 / CH;  // RPL: rows of V a load of the wave covers
  constexpr int OP = HD + 4;                                           // floats of a row of O in LDS
  __shared__ __align__(16) char lds[4 * 16 * OP * 4];
  __shared__ float stat[2][4][16];
  static_assert(sizeof(lds) >= 4 * 32 * HD * 2, "V tiles");
  const int b = blockIdx.z, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int groups = (a.group + 15) / 16, kvh = blockIdx.y / groups, g0 = (blockIdx.y % groups) * 16;
  const int chunk = blockIdx.x;
  const int n = kv_length(a.t, b, tid == 0 && chunk == 0 && blockIdx.y == 0);
  if (chunk >= chunks_of(n)) return;
  const int csl = chunk_slots(n), s0 = chunk * csl, s1 = min(n, s0 + csl), last = max(n - 1, 0);
  const int col = lane & 15, quad = lane >> 4;
  const int nq = min(a.group - g0, 16), head0 = kvh * a.group + g0;  // query heads of this workgroup
  const int pl = a.t.page_log2, low = (1 << pl) - 1;

  bf16x8_t q[NC];
  {
    const bf16_t* qr = a.q + b * a.ldq + (int64_t)(head0 + min(col, nq - 1)) * HD + quad * 8;
#pragma unroll
    for (int c = 0; c < NC; ++c) q[c] = *reinterpret_cast<const bf16x8_t*>(qr + c * 32);
  }
  f32x4_t o[ND];
#pragma unroll
  for (int j = 0; j < ND; ++j) o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  char* vt = lds + wave * (32 * HD * 2);

  for (int t0 = s0 + wave * 32; t0 < s1; t0 += 128) {
    // the tile's two halves of 16 slots lie in one page each; slots past the last read it
    const int e0 = min(t0, last), e1 = min(t0 + 16, last);
    bool ok0, ok1;
    const int p0 = kv_page(a.t, b, e0, ok0, true), p1 = kv_page(a.t, b, e1, ok1, true);
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

  // the four waves' parts, in order
  l = group_sumf(l);
  if (quad == 0) {
    stat[0][wave][col] = m;
    stat[1][wave][col] = l;
  }
  __syncthreads();
  const float top = fmaxf(fmaxf(stat[0][0][col], stat[0][1][col]), fmaxf(stat[0][2][col], stat[0][3][col]));
  // (a part without a finite score is 0, or NaN and stays it)
  const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);
  float* ob = reinterpret_cast<float*>(lds) + wave * 16 * OP;
#pragma unroll
  for (int j = 0; j < ND; ++j) {
    f32x4_t x = o[j];
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] *= f;
    *reinterpret_cast<f32x4_t*>(ob + col * OP + j * 16 + quad * 4) = x;
  }
  __syncthreads();
  const int nch = chunks_of(n);
  for (int i = tid; i < nq * (HD / 4); i += 256) {
    const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
    float mt = -INFINITY, lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, stat[0][w][r]);
    f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = stat[0][w][r];
      lt += stat[1][w][r] * (mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mw - mt));
      x += *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(lds) + (w * 16 + r) * OP + d);
    }
    const int64_t row = (int64_t)b * a.heads + head0 + r;
    if (nch == 1) {
      const float inv = lt > 0.f || lt != lt ? 1.f / lt : 0.f;
      *reinterpret_cast<u32x2_t*>(a.o + b * a.ldo + (int64_t)(head0 + r) * HD + d) =
          u32x2_t{pack_bf2(x[0] * inv, x[1] * inv), pack_bf2(x[2] * inv, x[3] * inv)};
      if (d == 0) {
        const float e = lt > 0.f || lt != lt ? mt + __builtin_amdgcn_logf(lt) : -INFINITY;
        if (a.lse != nullptr) a.lse[row] = e * 0.6931471805599453f;
        if (SCORES) a.lse2[row] = e;
      }
    } else {
      *reinterpret_cast<f32x4_t*>(a.part + (row * a.nchunk + chunk) * HD + d) = x;
      if (d == 0) {
        a.ml[(row * a.nchunk + chunk) * 2] = mt;
        a.ml[(row * a.nchunk + chunk) * 2 + 1] = lt;
      }
    }
  }
}

// Joins the chunks of one query head: a wave a row.
template <int HD, bool SCORES>
__global__ __launch_bounds__(64) void kv_join_kernel(Args a) {
  constexpr int V = HD / 64;
  const int head = blockIdx.x, b = blockIdx.y, lane = threadIdx.x;
  const int n = kv_length(a.t, b, false), nch = chunks_of(n);
  if (nch == 1) return;
  const int64_t row = (int64_t)b * a.heads + head;
  const float* ml = a.ml + row * a.nchunk * 2;
  float top = -INFINITY;
  for (int c = lane; c < nch; c += 64) top = fmaxf(top, ml[2 * c]);
  top = wave_max<64>(top);
  float x[V] = {}, lt = 0.f;
  const float* part = a.part + row * a.nchunk * HD + lane * V;
  for (int c = 0; c < nch; ++c) {
    const float mc = ml[2 * c], f = mc == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mc - top);
    lt = fmaf(ml[2 * c + 1], f, lt);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = fmaf(part[(int64_t)c * HD + i], f, x[i]);
  }
  const float inv = lt > 0.f || lt != lt ? 1.f / lt : 0.f;
  bf16_t* o = a.o + b * a.ldo + (int64_t)head * HD + lane * V;
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = f2bf(x[i] * inv);
  if (lane == 0) {
    const float e = lt > 0.f || lt != lt ? top + __builtin_amdgcn_logf(lt) : -INFINITY;
    if (a.lse != nullptr) a.lse[row] = e * 0.6931471805599453f;
    if (SCORES) a.lse2[row] = e;
  }
}

// weights of a key head's slots: the probabilities summed over its query heads, in their order
__global__ __launch_bounds__(256) void kv_weights_kernel(Args a, int add) {
  const int b = blockIdx.z, kvh = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
  const int n = kv_length(a.t, b, false);
  if (i >= n) return;
  bool ok;
  const int p = kv_page(a.t, b, i, ok, false);
  if (!ok) return;
  const int64_t row0 = (int64_t)b * a.heads + (int64_t)kvh * a.group;
  float sum = 0.f;
  for (int g = 0; g < a.group; ++g) {
    const float e = a.lse2[row0 + g];
    sum += e == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(a.score[(row0 + g) * a.ld_score + i] - e);
  }
  float* w = a.w.p + p * a.w.ps + kvh * a.w.hs + (i & ((1 << a.t.page_log2) - 1));
  *w = add ? *w + sum : sum;
}

// floats of the workspace's parts, each a multiple of 4
struct Space {
  int64_t part, ml, lse2, score, ld_score;
  int64_t floats() const { return part + ml + lse2 + score; }
};
Space space_of(int batch, int heads, int head_dim, int most, bool weights) {
  const int64_t rows = (int64_t)batch * heads, nc = chunks_bound(most);
  Space s{};
  if (nc > 1) {
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
  const int groups = (a.group + 15) / 16;
  DITK_REQUIRE(kv_heads * groups <= 65535, "%s: too many heads", what);
  const dim3 grid((unsigned)a.nchunk, (unsigned)(kv_heads * groups), (unsigned)batch);
  const bool s = weights != nullptr;
  auto kern = head_dim == 128 ? (s ? kv_attn_kernel<128, true> : kv_attn_kernel<128, false>)
                              : (s ? kv_attn_kernel<64, true> : kv_attn_kernel<64, false>);
  kern<<<grid, 256, 0, stream>>>(a);
  if (int rc = ditk_check_launch(what)) return rc;
  if (a.nchunk > 1) {
    auto join = head_dim == 128 ? (s ? kv_join_kernel<128, true> : kv_join_kernel<128, false>)
                                : (s ? kv_join_kernel<64, true> : kv_join_kernel<64, false>);
    join<<<dim3((unsigned)heads, (unsigned)batch), 64, 0, stream>>>(a);
    if (int rc = ditk_check_launch(what)) return rc;
  }
  if (s && most > 0) {
    kv_weights_kernel<<<dim3((unsigned)((most + 255) / 256), (unsigned)kv_heads, (unsigned)batch), 256, 0, stream>>>(a, add);
    if (int rc = ditk_check_launch(what)) return rc;
  }
  return 0;
}
