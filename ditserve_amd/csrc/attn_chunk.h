// Attention of up to 16 query rows over a range of keys by one wave: what kv_attn.hip (one new token over a paged cache)
// and causal_few.hip (few queries over many packed keys) share.
//
// A wave takes 32 keys at a time,
//   S^T = K Q^T         (A = 16 keys x 32 dims straight from memory, B = Q)
//   O^T += V^T P^T      (A = V^T by transposing LDS reads, B = P^T)
// with v_mfma_f32_16x16x32_bf16.  A lane's accumulators of the two score tiles are keys 4 quad .. + 3 of each half of 16,
// and these are the 8 keys it holds of the second product's B operand, whose A operand reads V's rows in that order: no
// shuffles between the two.
// P is taken as the sum of two bf16 numbers (16 bits of it at least), so that only the output is rounded to 8 bits: the
// matrix pipe is idle most of the time anyway.  Scores are in log2 units; m, l and O stay fp32.
#pragma once

#include "ditk_common.h"

// 32-byte piece of a V row in LDS that holds its piece 0 (piece j lies at j ^ that): the 8 rows that 32 lanes of a
// transposing read look at lie in different banks
template <int HD>
__device__ __forceinline__ int v_swizzle(int row) {
  return HD == 128 ? row & 7 : (row >> 1) & 3;
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

// Factors of two neighbouring parts, and the top and l of their sum.  (A part without a finite score is 0, or NaN and stays
// it.)  Parts are joined in such pairs first, wherever that is done, by these operations.
struct Pair {
  float m, l, fa, fb;
};
__device__ __forceinline__ Pair join_pair(float ma, float la, float mb, float lb) {
  Pair p;
  p.m = fmaxf(ma, mb);
  p.fa = ma == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ma - p.m);
  p.fb = mb == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mb - p.m);
  p.l = fmaf(lb, p.fb, la * p.fa);
  return p;
}
__device__ __forceinline__ f32x4_t join_pair(const Pair& p, f32x4_t a, f32x4_t b) {
  f32x4_t y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = fmaf(b[e], p.fb, a[e] * p.fa);
  return y;
}

// What a wave gathers of one range: lane (quad, col) holds dims 16 j + 4 quad .. + 3 of query row `col`'s sums of
// p v, and its m and its l.
//
// Src says where keys are: tile(t0, s0, s1) looks up the tile's two halves of 16 keys; then k(half) and v(half) point at
// the half's first row (for a half behind the last key or that is absent: at some row), k_stride() and v_stride() are the
// rows' distances, and ok(half) says whether the half is there.  All of it is uniform.  Src::once: whether the rows are
// read past the caches.
// The next tile's loads are issued as soon as this one's registers are free: the scores are made and the values in LDS.
// EACH: the queries may see different numbers of keys.
template <int HD, bool EACH>
struct Chunk {
  static constexpr int NC = HD / 32, ND = HD / 16, CH = HD / 8, RPL = 64 / CH;  // RPL: rows of V a load of the wave covers
  f32x4_t o[ND];
  float m, l;

  struct Tile {
    bf16x8_t k[2][NC];
    u32x4_t v[32 / RPL];
    int n0, n1;  // keys that are there of its halves
  };

  template <bool ONCE, class T>
  static __device__ __forceinline__ T fetch(const T* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    return *p;
  }

  template <class Src>
  __device__ __forceinline__ void load(Src& src, int t0, int s0, int s1, Tile& x) const {
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    src.tile(t0, s0, s1);
    if (t0 + 32 <= s1) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16_t *kr = src.k(h), *vr = src.v(h);
        const uint32_t ko = (uint32_t)col * src.k_stride() + quad * 8, vo = (uint32_t)(lane / CH) * src.v_stride() + (lane % CH) * 8;
#pragma unroll
        for (int c = 0; c < NC; ++c) x.k[h][c] = fetch<Src::once>(reinterpret_cast<const bf16x8_t*>(kr + ko + c * 32));
#pragma unroll
        for (int i = 0; i < 16 / RPL; ++i)
          x.v[h * (16 / RPL) + i] = fetch<Src::once>(reinterpret_cast<const u32x4_t*>(vr + (int64_t)i * RPL * src.v_stride() + vo));
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int most = max(min(s1 - t0 - 16 * h, 16) - 1, 0);  // (keys past the last read it)
        const bf16_t *kr = src.k(h), *vr = src.v(h);
        const uint32_t ko = (uint32_t)min(col, most) * src.k_stride() + quad * 8;
#pragma unroll
        for (int c = 0; c < NC; ++c) x.k[h][c] = fetch<Src::once>(reinterpret_cast<const bf16x8_t*>(kr + ko + c * 32));
#pragma unroll
        for (int i = 0; i < 16 / RPL; ++i)
          x.v[h * (16 / RPL) + i] = fetch<Src::once>(reinterpret_cast<const u32x4_t*>(
              vr + (uint32_t)min(i * RPL + lane / CH, most) * src.v_stride() + (lane % CH) * 8));
      }
    }
    x.n0 = src.ok(0) ? min(s1 - t0, 16) : 0;
    x.n1 = src.ok(1) ? min(s1 - t0 - 16, 16) : 0;
  }

  // One tile at t0, in x; then x is the next one.  lim: keys this lane's query sees (all_see: the fewest that any query
  // sees).  score: where the scores of this lane's query go, or null.
  template <class Src>
  __device__ __forceinline__ void step(Src& src, Tile& x, const bf16x8_t (&q)[NC], float scale2, int t0, int s0, int s1,
                                       int lim, int all_see, float* score, char* vt) {
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    // values of absent keys may be anything: they count as 0
    const int n0 = x.n0, n1 = x.n1;
    const bool here = n0 == 16 && n1 == 16, whole = here && t0 + 32 <= all_see;
    if (!here) {
#pragma unroll
      for (int i = 0; i < 32 / RPL; ++i) {
        const int row = i * RPL + lane / CH;
        if (i * RPL < 16 ? row >= n0 : row - 16 >= n1) x.v[i] = u32x4_t{0, 0, 0, 0};
      }
    }
    f32x4_t s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.k[i][c], q[c], s[i], 0, 0, 0);
    }
    {
      const int row = lane / CH, ch = lane % CH;
      char* w = vt + row * (HD * 2) + ((ch >> 1) ^ v_swizzle<HD>(row)) * 32 + (ch & 1) * 16;
      char* w4 = HD == 128 ? vt + row * (HD * 2) + ((ch >> 1) ^ v_swizzle<HD>(row + 4)) * 32 + (ch & 1) * 16 : w;
#pragma unroll
      for (int i = 0; i < 32 / RPL; ++i) *reinterpret_cast<u32x4_t*>((i & 1 ? w4 : w) + i * RPL * (HD * 2)) = x.v[i];
    }
    // a value that some queries do not see and that is not finite would reach them (0 times it is NaN) through the product
    const bool odd = EACH && !whole && !all_finite(x.v);
    if (!odd && t0 + 32 < s1) load(src, t0 + 32, s0, s1, x);
    float y[8], top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = s[e >> 2][e & 3] * scale2;
      const int row = quad * 4 + (e & 3);
      if (!whole && (row >= (e < 4 ? n0 : n1) || t0 + (e & 4) * 4 + row >= lim)) y[e] = -INFINITY;
      top = fmaxf(top, y[e]);
    }
    if (score != nullptr) {
      *reinterpret_cast<f32x4_t*>(score + t0 + quad * 4) = f32x4_t{y[0], y[1], y[2], y[3]};
      *reinterpret_cast<f32x4_t*>(score + t0 + 16 + quad * 4) = f32x4_t{y[4], y[5], y[6], y[7]};
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
    if (odd) {
      step_odd(y, base, t0, n0, n1, lim, vt);
      if (t0 + 32 < s1) load(src, t0 + 32, s0, s1, x);
      return;
    }
    bf16x8_t hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = __builtin_amdgcn_exp2f(y[e] - base);
      l += p;
      // hi cut off, so that lo is not negative, and lo not 0 unless p is: an infinite value stays one
      const float cut = __uint_as_float(__float_as_uint(p) & 0xffff0000u);
      hi[e] = __builtin_bit_cast(__bf16, (uint16_t)(__float_as_uint(p) >> 16));
      lo[e] = (__bf16)fmaxf(p - cut, fminf(p, 1.17549435e-38f));
    }
    // lane i of a quad reads 8 bytes of row 4 quad + i / 4 and gets 4 rows of column i.  (The address is made again for
    // every tile: kept for all j it would take 8 registers.)
    uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)vt;
    {
      const int row = quad * 4 + (col >> 2);
      at += row * (HD * 2) + v_swizzle<HD>(row) * 32 + (col & 3) * 8;
    }
    asm volatile("" : "+v"(at));
#pragma unroll
    for (int j = 0; j < ND; ++j) {
      s16x4 w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        w[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(uintptr_t)((at ^ (uint32_t)(j * 32)) + i * 16 * (HD * 2)));
      union { s16x4 h[2]; bf16x8_t f; } f;
      f.h[0] = w[0];
      f.h[1] = w[1];
      o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.f, hi, o[j], 0, 0, 0);
      o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.f, lo, o[j], 0, 0, 0);
    }
  }

  static __device__ __forceinline__ bool all_finite(const u32x4_t (&v)[32 / RPL]) {
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 32 / RPL; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= ((v[i][e] & 0x7f80u) == 0x7f80u) | ((v[i][e] & 0x7f800000u) == 0x7f800000u);
    return !__any(bad != 0);
  }

  // P and O of a tile with values that are not finite, each of them only where it is seen: products one by one
  __device__ __forceinline__ void step_odd(const float (&y)[8], float base, int t0, int n0, int n1, int lim, const char* vt) {
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float mine = __builtin_amdgcn_exp2f(y[e] - base);
      l += mine;
#pragma unroll 1
      for (int g = 0; g < 4; ++g) {
        const int in = 4 * g + (e & 3), row = (e & 4) * 4 + in;
        const float p = __shfl(mine, g * 16 + col, 64);
        if (in >= (e < 4 ? n0 : n1) || t0 + row >= lim) continue;
#pragma unroll
        for (int j = 0; j < ND; ++j) {
          const u32x2_t w = *reinterpret_cast<const u32x2_t*>(vt + row * (HD * 2) + (j ^ v_swizzle<HD>(row)) * 32 + quad * 8);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            o[j][2 * r] = fmaf(p, __uint_as_float(w[r] << 16), o[j][2 * r]);
            o[j][2 * r + 1] = fmaf(p, __uint_as_float(w[r] & 0xffff0000u), o[j][2 * r + 1]);
          }
        }
      }
    }
  }

  // keys [s0, s1); qr: this lane's query row, + 8 quad; vt: 32 HD bf16 of LDS, aligned to 256 bytes
  template <class Src>
  __device__ __forceinline__ void run(Src& src, const bf16_t* qr, float scale2, int s0, int s1, int lim, int all_see,
                                      float* score, char* vt) {
    run_two(src, qr, scale2, s0, s1, s1, lim, all_see, score, vt);
  }

  // keys [s0, s1) and [s1, s2) (whole tiles up to s1), each by itself, then joined; the second's first tile is asked for
  // with the first's last
  template <class Src>
  __device__ __forceinline__ void run_two(Src& src, const bf16_t* qr, float scale2, int s0, int s1, int s2, int lim,
                                          int all_see, float* score, char* vt) {
    Tile x;
    if (s0 < s2) load(src, s0, s0, s2, x);
    bf16x8_t q[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) q[i] = *reinterpret_cast<const bf16x8_t*>(qr + i * 32);
    clear();
    for (int t0 = s0; t0 < s1; t0 += 32) step(src, x, q, scale2, t0, s0, s2, lim, all_see, score, vt);
    l = group_sumf(l);
    if (s1 >= s2) return;
    const Chunk y = *this;
    clear();
    for (int t0 = s1; t0 < s2; t0 += 32) step(src, x, q, scale2, t0, s0, s2, lim, all_see, score, vt);
    l = group_sumf(l);
    const Pair p = join_pair(y.m, y.l, m, l);
    m = p.m;
    l = p.l;
#pragma unroll
    for (int j = 0; j < ND; ++j) o[j] = join_pair(p, y.o[j], o[j]);
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < ND; ++j) o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }
};

// Packed rows
struct RowsSrc {
  static constexpr bool once = false;
  const bf16_t *kb, *vb;  // first key's row of the head
  int ldk, ldv, last;
  int t0 = 0, t1 = 0;
  __device__ __forceinline__ void tile(int t, int, int) {
    t0 = t;
    t1 = t + 16 <= last ? t + 16 : t;
  }
  __device__ __forceinline__ bool ok(int) const { return true; }
  __device__ __forceinline__ const bf16_t* k(int half) const { return kb + (int64_t)(half ? t1 : t0) * ldk; }
  __device__ __forceinline__ const bf16_t* v(int half) const { return vb + (int64_t)(half ? t1 : t0) * ldv; }
  __device__ __forceinline__ int k_stride() const { return ldk; }
  __device__ __forceinline__ int v_stride() const { return ldv; }
};

// 1 / l, 0 for a row without keys
__device__ __forceinline__ float inverse(float l) { return l > 0.f || l != l ? 1.f / l : 0.f; }
// log2 of a row's sum, -inf without keys
__device__ __forceinline__ float row_lse2(float m, float l) {
  return l > 0.f || l != l ? m + __builtin_amdgcn_logf(l) : -INFINITY;
}

// Joins the parts of eight waves, a wave's 16 rows of HD + 4 floats in `lds` and its m and l in stat[0..1][row][wave]:
// the sum of four dims from d on of row r, its top and its l.  Products are rounded, then added in order.
template <int HD>
__device__ __forceinline__ f32x4_t join8(const float* lds, const float (*stat)[16][8], int r, int d, float& top, float& lt) {
#pragma clang fp contract(off)
  Pair p[4];
  top = -INFINITY;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    p[c] = join_pair(stat[0][r][2 * c], stat[1][r][2 * c], stat[0][r][2 * c + 1], stat[1][r][2 * c + 1]);
    top = fmaxf(top, p[c].m);
  }
  f32x4_t y = {0.f, 0.f, 0.f, 0.f};
  float l[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float f = p[c].m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(p[c].m - top);
    l[c] = p[c].l * f;
    const float* at = lds + (c * 2 * 16 + r) * (HD + 4) + d;
    const f32x4_t z = join_pair(p[c], *reinterpret_cast<const f32x4_t*>(at), *reinterpret_cast<const f32x4_t*>(at + 16 * (HD + 4)));
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += z[e] * f;
  }
  lt = (l[0] + l[2]) + (l[1] + l[3]);  // wave_sum's order of four lanes
  return y;
}
