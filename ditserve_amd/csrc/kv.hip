// Writing to and evicting from paged key-value caches (kv_common.h).  Both move bytes.
#include "kv_common.h"

int kv_check_pages(const char* what, const void* table, const void* lengths, const void* status, int batch, int width,
                   int64_t ldt, int pages, int page, int kv_heads, int head_dim) {
  DITK_REQUIRE(batch >= 0 && batch <= 65535, "%s: %d sequences (65535 at most)", what, batch);
  DITK_REQUIRE(kv_heads > 0 && kv_heads <= 65535, "%s: bad key head count %d", what, kv_heads);
  DITK_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128, got %d", what, head_dim);
  DITK_REQUIRE(page == 16 || page == 32 || page == 64 || page == 128 || page == 256,
               "%s: a page holds 16, 32, 64, 128 or 256 slots, got %d", what, page);
  DITK_REQUIRE(pages > 0, "%s: the cache has no pages", what);
  DITK_REQUIRE(status != nullptr && (batch == 0 || (table && lengths)), "%s: null table", what);
  DITK_REQUIRE(width >= 0 && ldt >= width && (int64_t)width * page < (1ll << 30), "%s: bad page table", what);
  return 0;
}

int kv_check_tensor(const char* what, const void* p, int64_t ps, int64_t hs, int page, int head_dim) {
  DITK_REQUIRE(p != nullptr, "%s: null cache", what);
  DITK_REQUIRE(((uintptr_t)p % 16) == 0 && ps % 8 == 0 && hs % 8 == 0 && ps >= 0 && hs >= 0,
               "%s: the cache's heads must be 16-byte aligned", what);
  return 0;
}

namespace {

constexpr int kCuLds = 1024;

// Rows of new keys and values into the slots behind each sequence's last: row i of segment b goes to slot lengths[b] + i.
// A thread moves 16 bytes; `per` of them make a row of K or V, and the grid's second dimension is K or V.
template <int LOG_CH>
__global__ __launch_bounds__(256) void kv_append_kernel(KvPages t, KvTensor kc, KvTensor vc, KvWeights w,
                                                        const bf16_t* __restrict__ k, int64_t ldk,
                                                        const bf16_t* __restrict__ v, int64_t ldv,
                                                        int32_t* __restrict__ new_lengths,
                                                        const int32_t* __restrict__ cu, int nseg, int T, int per) {
  __shared__ int32_t cus[kCuLds + 1];
  const bool in_lds = cu != nullptr && nseg <= kCuLds;
  if (in_lds) {
    for (int i = threadIdx.x; i <= nseg; i += 256) cus[i] = cu[i];
    __syncthreads();
  }
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int b = threadIdx.x; b < nseg; b += 256) {
      const int n = kv_length(t, b, true), add = cu != nullptr ? cu[b + 1] - cu[b] : 1;
      if (n + (int64_t)add > t.most) *t.status = 1;
      new_lengths[b] = (int)min((int64_t)t.most, n + (int64_t)add);
    }
  const bool is_v = blockIdx.y != 0;
  const int64_t total = (int64_t)T * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int row = (int)(i / per), c = (int)(i - (int64_t)row * per);
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>((is_v ? v + row * ldv : k + row * ldk) + c * 8);
    int b = row, at = 0;
    if (cu != nullptr) {
      b = in_lds ? find_segment(cus, nseg, row) : find_segment(cu, nseg, row);
      at = row - (in_lds ? cus[b] : cu[b]);
    }
    const int64_t slot = (int64_t)kv_length(t, b, false) + at;
    if (slot >= t.most) continue;
    bool ok;
    const int p = kv_page(t, b, (int)slot, ok, true);
    if (!ok) continue;
    const int h = c >> LOG_CH, j = (int)slot & ((1 << t.page_log2) - 1);
    const KvTensor& to = is_v ? vc : kc;
    *reinterpret_cast<u32x4_t*>(to.p + p * to.ps + h * to.hs + (((int64_t)j << LOG_CH) + (c & ((1 << LOG_CH) - 1))) * 8) = x;
    if (w.p != nullptr && !is_v && (c & ((1 << LOG_CH) - 1)) == 0) w.p[p * w.ps + h * w.hs + j] = 0.f;
  }
}

// fp32 -> uint32 whose order is the floats': -0 is 0, and a NaN is -inf
__device__ __forceinline__ uint32_t order_of(float f) {
  uint32_t u = __float_as_uint(f);
  if (f != f) u = 0xff800000u;
  if (u == 0x80000000u) u = 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float weight_at(const KvPages& t, const KvWeights& w, int b, int h, int i) {
  bool ok;
  const int p = kv_page(t, b, i, ok, true);
  return ok ? w.p[p * w.ps + h * w.hs + (i & ((1 << t.page_log2) - 1))] : -INFINITY;
}

// The slots that stay, ascending: one workgroup per (key head, sequence).  The threshold is the (m - recent)-th largest
// weight of the others, found 8 bits at a time; of the slots that hold just it, the lowest stay.
__global__ __launch_bounds__(1024) void kv_select_kernel(KvPages t, KvWeights w, int keep, int recent,
                                                         int32_t* __restrict__ slots, int32_t* __restrict__ new_lengths) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t pick[2];      // the digit, and how many of it are wanted
  __shared__ int above[16], ties[16];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int n = kv_length(t, b, tid == 0), m = min(n, keep), r = min(recent, m), old = n - r;
  int32_t* out = slots + ((int64_t)b * gridDim.x + h) * keep;
  if (h == 0 && tid == 0) new_lengths[b] = m;
  uint32_t want = (uint32_t)(m - r), top = 0, mask = 0;
  if (n > m && want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < old; i += 1024) {
        const uint32_t u = order_of(weight_at(t, w, b, h, i));
        if ((u & mask) == top) atomicAdd(&hist[(u >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t left = want;
        int d = 255;
        while (d > 0 && hist[d] < left) left -= hist[d--];
        pick[0] = (uint32_t)d;
        pick[1] = left;
      }
      __syncthreads();
      top |= pick[0] << shift;
      mask |= 0xffu << shift;
      want = pick[1];
      __syncthreads();
    }
  }
  // now: slots above `top` stay, and the first `want` that equal it.  Wave w takes a part of the slots.
  const bool all = n <= m, none = !all && m == r;
  const int part = ((old + 15) / 16 + 63) & ~63, i0 = min(wave * part, old), i1 = min(i0 + part, old);
  int na = 0, nt = 0;
  for (int i = i0 + lane; i < i1; i += 64) {
    const uint32_t u = all || none ? 0u : order_of(weight_at(t, w, b, h, i));
    na += all || (!none && u > top);
    nt += !all && !none && u == top;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    na += __shfl_xor(na, off, 64);
    nt += __shfl_xor(nt, off, 64);
  }
  if (lane == 0) above[wave] = na, ties[wave] = nt;
  __syncthreads();
  int at = 0, tie = 0;  // slots that stay, and equal ones, before this wave's part
  for (int i = 0; i < wave; ++i) {
    at += above[i];
    tie += ties[i];
  }
  at += min(tie, (int)want) * (all || none ? 0 : 1);
  for (int i = i0; i < i1; i += 64) {
    const bool in = i + lane < i1;
    const uint32_t u = all || none || !in ? 0u : order_of(weight_at(t, w, b, h, i + lane));
    const bool eq = in && !all && !none && u == top;
    const uint64_t eqs = __ballot(eq), before = (1ull << lane) - 1;
    const bool stay = in && (all || (!none && u > top) || (eq && tie + __popcll(eqs & before) < (int)want));
    const uint64_t stays = __ballot(stay);
    if (stay) out[at + __popcll(stays & before)] = i + lane;
    at += __popcll(stays);
    tie += __popcll(eqs);
  }
  for (int i = tid; i < r; i += 1024) out[m - r + i] = old + i;
}

// Copies the slots that stay into the pages of `to`: 16 slots of a (key head, sequence) a workgroup, 16 bytes a thread.
template <int LOG_CH>
__global__ __launch_bounds__(256) void kv_move_kernel(KvPages t, KvPages to, KvTensor kc, KvTensor vc, KvWeights w,
                                                      int keep, const int32_t* __restrict__ slots) {
  constexpr int kSlots = 256 >> LOG_CH;
  const int h = blockIdx.y, b = blockIdx.z;
  const int m = min(kv_length(t, b, false), keep);
  const int j = blockIdx.x * kSlots + (threadIdx.x >> LOG_CH), c = threadIdx.x & ((1 << LOG_CH) - 1);
  if (j >= m) return;
  const int i = slots[((int64_t)b * gridDim.y + h) * keep + j], low = (1 << t.page_log2) - 1;
  bool ok, ok_to;
  const int p = kv_page(t, b, i, ok, false), q = kv_page(to, b, j, ok_to, true);
  if (!ok_to) return;
  const int64_t src = (((int64_t)(i & low) << LOG_CH) + c) * 8, dst = (((int64_t)(j & low) << LOG_CH) + c) * 8;
  u32x4_t k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
  if (ok) {
    k = *reinterpret_cast<const u32x4_t*>(kc.p + p * kc.ps + h * kc.hs + src);
    v = *reinterpret_cast<const u32x4_t*>(vc.p + p * vc.ps + h * vc.hs + src);
  }
  *reinterpret_cast<u32x4_t*>(kc.p + q * kc.ps + h * kc.hs + dst) = k;
  *reinterpret_cast<u32x4_t*>(vc.p + q * vc.ps + h * vc.hs + dst) = v;
  if (c == 0) w.p[q * w.ps + h * w.hs + (j & low)] = ok ? w.p[p * w.ps + h * w.hs + (i & low)] : 0.f;
}

int log2_of(int page) { return __builtin_ctz((unsigned)page); }

}  // namespace

DITK_EXPORT int ditk_kv_append(const void* k, int64_t ldk, const void* v, int64_t ldv, void* k_cache, int64_t k_ps,
                               int64_t k_hs, void* v_cache, int64_t v_ps, int64_t v_hs, float* weights, int64_t w_ps,
                               int64_t w_hs, int pages, int page, const int32_t* table, int64_t ldt, int width,
                               const int32_t* lengths, int32_t* new_lengths, const int32_t* cu_seqlens, int batch,
                               int T, int kv_heads, int head_dim, int32_t* status, hipStream_t stream) {
  const char* what = "ditk_kv_append";
  if (int rc = kv_check_pages(what, table, lengths, status, batch, width, ldt, pages, page, kv_heads, head_dim)) return rc;
  if (int rc = kv_check_tensor(what, k_cache, k_ps, k_hs, page, head_dim)) return rc;
  if (int rc = kv_check_tensor(what, v_cache, v_ps, v_hs, page, head_dim)) return rc;
  const int64_t row = (int64_t)kv_heads * head_dim;
  DITK_REQUIRE(T >= 0 && T < (1 << 30) && row < (1 << 30) && (T == 0 || (k && v)), "%s: bad rows", what);
  DITK_REQUIRE(cu_seqlens != nullptr || T == batch, "%s: %d rows for %d sequences", what, T, batch);
  DITK_REQUIRE(ldk % 8 == 0 && ldv % 8 == 0 && (T <= 1 || (ldk >= row && ldv >= row)) && ((uintptr_t)k % 16) == 0 &&
                   ((uintptr_t)v % 16) == 0,
               "%s: rows must be 16-byte aligned", what);
  DITK_REQUIRE(batch == 0 || new_lengths, "%s: null lengths", what);
  if (batch == 0) return 0;
  const KvPages t{table, ldt, lengths, pages, log2_of(page), width * page, status};
  const KvTensor kc{(bf16_t*)k_cache, k_ps, k_hs}, vc{(bf16_t*)v_cache, v_ps, v_hs};
  const KvWeights w{weights, w_ps, w_hs};
  const int per = (int)(row / 8);
  const int64_t wgs = ((int64_t)T * per + 255) / 256;
  const dim3 grid((unsigned)(wgs < 1 ? 1 : wgs > (1 << 20) ? 1 << 20 : wgs), T ? 2 : 1);
  auto kern = head_dim == 128 ? kv_append_kernel<4> : kv_append_kernel<3>;
  kern<<<grid, 256, 0, stream>>>(t, kc, vc, w, (const bf16_t*)k, ldk, (const bf16_t*)v, ldv, new_lengths, cu_seqlens,
                                 batch, T, per);
  return ditk_check_launch(what);
}

DITK_EXPORT int ditk_kv_evict(void* k_cache, int64_t k_ps, int64_t k_hs, void* v_cache, int64_t v_ps, int64_t v_hs,
                              float* weights, int64_t w_ps, int64_t w_hs, int pages, int page, const int32_t* table,
                              int64_t ldt, int width, const int32_t* lengths, int max_len, const int32_t* out_table,
                              int64_t ldo, int out_width, int32_t* new_lengths, int keep, int recent, int32_t* slots,
                              int batch, int kv_heads, int head_dim, int32_t* status, hipStream_t stream) {
  const char* what = "ditk_kv_evict";
  if (int rc = kv_check_pages(what, table, lengths, status, batch, width, ldt, pages, page, kv_heads, head_dim)) return rc;
  if (int rc = kv_check_pages(what, out_table, lengths, status, batch, out_width, ldo, pages, page, kv_heads, head_dim)) return rc;
  if (int rc = kv_check_tensor(what, k_cache, k_ps, k_hs, page, head_dim)) return rc;
  if (int rc = kv_check_tensor(what, v_cache, v_ps, v_hs, page, head_dim)) return rc;
  DITK_REQUIRE(weights != nullptr, "%s: the cache has no weights", what);
  DITK_REQUIRE(keep > 0 && recent >= 0 && recent <= keep && max_len >= 0, "%s: bad keep %d, recent %d or max_len %d",
               what, keep, recent, max_len);
  DITK_REQUIRE(batch == 0 || (new_lengths && slots), "%s: null output or workspace", what);
  if (batch == 0) return 0;
  const int most = width * page < max_len ? width * page : max_len, m = most < keep ? most : keep;
  DITK_REQUIRE((int64_t)out_width * page >= m, "%s: the new pages hold %lld slots, %d stay", what,
               (long long)out_width * page, m);
  const KvPages t{table, ldt, lengths, pages, log2_of(page), most, status};
  const KvPages to{out_table, ldo, lengths, pages, log2_of(page), out_width * page, status};
  const KvTensor kc{(bf16_t*)k_cache, k_ps, k_hs}, vc{(bf16_t*)v_cache, v_ps, v_hs};
  const KvWeights w{weights, w_ps, w_hs};
  kv_select_kernel<<<dim3(kv_heads, batch), 1024, 0, stream>>>(t, w, keep, recent, slots, new_lengths);
  if (int rc = ditk_check_launch(what)) return rc;
  if (m == 0) return 0;
  const int per = head_dim == 128 ? 16 : 32;
  auto kern = head_dim == 128 ? kv_move_kernel<4> : kv_move_kernel<3>;
  kern<<<dim3((m + per - 1) / per, kv_heads, batch), 256, 0, stream>>>(t, to, kc, vc, w, keep, slots);
  return ditk_check_launch(what);
}
