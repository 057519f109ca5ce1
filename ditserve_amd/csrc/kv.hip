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
  DITK_REQUIRE(status != nullptr && (batch == 0 || ((table || width == 0) && lengths)), "%s: null table", what);
  DITK_REQUIRE(width >= 0 && ldt >= width && (int64_t)width * page < (1ll << 30), "%s: bad page table", what);
  return 0;
}

int kv_check_tensor(const char* what, const void* p, int64_t ps, int64_t hs) {
  DITK_REQUIRE(p != nullptr, "%s: null cache", what);
  DITK_REQUIRE(((uintptr_t)p % 16) == 0 && ps % 8 == 0 && hs % 8 == 0 && ps >= 0 && hs >= 0,
               "%s: the cache's heads must be 16-byte aligned", what);
  return 0;
}

int kv_check_weights(const char* what, const float* p, int64_t ps, int64_t hs) {
  DITK_REQUIRE(p == nullptr || (((uintptr_t)p % 4) == 0 && ps >= 0 && hs >= 0), "%s: bad strides or address of the weights", what);
  return 0;
}

namespace {

constexpr int kCuLds = 1024;

// Rows of new keys and values into the slots behind each sequence's last: row i of segment b goes to slot lengths[b] + i.
// A thread moves 16 bytes of K and of V; `per` of them make a row.  Memory bounds it: 16384 rows of 8 heads of 128, 134 MB
// read and written, 28 us (4.8 TB/s); one row each of 64 sequences 3.5 us, a launch and three reads after one another.
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
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < nseg; b += 256) {
      const int n = kv_length(t, b, true), add = cu != nullptr ? cu[b + 1] - cu[b] : 1;
      if (n + (int64_t)add > t.most) *t.status = 1;
      new_lengths[b] = (int)min((int64_t)t.most, n + (int64_t)add);
    }
  const int64_t total = (int64_t)T * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int row = total < (1ll << 32) ? (int)((uint32_t)i / (uint32_t)per) : (int)(i / per);
    const int c = (int)(i - (int64_t)row * per);
    const u32x4_t xk = *reinterpret_cast<const u32x4_t*>(k + row * ldk + c * 8);
    const u32x4_t xv = *reinterpret_cast<const u32x4_t*>(v + row * ldv + c * 8);
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
    const int64_t dst = (((int64_t)j << LOG_CH) + (c & ((1 << LOG_CH) - 1))) * 8;
    *reinterpret_cast<u32x4_t*>(kc.p + p * kc.ps + h * kc.hs + dst) = xk;
    *reinterpret_cast<u32x4_t*>(vc.p + p * vc.ps + h * vc.hs + dst) = xv;
    if (w.p != nullptr && (c & ((1 << LOG_CH) - 1)) == 0) w.p[p * w.ps + h * w.hs + j] = 0.f;
  }
}

// fp32 -> uint32 whose order is the floats', from -inf's 0x7fffff to +inf's 0xff800000: -0 is 0, and a NaN is -inf
__device__ __forceinline__ uint32_t order_of(float f) {
  const uint32_t u = __float_as_uint(fmaxf(f + 0.f, -INFINITY));
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}

// The slots that stay, ascending, of a (sequence, key head): of its `old` slots before the recent ones those above a
// threshold weight, and the lowest of those at it.  The threshold is the want-th largest of the weights' 32-bit order
// (order_of), found 11, 11 and 10 bits at a time by counting digits in LDS, the largest first.
//
// A workgroup of 1024 threads keeps KPT weights a thread in registers; wave w has KPT * 64 slots from its part's start +
// w * KPT * 64 on, 64 consecutive ones in each register, so ballots give the places in the list.  Rows that one
// workgroup holds take one launch (kv_select_kernel).  Longer ones are cut into parts of 1024 * KPT slots and take four,
// each of every part: counts of the first digit; that digit from all parts' counts, and counts of the second; the same
// for the third; the threshold and the list (kv_count_kernel, kv_list_kernel).  Counts have a place for each part, so
// that nothing has to be cleared and no order matters.
//
// Latency bounds it: reads that wait for each other, and some 300 vector operations a wave on the few CUs that have one
// of the workgroups.  64 rows of 8192 slots 10 us; 8 of 131072 in 16 parts 4.5, 6, 6 and 8 us for the four launches.
constexpr int kBins = 2048, kCopies = 4;
constexpr int kShift[3] = {21, 10, 0};

struct Row {
  int n, m, r, old, want;  // slots, slots that stay, recent and older ones, and how many of these stay
  bool sort;               // whether weights decide
};
__device__ __forceinline__ Row row_of(const KvPages& t, int b, int keep, int recent, bool tell) {
  Row x;
  x.n = kv_length(t, b, tell);
  x.m = min(x.n, keep);
  x.r = min(recent, x.m);
  x.old = x.n - x.r;
  x.want = x.m - x.r;
  x.sort = x.n > x.m && x.want > 0;
  return x;
}

// A thread's keys, 0 behind the last slot.  Its table entries (of slots that the call's lengths may have) are asked for before the sequence's
// length is there, and its weights become keys after whatever else a launch reads is asked for: 64 rows of 8192 slots
// 12.2 -> 10.6 us.
template <int KPT>
struct Keys {
  int page[KPT];
  float raw[KPT];
  uint32_t key[KPT];

  __device__ __forceinline__ int slot(int first, int i) const {
    return first + (int)(threadIdx.x >> 6) * (KPT * 64) + (int)(threadIdx.x & 63) + i * 64;
  }
  __device__ __forceinline__ void load_pages(const KvPages& t, int b, int first) {
    if (t.most == 0) return;  // (no table: no keys either)
    const int32_t* row = t.table + b * t.ldt;
#pragma unroll
    for (int i = 0; i < KPT; ++i) page[i] = row[(uint32_t)min(slot(first, i), t.most - 1) >> t.page_log2];
  }
  // (of a page that the cache lacks, and behind the last slot, some other weight: without branches all loads go out at once)
  __device__ __forceinline__ void load_weights(const KvPages& t, const KvWeights& w, int h, int first, int old) {
    const float* row = w.p + h * w.hs;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const int at = slot(first, i);
      const bool ok = (unsigned)page[i] < (unsigned)t.pages;
      bad |= !ok && at < old;
      raw[i] = row[(uint64_t)(ok ? (uint32_t)page[i] : 0u) * (uint32_t)w.ps + (at & ((1 << t.page_log2) - 1))];
    }
    if (bad) *t.status = 1;
  }
  __device__ __forceinline__ void make(const KvPages& t, int first, int old) {
#pragma unroll
    for (int i = 0; i < KPT; ++i)
      key[i] = slot(first, i) < old ? order_of((unsigned)page[i] < (unsigned)t.pages ? raw[i] : -INFINITY) : 0u;
  }
  // every slot stays, or none: keys above a threshold of 0, or not.  (No weights are read: pages that the cache lacks are
  // reported here.)
  __device__ __forceinline__ void make_all(const KvPages& t, int first, int old, bool stay) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const bool mine = slot(first, i) < old;
      bad |= mine && (unsigned)page[i] >= (unsigned)t.pages;
      key[i] = stay && mine ? 1u : 0u;
    }
    if (bad) *t.status = 1;
  }
};

// counts[d] += keys of this workgroup whose k-th digit is d and that agree with `top` above it.  Neighbouring lanes count in
// kCopies places, so that keys of few digits (a first digit is a sign, an exponent and two bits) meet less.
template <int KPT>
__device__ __forceinline__ void count_digits(const uint32_t (&key)[KPT], int k, uint32_t top, int (*counts)[kCopies]) {
  int* mine = counts[0] + (threadIdx.x % kCopies);
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const uint32_t d = k == 0 ? key[i] >> kShift[0] : k == 1 ? (key[i] >> kShift[1]) % kBins : key[i] % (1u << kShift[1]);
    if (k == 0 ? key[i] != 0 : (key[i] ^ top) < 1u << kShift[k - 1]) atomicAdd(&mine[d * kCopies], 1);
  }
}

__device__ __forceinline__ void clear_counts(int (*counts)[kCopies]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) *reinterpret_cast<u32x4_t*>(counts[i * 1024 + threadIdx.x]) = u32x4_t{0, 0, 0, 0};
}

// counts of a thread's two digits, 2047 - 2 tid and the one below: the larger first
__device__ __forceinline__ void my_digits(const int (*counts)[kCopies], int (&v)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(counts[kBins - 1 - 2 * threadIdx.x - i]);
    v[i] = (int)((x[0] + x[1]) + (x[2] + x[3]));
  }
}

// sum of the first `wave` of 16 numbers in LDS (read side by side: one after another they cost a latency each)
__device__ __forceinline__ int sum_before(const int (&sums)[16], int wave) {
  int x[16], n = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = sums[i];
#pragma unroll
  for (int i = 0; i < 16; ++i) n += i < wave ? x[i] : 0;
  return n;
}

// the digit of the want-th largest, how many of its keys are wanted, and whether that is all of them (then the digits
// below do not matter: with them 0, the threshold is at or below each of these keys): v as my_digits gives it
__device__ __forceinline__ bool find_digit(const int (&v)[2], int& want, int& digit, int (*sums)[16], int* pick) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = kBins - 1 - 2 * tid;
  int incl = wave_scan(v[0] + v[1]);
  if (lane == 63) sums[0][wave] = incl;
  __syncthreads();
  incl += sum_before(sums[0], wave);
  const int before = incl - v[0] - v[1];
  if (before < want && want <= incl) {
    const bool in0 = before + v[0] >= want;
    pick[0] = in0 ? hi : hi - 1;
    pick[1] = in0 ? want - before : want - before - v[0];
    pick[2] = pick[1] == (in0 ? v[0] : v[1]);
  }
  __syncthreads();
  digit = pick[0];
  want = pick[1];
  const bool all = pick[2] != 0;
  __syncthreads();
  return all;
}

// Writes this workgroup's slots that stay: those above `top`, and those equal to it while fewer than `want` of them came
// before.  at, tie: slots that stay, and equal ones, in the parts before.
template <int KPT>
__device__ __forceinline__ void write_list(const uint32_t (&key)[KPT], int first, uint32_t top, int want, int at, int tie,
                                           int (*sums)[16], int32_t* out) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int na = 0, nt = 0;
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    na += __popcll(__ballot(key[i] > top));
    nt += __popcll(__ballot(key[i] == top));
  }
  if (lane == 0) sums[0][wave] = na, sums[1][wave] = nt;
  __syncthreads();
  tie = __builtin_amdgcn_readfirstlane(tie + sum_before(sums[1], wave));
  at = __builtin_amdgcn_readfirstlane(at + sum_before(sums[0], wave) + min(tie, want));
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const uint64_t eqs = __ballot(key[i] == top);
    uint64_t stays = __ballot(key[i] > top);
    if (tie < want) {
      const bool low = tie + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(eqs >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)eqs, 0)) < want;
      stays |= eqs & __ballot(low);
      tie += __popcll(eqs);
    }
    if (stays >> lane & 1)
      out[at + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(stays >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)stays, 0))] =
          first + wave * (KPT * 64) + i * 64 + lane;
    at += __popcll(stays);
  }
}

template <int KPT>
__global__ __launch_bounds__(1024) void kv_select_kernel(KvPages t, KvWeights w, int keep, int recent,
                                                         int32_t* __restrict__ slots, int32_t* __restrict__ new_lengths) {
  __shared__ __align__(16) int counts[2][kBins][kCopies];
  __shared__ int sums[2][16], pick[3];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  Keys<KPT> keys;
  keys.load_pages(t, b, 0);
  const Row x = row_of(t, b, keep, recent, tid == 0);
  int32_t* out = slots + ((int64_t)b * gridDim.x + h) * keep;
  if (h == 0 && tid == 0) new_lengths[b] = x.m;
  for (int i = tid; i < x.r; i += 1024) out[x.m - x.r + i] = x.old + i;
  uint32_t top = 0;
  int want = x.want;
  if (x.sort) {
    keys.load_weights(t, w, h, 0, x.old);
    clear_counts(counts[0]);
    __syncthreads();
    keys.make(t, 0, x.old);
    bool all = false;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (all) break;
      if (k < 2) clear_counts(counts[(k + 1) & 1]);  // (read two digits ago)
      count_digits<KPT>(keys.key, k, top, counts[k & 1]);
      __syncthreads();
      int d, v[2];
      my_digits(counts[k & 1], v);
      all = find_digit(v, want, d, sums, pick);
      top |= (uint32_t)d << kShift[k];
    }
    if (all) {  // every key that agrees with `top` stays, as one above it (no key is below 2^21, -inf's first digit)
      top -= 1;
      want = 0;
    }
  } else {
    keys.make_all(t, 0, x.old, x.n <= x.m);
    want = 0;
  }
  write_list<KPT>(keys.key, 0, top, want, 0, 0, sums, out);
}

// what the launches for long rows keep of a row
struct Counts {
  uint32_t* digits;  // [rows][parts][3][kBins / 2]: counts of 16 bits (a part holds 32768 keys at most), the lower digit's first
  int* above;   // [rows][parts][2]: keys above the first digit, and at it but above the second
  int* pick;    // [rows][2][2]: digits found, and how many are wanted of what agrees with them (0: all of it)
  int parts;
};

// counts of this thread's two digits (as my_digits): in all parts, and in those before `part`.  Sixteen parts' loads at a
// time.
__device__ __forceinline__ void sum_parts(const Counts& c, int64_t row, int digit, int parts, int part, int (&all)[2],
                                          int (&before)[2]) {
  all[0] = all[1] = before[0] = before[1] = 0;
  const uint32_t* from = c.digits + (row * c.parts * 3 + digit) * (kBins / 2) + kBins / 2 - 1 - threadIdx.x;
  for (int p = 0; p < parts; p += 16) {
    uint32_t v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = from[(int64_t)min(p + k, parts - 1) * 3 * (kBins / 2)];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int n[2] = {(int)(v[k] >> 16), (int)(v[k] & 0xffffu)};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        all[i] += p + k < parts ? n[i] : 0;
        before[i] += p + k < part ? n[i] : 0;
      }
    }
  }
}

// counts of digit PASS of a part; PASS > 0: finds the digit before it first
template <int KPT, int PASS>
__global__ __launch_bounds__(1024) void kv_count_kernel(KvPages t, KvWeights w, int keep, int recent, Counts c) {
  __shared__ __align__(16) int counts[kBins][kCopies];
  __shared__ int sums[2][16], pick[3];
  const int part = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, first = part * (KPT * 1024);
  Keys<KPT> keys;
  keys.load_pages(t, b, first);
  const Row x = row_of(t, b, keep, recent, false);
  if (!x.sort || first >= x.old) return;
  const int64_t row = (int64_t)b * gridDim.y + h;
  const int parts = (x.old - 1) / (KPT * 1024) + 1;
  if (PASS == 2 && c.pick[row * 4 + 1] == 0) {  // the first digit was enough
    if (tid == 0) {
      c.above[(row * c.parts + part) * 2 + 1] = 0;
      if (part == 0) c.pick[row * 4 + 2] = c.pick[row * 4 + 3] = 0;
    }
    return;
  }
  uint32_t top = 0;
  keys.load_weights(t, w, h, first, x.old);
  clear_counts(counts);
  if constexpr (PASS > 0) {
    int v[2], mine[2];
    sum_parts(c, row, PASS - 1, parts, part, v, mine);
    int want = x.want, d;
    if (PASS == 2) {
      top = (uint32_t)c.pick[row * 4] << kShift[0];
      want = c.pick[row * 4 + 1];
    }
    // this part's keys above the digit (all: and at it), among those that agree with the digits before
    const uint32_t past = PASS == 2 ? top + (1u << kShift[0]) : 0u;
    const bool all = find_digit(v, want, d, sums, pick);
    keys.make(t, first, x.old);
    top |= (uint32_t)d << kShift[PASS - 1];
    if (part == 0 && tid == 0) {
      c.pick[row * 4 + 2 * (PASS - 1)] = d;
      c.pick[row * 4 + 2 * (PASS - 1) + 1] = all ? 0 : want;
    }
    const uint32_t least = all ? top : top + (1u << kShift[PASS - 1]);
    int na = 0;
#pragma unroll
    for (int i = 0; i < KPT; ++i) na += __popcll(__ballot(keys.key[i] - least < past - least));
    if ((tid & 63) == 0) sums[1][tid >> 6] = na;
    __syncthreads();
    if (tid == 0) c.above[(row * c.parts + part) * 2 + PASS - 1] = sum_before(sums[1], 16);
    if (all) return;
  } else {
    __syncthreads();
    keys.make(t, first, x.old);
  }
  count_digits<KPT>(keys.key, PASS, top, counts);
  __syncthreads();
  int n[2];
  my_digits(counts, n);
  c.digits[((row * c.parts + part) * 3 + PASS) * (kBins / 2) + kBins / 2 - 1 - tid] = (uint32_t)n[0] << 16 | (uint32_t)n[1];
}

template <int KPT>
__global__ __launch_bounds__(1024) void kv_list_kernel(KvPages t, KvWeights w, int keep, int recent, Counts c,
                                                       int32_t* __restrict__ slots, int32_t* __restrict__ new_lengths) {
  __shared__ int sums[2][16], pick[3], before[2];
  const int part = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int first = part * (KPT * 1024);
  Keys<KPT> keys;
  keys.load_pages(t, b, first);
  const Row x = row_of(t, b, keep, recent, part == 0 && tid == 0);
  const int64_t row = (int64_t)b * gridDim.y + h;
  int32_t* out = slots + row * keep;
  if (part == 0 && h == 0 && tid == 0) new_lengths[b] = x.m;
  for (int i = part * 1024 + tid; i < x.r; i += gridDim.x * 1024) out[x.m - x.r + i] = x.old + i;
  if (first >= x.old) return;
  uint32_t top = 0;
  int want = x.want, at = first, tie = 0;  // (all stay: every slot before)
  if (x.sort) {
    const int parts = (x.old - 1) / (KPT * 1024) + 1;
    keys.load_weights(t, w, h, first, x.old);
    if (tid < 2) before[tid] = 0;
    int na = 0;
    for (int p = tid; p < part; p += 1024) na += c.above[(row * c.parts + p) * 2] + c.above[(row * c.parts + p) * 2 + 1];
    top = (uint32_t)c.pick[row * 4] << kShift[0] | (uint32_t)c.pick[row * 4 + 2] << kShift[1];
    want = c.pick[row * 4 + 3];
    if (want == 0) {  // all that agrees with the digits found stays
      top -= 1;
      __syncthreads();
    } else {
      int v[2], mine[2], d;  // counts of the last digit
      sum_parts(c, row, 2, parts, part, v, mine);
      find_digit(v, want, d, sums, pick);
      top |= (uint32_t)d;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int bin = kBins - 1 - 2 * tid - i;
        if (bin > d) na += mine[i];
        if (bin == d) before[1] = mine[i];
      }
    }
    keys.make(t, first, x.old);
    if (na) atomicAdd(&before[0], na);  // (whole numbers: no order matters)
    __syncthreads();
    at = before[0];
    tie = before[1];
  } else {
    keys.make_all(t, first, x.old, x.n <= x.m);
    want = 0;
  }
  write_list<KPT>(keys.key, first, top, want, at, tie, sums, out);
}

// Copies the slots that stay into the pages of `to`: 16 slots of a (key head, sequence) a workgroup, 16 bytes a thread.
// One whose page the cache lacks becomes zeros, weight too, and is reported (of the recent ones no other kernel sees the
// pages): the slots behind it keep their places, as in every key head.
// The old slots are not read again and go past the caches (134 MB copied 30.4 -> 26.0 us: 5.2 TB/s, what a copy reaches);
// the next step reads the new ones.
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
  const int p = kv_page(t, b, i, ok, false), q = kv_page(to, b, j, ok_to, false);
  if (!ok || !ok_to) *t.status = 1;  // (once both are there: a branch behind the first alone, 8 x 8192 slots 33 us for 32)
  if (!ok_to) return;
  const int64_t src = (((int64_t)(i & low) << LOG_CH) + c) * 8, dst = (((int64_t)(j & low) << LOG_CH) + c) * 8;
  u32x4_t k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
  if (ok) {
    k = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(kc.p + p * kc.ps + h * kc.hs + src));
    v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(vc.p + p * vc.ps + h * vc.hs + src));
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
  if (int rc = kv_check_tensor(what, k_cache, k_ps, k_hs)) return rc;
  if (int rc = kv_check_tensor(what, v_cache, v_ps, v_hs)) return rc;
  if (int rc = kv_check_weights(what, weights, w_ps, w_hs)) return rc;
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
  const unsigned grid = (unsigned)(wgs < 1 ? 1 : wgs > (1 << 20) ? 1 << 20 : wgs);
  auto kern = head_dim == 128 ? kv_append_kernel<4> : kv_append_kernel<3>;
  kern<<<grid, 256, 0, stream>>>(t, kc, vc, w, (const bf16_t*)k, ldk, (const bf16_t*)v, ldv, new_lengths, cu_seqlens,
                                 batch, T, per);
  return ditk_check_launch(what);
}

namespace {
// launches of the selection: rows of up to 1024 * kpt slots by one workgroup each (parts 1), longer ones in parts.  Parts of
// 8192 slots put more CUs to a row, parts of 32768 leave fewer counts, which each workgroup of a row reads whole (sixteen
// parts at a time: the border).  Eight key heads, the whole call, us with parts of 8192 and of 32768: 1 x 40000 slots 31 and 53,
// 1 x 131072 49 and 71, 8 x 131072 289 and 278; beyond the border 1 x 262144 54 and 72, 1 x 524288 71 and 72, 8 x 262144
// 350 and 334, 1 x 1000000 147 and 80, 4 x 1000000 500 and 301.
struct SelectPlan {
  int kpt, parts;
};
SelectPlan select_plan(int most) {
  for (int kpt : {1, 4, 8, 32})
    if (most <= 1024 * kpt) return {kpt, 1};
  const int kpt = most <= 16 * 8192 ? 8 : 32;
  return {kpt, (most - 1) / (1024 * kpt) + 1};
}
}  // namespace

DITK_EXPORT int64_t ditk_kv_evict_workspace(int batch, int kv_heads, int most, int keep) {
  if (batch <= 0 || kv_heads <= 0 || most < 0 || most >= (1 << 30) || keep <= 0) return 0;
  const int64_t rows = (int64_t)batch * kv_heads;
  const SelectPlan pl = select_plan(most);
  return 4 * (rows * keep + (pl.parts > 1 ? rows * ((int64_t)pl.parts * (3 * kBins / 2 + 2) + 4) : 0));
}

DITK_EXPORT int ditk_kv_evict(void* k_cache, int64_t k_ps, int64_t k_hs, void* v_cache, int64_t v_ps, int64_t v_hs,
                              float* weights, int64_t w_ps, int64_t w_hs, int pages, int page, const int32_t* table,
                              int64_t ldt, int width, const int32_t* lengths, int max_len, const int32_t* out_table,
                              int64_t ldo, int out_width, int32_t* new_lengths, int keep, int recent, void* workspace,
                              int64_t workspace_bytes, int batch, int kv_heads, int head_dim, int32_t* status,
                              hipStream_t stream) {
  const char* what = "ditk_kv_evict";
  if (int rc = kv_check_pages(what, table, lengths, status, batch, width, ldt, pages, page, kv_heads, head_dim)) return rc;
  if (int rc = kv_check_pages(what, out_table, lengths, status, batch, out_width, ldo, pages, page, kv_heads, head_dim)) return rc;
  if (int rc = kv_check_tensor(what, k_cache, k_ps, k_hs)) return rc;
  if (int rc = kv_check_tensor(what, v_cache, v_ps, v_hs)) return rc;
  if (int rc = kv_check_weights(what, weights, w_ps, w_hs)) return rc;
  DITK_REQUIRE(weights != nullptr, "%s: the cache has no weights", what);
  DITK_REQUIRE(w_ps < (1ll << 32), "%s: the weights' pages are too far apart", what);
  DITK_REQUIRE(keep > 0 && recent >= 0 && recent <= keep && max_len >= 0, "%s: bad keep %d, recent %d or max_len %d",
               what, keep, recent, max_len);
  if (batch == 0) return 0;
  const int most = width * page < max_len ? width * page : max_len, m = most < keep ? most : keep;
  DITK_REQUIRE(new_lengths && workspace && ((uintptr_t)workspace % 16) == 0 &&
                   workspace_bytes >= ditk_kv_evict_workspace(batch, kv_heads, most, keep),
               "%s: null output, or a workspace below %lld bytes", what,
               (long long)ditk_kv_evict_workspace(batch, kv_heads, most, keep));
  DITK_REQUIRE((int64_t)out_width * page >= m, "%s: the new pages hold %lld slots, %d stay", what,
               (long long)out_width * page, m);
  const KvPages t{table, ldt, lengths, pages, log2_of(page), most, status};
  const KvPages to{out_table, ldo, lengths, pages, log2_of(page), out_width * page, status};
  const KvTensor kc{(bf16_t*)k_cache, k_ps, k_hs}, vc{(bf16_t*)v_cache, v_ps, v_hs};
  const KvWeights w{weights, w_ps, w_hs};
  const int64_t rows = (int64_t)batch * kv_heads;
  const SelectPlan pl = select_plan(most);
  int32_t* slots = (int32_t*)workspace;
  if (pl.parts == 1) {
    auto kern = pl.kpt == 1 ? kv_select_kernel<1> : pl.kpt == 4 ? kv_select_kernel<4>
                : pl.kpt == 8 ? kv_select_kernel<8> : kv_select_kernel<32>;
    kern<<<dim3(kv_heads, batch), 1024, 0, stream>>>(t, w, keep, recent, slots, new_lengths);
    if (int rc = ditk_check_launch(what)) return rc;
  } else {
    Counts c;
    c.above = slots + rows * keep;
    c.pick = c.above + rows * pl.parts * 2;
    c.digits = (uint32_t*)(c.pick + rows * 4);
    c.parts = pl.parts;
    const dim3 grid(pl.parts, kv_heads, batch);
    const bool few = pl.kpt == 8;
    auto count0 = few ? kv_count_kernel<8, 0> : kv_count_kernel<32, 0>;
    auto count1 = few ? kv_count_kernel<8, 1> : kv_count_kernel<32, 1>;
    auto count2 = few ? kv_count_kernel<8, 2> : kv_count_kernel<32, 2>;
    auto list = few ? kv_list_kernel<8> : kv_list_kernel<32>;
    for (auto count : {count0, count1, count2}) {
      count<<<grid, 1024, 0, stream>>>(t, w, keep, recent, c);
      if (int rc = ditk_check_launch(what)) return rc;
    }
    list<<<grid, 1024, 0, stream>>>(t, w, keep, recent, c, slots, new_lengths);
    if (int rc = ditk_check_launch(what)) return rc;
  }
  if (m == 0) return 0;
  const int per = head_dim == 128 ? 16 : 32;
  auto kern = head_dim == 128 ? kv_move_kernel<4> : kv_move_kernel<3>;
  kern<<<dim3((m + per - 1) / per, kv_heads, batch), 256, 0, stream>>>(t, to, kc, vc, w, keep, slots);
  return ditk_check_launch(what);
}
