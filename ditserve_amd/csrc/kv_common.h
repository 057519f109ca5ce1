// Paged key-value caches, as every ditk_kv_* entry point reads and writes them.
//
// A cache holds `pages` pages of `page` slots (16, 32, 64, 128 or 256): keys and values of a
// (page, key head) are [page][head_dim] bf16, contiguous; pages and heads have strides of their
// own, so K and V may share a buffer.  Weights (optional) are one fp32 per (page, key head, slot).
// Slot i of sequence b is slot i % page of page table[b][i / page].
//
// Tables and lengths live on the device and are a caller's: a length outside [0, most] (most: what
// the table and the call's max_len hold) is clamped, a page outside [0, pages) is neither read nor
// written (its slots count as absent), and either sets a sticky word in pinned host memory.
#pragma once

#include "ditk_common.h"

struct KvPages {
  const int32_t* table;  // [batch][ldt]
  int64_t ldt;
  const int32_t* lengths;  // [batch]
  int pages, page_log2, most;
  int32_t* status;
};

struct KvTensor {
  bf16_t* p;
  int64_t ps, hs;  // strides of a page and of a key head, in elements
};

struct KvWeights {
  float* p;
  int64_t ps, hs;
};

// a sequence's length, clamped; `tell`: the thread that reports a bad one
__device__ __forceinline__ int kv_length(const KvPages& t, int b, bool tell) {
  const int n = t.lengths[b], c = min(max(n, 0), t.most);
  if (c != n && tell) *t.status = 1;
  return c;
}

// page of slot i (0 for one that is out of range, with ok = false)
__device__ __forceinline__ int kv_page(const KvPages& t, int b, int i, bool& ok, bool tell) {
  const int p = t.table[b * t.ldt + (i >> t.page_log2)];
  ok = (unsigned)p < (unsigned)t.pages;
  if (!ok && tell) *t.status = 1;
  return ok ? p : 0;
}

// host checks shared by the entry points
int kv_check_pages(const char* what, const void* table, const void* lengths, const void* status, int batch, int width,
                   int64_t ldt, int pages, int page, int kv_heads, int head_dim);
int kv_check_tensor(const char* what, const void* p, int64_t ps, int64_t hs);
int kv_check_weights(const char* what, const float* p, int64_t ps, int64_t hs);  // (none: fine)
