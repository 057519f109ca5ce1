// Causal attention of segments with few queries over many keys (causal_few.hip): which they are and how they are cut, by
// their own sizes alone, so that a segment's result does not depend on what it is packed with.
#pragma once

#include "ditk_common.h"

constexpr int kFewRows = 128, kFewKeys = 1024, kFewChunks = 128;

// The tiles of flash_fwd_asm give such a segment ceil(nq / 128) workgroups a query head that go through all its keys, 0.85
// us for every 64; here waves share them, for 16 (query, query head) rows of a key head at a time.  32 heads over 8: a
// query after 8192 keys 110 us there and 22 here, 16 109 and 36, 32 segments of 4 after 4000 317 and 115; 128 after 1000,
// one query head a key head, 21 and 18.
__host__ __device__ inline bool few_queries(int nq, int nk, int group) {
  return nq > 0 && nk >= kFewKeys && nq <= kFewRows && nq * group <= kFewRows;
}

// keys of a chunk: 256 or more (128 of few keys), whole tiles of 32; chunks and groups of 16 rows make kFewChunks at most.
// Measured: 10 queries of 5 heads a key head after 30000 keys 94 us with 256 chunks, 83 with 128; 32 segments of 4 queries
// after 4000 keys 131 us with chunks of 128 keys, 115 with 256; 32 queries after 2000 19 and 21.
__host__ __device__ inline int few_chunk(int nq, int nk, int group) {
  const int most = kFewChunks / ((nq * group + 15) / 16), c = (nk + most - 1) / most;
  const int least = nk < 2560 ? 128 : 256;
  return c <= least ? least : (c + 31) / 32 * 32;
}

// parts (rows times chunks) of a key head that a segment leaves for the join; 0 for the others
__host__ __device__ inline int few_parts(int nq, int nk, int group) {
  return few_queries(nq, nk, group) ? nq * group * ((nk - 1) / few_chunk(nq, nk, group) + 1) : 0;
}

// parts: of all segments together, a key head
int64_t causal_few_workspace(int64_t parts, int kv_heads, int head_dim);
int causal_few_launch(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* o,
                      int64_t ldo, float* lse, int64_t lse_ld, const int32_t* cu_q, const int32_t* cu_k, int nseg,
                      int heads, int kv_heads, int head_dim, float scale2, void* workspace, int64_t parts,
                      hipStream_t stream);
