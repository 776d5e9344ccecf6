// What the kernels of the paged 16-bit cache share.
#pragma once

#include "nkv_block.cuh"
#include "nkv_page_plan.h"

namespace nkv {

constexpr int MOST_KEPT = 64;        // caches of one launch that keeps accepted rows; more are cut

// Device arrays of nkv_page_cache from one of its sequences on.  Table, lengths and counts are device memory that the host
// does not see: whatever they hold, no access leaves the arrays.  What does not fit is left out and reported in the status word.
struct PageArrays {
  uint16_t* k;
  uint16_t* v;
  const int32_t* table;
  const int32_t* lengths;
  int kv_heads, pages, shift, row_pages;   // 1 << shift tokens a page
};
PageArrays page_arrays(const nkv_page_cache& c, int first);

constexpr int STATUS_PAGE = 920;     // a token without a page, a length, count or path out of range
constexpr int STATUS_TREE = 921;     // a parent that does not come before its node

__device__ __forceinline__ void report(int32_t* status, int code) { atomicCAS(status, 0, code); }

using page::Extent;
__device__ __forceinline__ Extent extent_of(const PageArrays& c, const int32_t* counts, int tokens, int b, bool& bad) {
  return page::extent_in(__ldg(c.lengths + b), counts ? __ldg(counts + b) : tokens, tokens, c.row_pages << c.shift, bad);
}

// page of a token; -1 where the table names none
__device__ __forceinline__ int page_of(const PageArrays& c, int b, int token) {
  const int entry = token >> c.shift;
  const int page = entry < c.row_pages ? __ldg(c.table + static_cast<size_t>(b) * c.row_pages + entry) : -1;
  return static_cast<unsigned>(page) < static_cast<unsigned>(c.pages) ? page : -1;
}
// element at which a token's row of a kv head begins
__device__ __forceinline__ size_t row_at(const PageArrays& c, int page, int head, int token, int d) {
  return ((static_cast<size_t>(page) * c.kv_heads + head) * (size_t(1) << c.shift) + (token & ((1 << c.shift) - 1))) * d;
}

// ---- attention ----
// One call, from one of its sequences on.  The queries of a kv head are rows r = token * group + (head within the group).
struct PageCall {
  const uint16_t* q;
  long long q_batch, q_token, q_head;
  uint16_t* out;
  float* lse;
  const int32_t* counts;   // or NULL
  const uint32_t* mask;    // [tokens][words] of a sequence
  long long mask_batch;    // words from one sequence's to the next; 0: shared
  int words, sight;
  int tokens, heads, group, rows;
  float scale_log2;        // scale * log2(e)
  int q_vector;            // the queries' rows start on 16 bytes
};

// page::sight_bits of query t of sequence b
__device__ __forceinline__ uint32_t sight_of(const PageCall& a, const Extent& e, int b, int t, int first) {
  return page::sight_bits(a.sight, e, t, first, [&](int w) {
    return static_cast<unsigned>(w) < static_cast<unsigned>(a.words)
               ? __ldg(a.mask + b * a.mask_batch + static_cast<long long>(t) * a.words + w) : 0u;
  });
}

// sequences [0, n) of `c` from one of the batch's on (nkv_page_tile.cu)
size_t page_tile_bytes(const PageArrays& c, int n, int rows, int d);
int page_tile(const PageArrays& c, const PageCall& a, int n, int dtype, int d, void* workspace, int32_t* status, cudaStream_t stream);

}  // namespace nkv
