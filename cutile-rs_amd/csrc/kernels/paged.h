// A batch of sequences whose keys and values lie on the pages of one cache, as the host hands it to the kernels and as they find their way in it.
//
// New tokens of sequence b: rows starts[b] .. starts[b + 1] of q, new_k, new_v or out; lens[b] tokens in the cache, the new ones last, so new
// token i stands at position lens[b] - (starts[b + 1] - starts[b]) + i.  Position p lies on page table[b, p / page_size], row p % page_size.
// All of this is device memory that no host check has seen: starts are cut to the rows there are, lengths to what the table can hold (2^30 at most), and a page
// outside the cache is neither read nor written.
#pragma once
#include <stdint.h>

namespace cutile {

struct PagedCache {
  const void *k, *v;                              // [pages, page_size, heads, D], both laid out alike
  const uint8_t *ks, *vs;                         // mxfp8: e8m0 scales [pages, page_size, heads, D / 32], alike too
  int64_t page_bytes, row_bytes, head_bytes;      // of k and v
  int64_t s_page, s_row, s_head;                  // of the scales
  const int32_t *table, *starts, *lens;
  int64_t table_row;                              // entries from one sequence's pages to the next one's
  int32_t pages, page_size, table_pages, batch, heads, tokens;
};

// How a launch of the attention deals out its work (paged_attention.hip).
struct PagedPlan {
  float* partials;                      // results of workgroups that share the keys of a tile; counters are 0 between launches
  uint32_t* counters;
  float scale_log2e;                    // of q's magnitude, above 0; its sign, and a scale of 0, are in the two masks
  uint32_t q_and, q_xor;
  int32_t window, group;                // keys a token sees (0: all), query heads of a KV head
  int32_t few_rows;                     // sequences of up to so many rows (token, head of the group) are tiles of their own
  int32_t tile_rows;                    // of the other sequences
  int32_t long_tiles, long_shares, long_keys;   // numbers of their tiles, workgroups to a tile, keys to a workgroup
  int32_t few_shares, few_keys;
  int32_t few_slot_rows;                // rows of a small tile's partial result
};

}  // namespace cutile

#ifdef __HIP_DEVICE_COMPILE__
#include <hip/hip_runtime.h>

namespace cutile {
namespace paged {

struct Sequence {
  int32_t first, count;   // its rows of the new tokens
  int32_t len, held;      // tokens it has, and those that the table has pages for
  __device__ __forceinline__ int32_t position(int32_t i) const { return len - count + i; }
};
__device__ __forceinline__ Sequence sequence(const PagedCache& c, int32_t b) {
  Sequence s;
  s.first = min(max(c.starts[b], 0), c.tokens);
  s.count = min(max(c.starts[b + 1], s.first), c.tokens) - s.first;
  s.len = max(c.lens[b], 0);
  s.held = (int32_t)min(min((int64_t)s.len, (int64_t)1 << 30), (int64_t)c.table_pages * c.page_size);
  return s;
}

// The last sequence b whose key(b) is at most `want` (key does not fall with b), or 0: found by a whole wavefront with the same `want`, 64 ways a step.
template <typename F>
__device__ __forceinline__ int32_t find_sequence(int32_t batch, int64_t want, F&& key) {
  const int32_t lane = threadIdx.x & 63;
  int32_t lo = 0, n = batch;
  while (n > 1) {
    const int32_t step = (n + 63) / 64;
    const bool there = (int64_t)lane * step < n && key(lo + lane * step) <= want;
    const int32_t before = max(__builtin_popcountll(__builtin_amdgcn_ballot_w64(there)), 1) - 1;
    lo += before * step;
    n = min(step, n - before * step);
  }
  return lo;
}

// The page that holds position p of sequence b, or -1 if the table names none of the cache.  p < Sequence::held.
__device__ __forceinline__ int32_t page_or_none(int32_t entry, int32_t pages) { return (uint32_t)entry < (uint32_t)pages ? entry : -1; }

}  // namespace paged
}  // namespace cutile
#endif
