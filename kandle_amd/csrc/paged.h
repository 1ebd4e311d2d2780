// Shared by the kernels of the paged KV cache: where a token of a ragged batch sits.
#pragma once

#include "common.h"

namespace kh {

// A cache whose rows lie in pages: key/value pools [num_pages, hkv, page_size, d], a page table
// [batch, table_width] of page ids (an id outside [0, num_pages): no page), and per sequence the number
// of cached rows, the new tokens' among them.  Sequence b's new tokens are rows starts[b] ..
// starts[b + 1] - 1 of the packed token tensors (starts == nullptr: token b alone); the last of them
// is the last cached row.
struct PagedBatch {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;
  int64_t table_stride;
  int32_t batch, tokens, num_pages, page_log, table_width;
  int32_t max_len;  // no row at or behind this one is read (<= table_width << page_log)

  __device__ __forceinline__ int len(int b) const { return max(lens[b], 0); }
  // First token and token count of sequence b, inside [0, tokens) whatever the starts hold.
  __device__ __forceinline__ int first(int b) const { return starts ? min(max(starts[b], 0), tokens) : b; }
  __device__ __forceinline__ int count(int b) const {
    return starts ? max(0, min(max(starts[b + 1], 0), tokens) - first(b)) : 1;
  }
  __device__ __forceinline__ bool is_page(int id) const { return (unsigned)id < (unsigned)num_pages; }
  // The sequence that token t belongs to (-1: none), for a whole wave at once with t uniform: the
  // last one that starts at or before t, if it reaches t.
  __device__ __forceinline__ int sequence_of(int t) const {
    if (!starts) return t < batch ? t : -1;
    const int lane = threadIdx.x & 63;
    int below = 0;  // starts at or before t
    for (int b0 = 0; b0 < batch; b0 += 64) {
      const bool at = b0 + lane < batch && starts[b0 + lane] <= t;
      const int n = __popcll(__ballot(at));
      below += n;
      if (n < 64) break;
    }
    const int b = below - 1;
    return b >= 0 && t < first(b) + count(b) ? b : -1;
  }
};

inline int log2_of(int64_t v) {
  int n = 0;
  while ((int64_t(1) << n) < v) ++n;
  return n;
}

// The checks that the paged entry points share; fills `pb`.  Returns KH_OK or an error code.
int paged_batch(const char* who, const int32_t* table, const int32_t* lens, const int32_t* starts, int64_t tokens,
                int64_t batch, int64_t num_pages, int64_t page_size, int64_t table_width, int64_t table_stride,
                int64_t max_kv_len, PagedBatch* pb);

}  // namespace kh
