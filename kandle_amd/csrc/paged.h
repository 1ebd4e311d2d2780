// Shared by the kernels of the paged KV cache: where a token of a ragged batch sits.
#pragma once

#include "common.h"
#include "spans.h"

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
    for (int b0 = 0; b0 < batch; b0 += 256) {
      int n = 0;
#pragma unroll
      for (int k = 0; k < 256; k += 64) n += __popcll(__ballot(b0 + k + lane < batch && starts[min(b0 + k + lane, batch)] <= t));
      below += n;
      if (n < 256) break;
    }
    const int b = below - 1;  // (where the starts do not grow, t may lie before its first token)
    return b >= 0 && t >= first(b) && t < first(b) + count(b) ? b : -1;
  }
};

struct PagedStrides {
  int64_t qt, qh, kp, kh, kr, vp, vh, vr, ot, oh;
};

// The (sequence, tile) of workgroup column x of a grid over tiles of `rows` packed rows: sequence b has
// ceil(min(n_b, max_new) * G / rows) tiles, none unless above < min(n_b, max_new) * G <= upto.  Every wave of the
// workgroup computes it for itself, from 256 sequences at a time, four per lane: workgroups start with this, and
// with one sequence per lane 256 ragged chunks of up to 300 tokens of 500 took 443 us rather than 389.  b = -1:
// nothing to do.
struct Tile {
  int b = -1, row0 = 0, rows = 0;  // first packed row, packed rows of the sequence
  int t0 = 0, n = 0, len = 0;      // first token, new tokens, cached rows
};
__device__ __forceinline__ Tile find_tile(const PagedBatch& pb, int x, int G, int rows, int max_new, int above, int upto) {
  Tile t;
  int at = x;
  if (pb.starts == nullptr) {
    const int per = (G + rows - 1) / rows;
    t.b = __builtin_amdgcn_readfirstlane(x / per);
    at = x - t.b * per;
    if (t.b >= pb.batch || G <= above || G > upto) t.b = -1;
    if (t.b < 0) return t;
    t.t0 = t.b;
    t.n = 1;
    t.len = pb.len(t.b);
  } else {
    constexpr int PER = 4;
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < pb.batch; b0 += 64 * PER) {
      int start[PER + 1], len[PER], tiles[PER];
      uint32_t sum = 0;  // (starts that overlap can make it pass 2^32; what comes out is looked at below)
#pragma unroll
      for (int k = 0; k <= PER; ++k) start[k] = min(max(pb.starts[min(b0 + PER * lane + k, pb.batch)], 0), pb.tokens);
#pragma unroll
      for (int k = 0; k < PER; ++k) len[k] = pb.len(min(b0 + PER * lane + k, pb.batch - 1));
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int n = min(max(0, start[k + 1] - start[k]), max_new);
        tiles[k] = n * G > above && n * G <= upto ? (n * G + rows - 1) / rows : 0;
        sum += (uint32_t)tiles[k];
      }
      uint32_t inc = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t u = __shfl_up(inc, o, 64);
        if (lane >= o) inc += u;
      }
      const int all = __builtin_amdgcn_readlane((int)inc, 63);
      if (at < all) {
        const int who = __ffsll((unsigned long long)__ballot((int)inc > at)) - 1;
        int rest = (int)((uint32_t)at - (inc - sum)), which = 0;  // in lane `who`: its sequence, and the tile there
        bool found = false;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          if (!found && rest < tiles[k]) {
            found = true;
            which = k;
            t.t0 = start[k];
            t.n = max(0, start[k + 1] - start[k]);
            t.len = len[k];
          }
          if (!found) rest = (int)((uint32_t)rest - (uint32_t)tiles[k]);
        }
        t.b = b0 + PER * who + __builtin_amdgcn_readlane(which, who);
        at = __builtin_amdgcn_readlane(rest, who);
        t.t0 = __builtin_amdgcn_readlane(t.t0, who);
        t.n = __builtin_amdgcn_readlane(t.n, who);
        t.len = __builtin_amdgcn_readlane(t.len, who);
        break;
      }
      at = (int)((uint32_t)at - (uint32_t)all);
    }
    if (t.b < 0) return t;
  }
  t.row0 = (int)((uint32_t)at * (uint32_t)rows);
  t.rows = min(t.n, max_new) * G;
  if (t.row0 < 0 || t.row0 >= t.rows) t.b = -1;  // (starts that overlap can claim more tiles than there are)
  return t;
}

// Keys that token j of the tile's sequence sees: those below the result (holes apart).
__device__ __forceinline__ int seen_by(const Tile& t, int j, int causal, int max_len) {
  return min(max_len, causal ? max(0, t.len - t.n + j + 1) : t.len);
}

// Partials of chunk s of packed row x of sequence b: its (token, head) pair's row in `part`, chunk s.
// O relative to m (not divided by l), then m (raw units) and l.
template <int D>
__device__ __forceinline__ float* part_o(float* part, int64_t row, int chunks, int s) {
  return part + (row * chunks + s) * D;
}
template <int D>
__device__ __forceinline__ float2* part_ml(float* part, int64_t all_rows, int chunks, int64_t row) {
  return reinterpret_cast<float2*>(part + all_rows * chunks * D) + row * chunks;
}
template <int D>
__device__ __forceinline__ const float2* part_ml(const float* part, int64_t all_rows, int chunks, int64_t row) {
  return reinterpret_cast<const float2*>(part + all_rows * chunks * D) + row * chunks;
}

// One call of kh_paged_attention.
struct PagedCall {
  const void *q, *k, *v;
  void* o;
  PagedBatch pb;
  int hq, hkv, G;
  PagedStrides st;
  float c2, sign;  // |scale| log2 e, and the scale's sign, which goes to the queries; scale 0: 1 and queries of 0
  int causal, max_new;
};

// Workgroup columns that cover every tile of `rows` packed rows of the sequences that have more than `above` and at
// most `upto` of them: a sequence's last tile may be part of one.
inline int64_t tiles_of(const PagedCall& c, int rows, int above = 0, int upto = INT32_MAX) {
  const int64_t most = (int64_t)c.max_new * c.G < upto ? (int64_t)c.max_new * c.G : upto, all = (int64_t)c.pb.tokens * c.G;
  const int64_t batch = c.pb.batch < all / (above + 1) ? c.pb.batch : all / (above + 1);
  const int64_t per = (most + rows - 1) / rows;
  return c.pb.starts == nullptr || per * batch < all / rows + batch ? per * batch : all / rows + batch;
}

// How a launch form covers its sequences: workgroups for `columns` (tiles x kv heads) by `used` chunks of `chunk` keys.
struct PagedPart {
  int columns, chunk, used;
};

// paged_tiles.hip, bfloat16, d 64 or 128: every sequence in tiles of 32 `waves` (4 or 8) packed rows; or sequences of more
// than few_rows of them in tiles of 128, the others in tiles of 32.  Chunks are multiples of 128 keys, with
// partials in part [rows, chunks] where a form uses more than one.
void launch_paged_tiles(const PagedCall& c, int d, int waves, const PagedPart& many, int chunks, float* part);
void launch_paged_mixed(const PagedCall& c, int d, int few_rows, const PagedPart& many, const PagedPart& few, int chunks,
                        float* part);

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
