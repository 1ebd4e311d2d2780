// The paged KV cache beside its attention: rows into pages (kh_paged_kv_write) and the bookkeeping of
// the pages (kh_pages_fork, kh_pages_reserve, kh_pages_compact, kh_pages_copy).
//
// The bookkeeping stays on the device, so that a captured step replays it: a page is free while its
// reference count is 0, and new pages are the lowest free ones in row order, which makes every result a
// function of the arguments alone (the counts are changed by integer atomics, whose order does not
// matter).  These kernels are short: each is bound by its chain of dependent loads and scans.
#include "paged.h"

using namespace kh;

namespace {

// ---- rows into pages -------------------------------------------------------------------------
struct WriteStrides {
  int64_t kt, kh, vt, vh, kp, kph, kpr, vp, vph, vpr;
};

// A workgroup takes one token: its threads copy the heads' K and V rows in pieces of E.  info (may be null): what
// pages_reserve left; where that changed nothing, the new tokens' rows are other rows' places.  6600 bf16 tokens of 8
// heads of 128: 11 us, 4.9 TB/s read and written, what a large copy reaches; one token of eight sequences: 2.8 us.
template <typename E>
__global__ __launch_bounds__(256) void paged_write_kernel(const E* __restrict__ K, const E* __restrict__ V,
                                                          E* __restrict__ KP, E* __restrict__ VP, PagedBatch pb, int hkv,
                                                          int pieces, WriteStrides st, const int32_t* __restrict__ info) {
  const int t = blockIdx.x;
  const bool lacking = info && (info[1] != 0 || info[2] != 0);
  const int b = pb.sequence_of(t);
  if (b < 0) return;
  const int pos = pb.len(b) - pb.count(b) + t - pb.first(b);
  if (pos < 0 || pos >= pb.max_len) return;
  const int id = pb.table[b * pb.table_stride + (pos >> pb.page_log)];
  if (lacking || !pb.is_page(id)) return;
  const int slot = pos & ((1 << pb.page_log) - 1);
  for (int i = threadIdx.x; i < hkv * pieces; i += 256) {
    const int h = i / pieces, c = i - h * pieces;
    KP[id * st.kp + h * st.kph + slot * st.kpr + c] = K[t * st.kt + h * st.kh + c];
    VP[id * st.vp + h * st.vph + slot * st.vpr + c] = V[t * st.vt + h * st.vh + c];
  }
}

// ---- fork -------------------------------------------------------------------------------------
// table'[s] = table[parents[s]], lens' likewise, counts' = counts (a parent outside [0, rows): an empty row).
__global__ __launch_bounds__(256) void pages_fork_kernel(const int32_t* __restrict__ table, int64_t stride,
                                                         const int32_t* __restrict__ lens,
                                                         const int32_t* __restrict__ refs,
                                                         const int32_t* __restrict__ parents, int rows, int width,
                                                         int num_pages, int32_t* __restrict__ new_table,
                                                         int32_t* __restrict__ new_lens, int32_t* __restrict__ new_refs) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows * width; i += step) {
    const int s = (int)(i / width), c = (int)(i - (int64_t)s * width), p = parents[s];
    new_table[i] = (unsigned)p < (unsigned)rows ? table[p * stride + c] : -1;
  }
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < num_pages; i += step) new_refs[i] = refs[i];
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows; i += step) {
    const int p = parents[i];
    new_lens[i] = (unsigned)p < (unsigned)rows ? lens[p] : 0;
  }
}

// counts'[page] += children(row) - 1 for every entry of every old row; a workgroup per row.
__global__ __launch_bounds__(256) void pages_fork_refs_kernel(const int32_t* __restrict__ table, int64_t stride,
                                                              const int32_t* __restrict__ parents, int rows, int width,
                                                              int num_pages, int32_t* __restrict__ new_refs) {
  __shared__ int children[4];
  const int s = blockIdx.x;
  int n = 0;
  for (int i = threadIdx.x; i < rows; i += 256) n += parents[i] == s;
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if ((threadIdx.x & 63) == 0) children[threadIdx.x >> 6] = n;
  __syncthreads();
  const int delta = children[0] + children[1] + children[2] + children[3] - 1;
  if (delta == 0) return;
  for (int c = threadIdx.x; c < width; c += 256) {
    const int id = table[s * stride + c];
    if ((unsigned)id < (unsigned)num_pages) atomicAdd(new_refs + id, delta);
  }
}

// Both at once for small tables, by one workgroup with the counts' changes in LDS: a beam step's 64 rows of 70 pages
// take 4.8 us instead of 2.7 + 2.6 and the gap between two launches; 256 rows of 64 would take 11.
constexpr int kForkPages = 16384, kForkRows = 2048, kForkEntries = 8192;
__global__ __launch_bounds__(1024) void pages_fork_small_kernel(const int32_t* __restrict__ table, int64_t stride,
                                                                const int32_t* __restrict__ lens,
                                                                const int32_t* __restrict__ refs,
                                                                const int32_t* __restrict__ parents, int rows, int width,
                                                                int num_pages, int32_t* __restrict__ new_table,
                                                                int32_t* __restrict__ new_lens,
                                                                int32_t* __restrict__ new_refs) {
  __shared__ int change[kForkPages];
  __shared__ int children[kForkRows];
  for (int i = threadIdx.x; i < num_pages; i += 1024) change[i] = 0;
  for (int i = threadIdx.x; i < rows; i += 1024) children[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const int p = parents[i];
    const bool has = (unsigned)p < (unsigned)rows;
    if (has) atomicAdd(children + p, 1);
    new_lens[i] = has ? lens[p] : 0;
  }
  __syncthreads();
#pragma unroll 4
  for (int i = threadIdx.x; i < rows * width; i += 1024) {
    const int s = i / width, c = i - s * width, p = parents[s], delta = children[s] - 1;
    const int mine = table[s * stride + c];
    new_table[i] = (unsigned)p < (unsigned)rows ? table[p * stride + c] : -1;
    if (delta != 0 && (unsigned)mine < (unsigned)num_pages) atomicAdd(change + mine, delta);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < num_pages; i += 1024) new_refs[i] = refs[i] + change[i];
}

// ---- reserve ----------------------------------------------------------------------------------
constexpr int kOne = 1024;      // threads of the one-workgroup kernels
constexpr int kMaxRows = 2048;  // rows that kh_pages_reserve's LDS holds

// Exclusive prefix sum over the workgroup's threads in thread order; *total receives the sum.
__device__ __forceinline__ int block_scan(int v, int* waves, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(inc, o, 64);
    if (lane >= o) inc += u;
  }
  __syncthreads();  // the previous use of `waves` is over
  if (lane == 63) waves[w] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kOne / 64; ++i) {
    if (i < w) before += waves[i];
    all += waves[i];
  }
  *total = all;
  return before + inc - v;
}

// The same for two flags at once: the number of threads before this one that have them.
__device__ __forceinline__ int2 block_places(bool a, bool b, int2* waves, int2* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t ma = __ballot(a), mb = __ballot(b), below = (1ull << lane) - 1;
  __syncthreads();  // the previous use of `waves` is over
  if (lane == 0) waves[w] = make_int2(__popcll(ma), __popcll(mb));
  __syncthreads();
  int2 before = make_int2(__popcll(ma & below), __popcll(mb & below)), all = make_int2(0, 0);
#pragma unroll
  for (int i = 0; i < kOne / 64; ++i) {
    const int2 n = waves[i];
    if (i < w) {
      before.x += n.x;
      before.y += n.y;
    }
    all.x += n.x;
    all.y += n.y;
  }
  *total = all;
  return before;
}

// One workgroup.  A row that grows from len to len + count takes a new page for every table entry behind
// its last page.  Of the rows that grow on one partly filled page, each gets a copy of it, also a new page, as long as
// another row holds it, too: row after row, while the count less the copies before is above 1.  Nothing changes
// unless all rows can grow.  64 rows that share tails in a pool of 685 pages: 6 us, a chain of four loads and three
// scans; the free pages among the first kKept * 1024 keep their places from the count, which has to come first, to
// the writes.  The pool is walked from its front, 1024 counts a step, and what lies behind the first kKept * 1024 twice:
// where the free pages are the last ones 5.7 us with 4000 pages, 9.5 with 20000 and 105 with 100000.
constexpr int kKept = 4;
__global__ __launch_bounds__(kOne) void pages_reserve_kernel(int32_t* __restrict__ table, int64_t stride,
                                                             int32_t* __restrict__ lens, int32_t* __restrict__ refs,
                                                             const int32_t* __restrict__ counts, int rows, int width,
                                                             int num_pages, int page_log, int32_t* __restrict__ moves,
                                                             int32_t* __restrict__ info) {
  __shared__ int tail[kMaxRows];    // the shared page of a partly filled tail that grows; then: the page to copy; or -1
  __shared__ int first[kMaxRows];   // the first table entry that gets a new page
  __shared__ int before[kMaxRows];  // new pages of the rows before this one
  __shared__ int number[kMaxRows];  // copies of the rows before this one
  __shared__ int waves[kOne / 64];
  __shared__ int2 flags[kOne / 64];
  constexpr int PER = kMaxRows / kOne;
  const int64_t page = int64_t(1) << page_log;
  int held[PER], grows[PER];  // this thread's rows: holders of the tail page, new rows
  bool bad[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = i * kOne + threadIdx.x;
    held[i] = 0;
    grows[i] = 0;
    bad[i] = false;
    if (s >= rows) continue;
    const int64_t len = max(lens[s], 0), end = len + max(counts[s], 0);
    int t = -1, f = -1;  // -1: the row does not grow
    if (end > len && end > width * page) {
      bad[i] = true;
    } else if (end > len) {
      f = (int)((len + page - 1) >> page_log);
      grows[i] = (int)((end + page - 1) >> page_log) - f;
      if (len & (page - 1)) {
        t = table[s * stride + (len >> page_log)];
        if ((unsigned)t >= (unsigned)num_pages) {
          t = -1;
          --f;  // no page in the tail's place: a new one, with nothing to copy
          ++grows[i];
        } else {
          held[i] = refs[t];
          if (held[i] <= 1) t = -1;
        }
      }
    }
    tail[s] = t;
    first[s] = f;
    moves[2 * s] = moves[2 * s + 1] = -1;
  }
  __syncthreads();
  int needed = 0, copied = 0, too_long = 0;
  bool mine[PER];  // whether this thread's rows copy their tail
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    mine[i] = false;
    if (i * kOne >= rows) break;
    const int s = i * kOne + threadIdx.x;
    const int t = s < rows ? tail[s] : -1;
    if (t >= 0) {
      int sharers = 0;  // before this row
#pragma unroll 8
      for (int r = 0; r < s; ++r) sharers += tail[r] == t;
      mine[i] = held[i] - sharers > 1;
    }
    int total = 0;
    int2 sums;
    const int b = block_scan(grows[i] + mine[i], waves, &total), m = block_places(mine[i], bad[i], flags, &sums).x;
    if (s < rows) {
      before[s] = needed + b;
      number[s] = copied + m;
    }
    needed += total;
    copied += sums.x;
    too_long += sums.y;
  }
  __syncthreads();  // every row has read the others' tails
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = i * kOne + threadIdx.x;
    if (s < rows) {
      if (mine[i])
        --first[s];
      else
        tail[s] = -1;
    }
  }
  // the r-th lowest free page goes to the row whose new pages r lies among
  auto give = [&](int p, int r) {
    int lo = 0, hi = rows;  // the last row with before[row] <= r (rows without new pages share the next one's)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= r)
        lo = mid;
      else
        hi = mid;
    }
    const int at = r - before[lo];
    table[lo * stride + first[lo] + at] = p;
    refs[p] = 1;
    if (at == 0 && tail[lo] >= 0) {
      moves[2 * number[lo]] = tail[lo];
      moves[2 * number[lo] + 1] = p;
    }
  };
  // the free pages, counted up to the number needed; place[i]: this thread's i-th page among them
  int found = 0, kept = 0, place[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    place[i] = -1;
    const int64_t p0 = (int64_t)i * kOne, p = p0 + threadIdx.x;
    if (p0 >= num_pages || found >= needed) continue;  // (the same for every thread)
    const bool free = p < num_pages && refs[p] <= 0;
    int2 n;
    const int r = found + block_places(free, false, flags, &n).x;
    if (free && r < needed) place[i] = r;
    found += n.x;
  }
  kept = found;
  for (int64_t p0 = (int64_t)kKept * kOne; p0 < num_pages && found < needed; p0 += kOne) {
    const int64_t p = p0 + threadIdx.x;
    int2 n;
    block_places(p < num_pages && refs[p] <= 0, false, flags, &n);
    found += n.x;
  }
  const bool ok = found >= needed && too_long == 0;
  if (threadIdx.x == 0) {
    info[0] = ok ? copied : 0;
    info[1] = found < needed ? needed - found : 0;
    info[2] = too_long;
  }
  if (!ok) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (place[i] >= 0) give(i * kOne + threadIdx.x, place[i]);
  found = kept;
  for (int64_t p0 = (int64_t)kKept * kOne; p0 < num_pages && found < needed; p0 += kOne) {
    const int64_t p = p0 + threadIdx.x;
    const bool free = p < num_pages && refs[p] <= 0;
    int2 n;
    const int r = found + block_places(free, false, flags, &n).x;
    found += n.x;
    if (free && r < needed) give((int)p, r);
  }
  __syncthreads();
  for (int s = threadIdx.x; s < rows; s += kOne) {
    if (tail[s] >= 0) atomicSub(refs + tail[s], 1);
    if (first[s] >= 0) lens[s] = max(lens[s], 0) + counts[s];
  }
}

// ---- compact ----------------------------------------------------------------------------------
// One workgroup: with n live pages, the i-th live page at or behind n moves to the i-th free page before n.
// to[page]: where a page is afterwards.  4000 pages: 7.0 us (two passes over the counts), and 4.6 for the table; 100000: 90 both.
__global__ __launch_bounds__(kOne) void pages_compact_kernel(const int32_t* __restrict__ refs, int num_pages,
                                                             int32_t* __restrict__ new_refs, int32_t* __restrict__ to,
                                                             int32_t* __restrict__ moves, int max_moves,
                                                             int32_t* __restrict__ info) {
  __shared__ int waves[kOne / 64];
  __shared__ int2 flags[kOne / 64];
  int mine = 0, live = 0;
  for (int64_t p = threadIdx.x; p < num_pages; p += kOne) mine += refs[p] > 0;
  block_scan(mine, waves, &live);
  int src = 0, dst = 0;
  for (int64_t p0 = 0; p0 < num_pages; p0 += kOne) {
    const int64_t p = p0 + threadIdx.x;
    const int ref = p < num_pages ? refs[p] : 0;
    const bool leaves = ref > 0 && p >= live, takes = p < num_pages && ref <= 0 && p < live;
    int2 n;
    const int2 at = block_places(leaves, takes, flags, &n);
    if (leaves) moves[2 * (src + at.x)] = (int)p;
    if (takes) moves[2 * (dst + at.y) + 1] = (int)p;
    if (p < num_pages) {
      new_refs[p] = leaves ? 0 : ref;
      to[p] = (int)p;
    }
    src += n.x;
    dst += n.y;
  }
  if (threadIdx.x == 0) {
    info[0] = src;
    info[1] = live;
  }
  __threadfence_block();
  __syncthreads();
  for (int i = threadIdx.x; i < max_moves; i += kOne) {
    if (i < src) {
      const int a = moves[2 * i], b = moves[2 * i + 1];
      to[a] = b;
      new_refs[b] = refs[a];
    } else {
      moves[2 * i] = moves[2 * i + 1] = -1;
    }
  }
}

__global__ __launch_bounds__(256) void pages_rename_kernel(const int32_t* __restrict__ table, int64_t stride, int rows,
                                                           int width, int num_pages, const int32_t* __restrict__ to,
                                                           int32_t* __restrict__ new_table) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)rows * width; i += step) {
    const int64_t s = i / width;
    const int id = table[s * stride + (i - s * width)];
    new_table[i] = (unsigned)id < (unsigned)num_pages ? to[id] : id;
  }
}

// ---- copy -------------------------------------------------------------------------------------
// A workgroup copies pieces of 16 KiB: piece i of move m of plane l, in the order (move, plane, piece).  A beam step's
// 12 MB, which the step reads again, in 5.6 us.  From kStream bytes on the loads and stores pass the caches by: 247 MB in
// 96 us = 5.1 TB/s read and written instead of 103, and the beam step's would take 7.4.
constexpr int kPiece = 16384;
constexpr int64_t kStream = int64_t(64) << 20;
template <bool STREAM>
__device__ __forceinline__ void copy_pieces(uint8_t* __restrict__ pages, int64_t plane_bytes, int64_t page_bytes,
                                            int num_pages, const int32_t* __restrict__ moves, int64_t planes, int64_t pieces,
                                            int64_t items) {
  typedef uint32_t v4u32 __attribute__((ext_vector_type(4)));
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const int64_t m = i / (planes * pieces), rest = i - m * planes * pieces, l = rest / pieces;
    const int64_t at = (rest - l * pieces) * kPiece;
    const int a = moves[2 * m], b = moves[2 * m + 1];
    if ((unsigned)a >= (unsigned)num_pages || (unsigned)b >= (unsigned)num_pages || a == b) continue;
    const uint8_t* from = pages + l * plane_bytes + a * page_bytes + at;
    uint8_t* into = pages + l * plane_bytes + b * page_bytes + at;
    const int64_t left = page_bytes - at;
#pragma unroll
    for (int j = 0; j < kPiece / 4096; ++j) {
      const int64_t o = j * 4096 + threadIdx.x * 16;
      if (o >= left) continue;
      const v4u32* x = reinterpret_cast<const v4u32*>(from + o);
      v4u32* y = reinterpret_cast<v4u32*>(into + o);
      if constexpr (STREAM)
        __builtin_nontemporal_store(__builtin_nontemporal_load(x), y);
      else
        *y = *x;
    }
  }
}
__global__ __launch_bounds__(256) void pages_copy_kernel(uint8_t* __restrict__ pages, int64_t planes, int64_t plane_bytes,
                                                         int64_t page_bytes, int num_pages,
                                                         const int32_t* __restrict__ moves, int max_moves,
                                                         const int32_t* __restrict__ info) {
  const int64_t pieces = (page_bytes + kPiece - 1) / kPiece, count = min(max(info[0], 0), max_moves);
  const int64_t items = count * planes * pieces;
  if (count * planes * page_bytes >= kStream)
    copy_pieces<true>(pages, plane_bytes, page_bytes, num_pages, moves, planes, pieces, items);
  else
    copy_pieces<false>(pages, plane_bytes, page_bytes, num_pages, moves, planes, pieces, items);
}

template <typename E>
void launch_write(const void* k, const void* v, void* kp, void* vp, const PagedBatch& pb, int hkv, int d, int per,
                  const int64_t* s, const int32_t* info) {
  WriteStrides st{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9]};
  int64_t* f = &st.kt;
  for (int i = 0; i < 10; ++i) f[i] /= per;
  paged_write_kernel<E><<<pb.tokens, 256, 0, stream()>>>((const E*)k, (const E*)v, (E*)kp, (E*)vp, pb, hkv, d / per, st,
                                                       info);
}

bool rows_ok(int64_t rows, int64_t width, int64_t stride, int64_t num_pages) {
  return rows >= 0 && rows <= 65535 && width >= 0 && width <= INT32_MAX && stride >= width && num_pages >= 0 &&
         num_pages <= INT32_MAX;
}

unsigned blocks_for(int64_t n) {
  const int64_t b = (n + 255) / 256, most = 8 * (int64_t)cu_count();
  return (unsigned)(b < 1 ? 1 : (b < most ? b : most));
}

}  // namespace

extern "C" {

int kh_paged_kv_write(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* page_table,
                      const int32_t* kv_lens, const int32_t* query_starts, int64_t tokens, int64_t batch, int hkv, int d,
                      int64_t num_pages, int64_t page_size, int64_t table_width, int64_t table_stride,
                      const int64_t* strides, int dtype) {
  return kh_paged_kv_write_reserved(k, v, k_pages, v_pages, page_table, kv_lens, query_starts, tokens, batch, hkv, d, num_pages,
                                    page_size, table_width, table_stride, strides, nullptr, dtype);
}

int kh_paged_kv_write_reserved(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* page_table,
                               const int32_t* kv_lens, const int32_t* query_starts, int64_t tokens, int64_t batch, int hkv,
                               int d, int64_t num_pages, int64_t page_size, int64_t table_width, int64_t table_stride,
                               const int64_t* strides, const int32_t* info, int dtype) {
  KH_REQUIRE_INIT();
  KH_REQUIRE(hkv > 0 && d > 0 && (int64_t)hkv * d <= INT32_MAX, "kh_paged_kv_write: bad extents (%d heads of %d)", hkv, d);
  KH_REQUIRE(dtype == KH_BF16 || dtype == KH_F32, "kh_paged_kv_write: unsupported dtype %d", dtype);
  PagedBatch pb;
  const int rc = paged_batch("kh_paged_kv_write", page_table, kv_lens, query_starts, tokens, batch, num_pages, page_size,
                             table_width, table_stride, INT64_MAX, &pb);
  if (rc != KH_OK) return rc;
  if (tokens == 0 || batch == 0 || num_pages == 0 || table_width == 0) return KH_OK;
  KH_REQUIRE(k && v && k_pages && v_pages && page_table && kv_lens && strides, "kh_paged_kv_write: null pointer");
  const int64_t size = dtype == KH_BF16 ? 2 : 4;
  const int per = (int)(16 / size);
  auto rows = [&](const void* at, const int64_t* s) { return Span(at, size * d, tokens, size * s[0], hkv, size * s[1]); };
  auto pool = [&](const void* at, const int64_t* s) {
    return Span(at, size * d, num_pages, size * s[0], hkv, size * s[1], page_size, size * s[2]);
  };
  const Span keys = rows(k, strides), values = rows(v, strides + 2), kp = pool(k_pages, strides + 4), vp = pool(v_pages, strides + 7),
             table = table_span(page_table, table_stride, batch, table_width), lens = ints(kv_lens, batch),
             starts = ints(query_starts, batch + 1), left = ints(info, 3);
  // (one pool may be keys and values at once where one tensor is, too)
  bool one = k == v && k_pages == v_pages && strides[0] == strides[2] && strides[1] == strides[3];
  for (int i = 0; i < 3; ++i) one = one && strides[4 + i] == strides[7 + i];
  KH_REQUIRE(!overlap({kp}, {keys, values, table, lens, starts, left}) && !overlap({vp}, {keys, values, table, lens, starts, left}) &&
                 (one || apart(kp, vp)),
             "kh_paged_kv_write: the pages must not share memory with the inputs or each other");
  bool wide = d % per == 0 && aligned16(k) && aligned16(v) && aligned16(k_pages) && aligned16(v_pages);
  for (int i = 0; i < 10; ++i) wide = wide && strides[i] % per == 0;
  if (wide)
    launch_write<uint4>(k, v, k_pages, v_pages, pb, hkv, d, per, strides, info);
  else if (dtype == KH_BF16)
    launch_write<uint16_t>(k, v, k_pages, v_pages, pb, hkv, d, 1, strides, info);
  else
    launch_write<uint32_t>(k, v, k_pages, v_pages, pb, hkv, d, 1, strides, info);
  KH_CHECK_LAUNCH();
  return KH_OK;
}

int kh_pages_fork(const int32_t* page_table, int64_t table_stride, const int32_t* kv_lens, const int32_t* page_refs,
                  const int32_t* parents, int64_t rows, int64_t table_width, int64_t num_pages, int32_t* new_table,
                  int32_t* new_lens, int32_t* new_refs) {
  KH_REQUIRE_INIT();
  KH_REQUIRE(rows_ok(rows, table_width, table_stride, num_pages), "kh_pages_fork: bad extents");
  KH_REQUIRE((rows == 0 || (kv_lens && parents && new_lens)) && (rows == 0 || table_width == 0 || (page_table && new_table)) &&
                 (num_pages == 0 || (page_refs && new_refs)),
             "kh_pages_fork: null pointer");
  KH_REQUIRE(!overlap({ints(new_table, rows * table_width), ints(new_lens, rows), ints(new_refs, num_pages)},
                      {table_span(page_table, table_stride, rows, table_width), ints(kv_lens, rows), ints(page_refs, num_pages),
                       ints(parents, rows)}),
             "kh_pages_fork: the results must not share memory with the inputs or each other");
  if (rows == 0 && num_pages == 0) return KH_OK;
  if (num_pages <= kForkPages && rows <= kForkRows && rows * table_width <= kForkEntries) {
    pages_fork_small_kernel<<<1, 1024, 0, stream()>>>(page_table, table_stride, kv_lens, page_refs, parents, (int)rows,
                                                      (int)table_width, (int)num_pages, new_table, new_lens, new_refs);
    KH_CHECK_LAUNCH();
    return KH_OK;
  }
  int64_t n = rows * table_width;
  if (n < num_pages) n = num_pages;
  pages_fork_kernel<<<blocks_for(n), 256, 0, stream()>>>(page_table, table_stride, kv_lens, page_refs, parents, (int)rows,
                                                         (int)table_width, (int)num_pages, new_table, new_lens, new_refs);
  KH_CHECK_LAUNCH();
  if (rows > 0 && table_width > 0 && num_pages > 0) {
    pages_fork_refs_kernel<<<(unsigned)rows, 256, 0, stream()>>>(page_table, table_stride, parents, (int)rows,
                                                                 (int)table_width, (int)num_pages, new_refs);
    KH_CHECK_LAUNCH();
  }
  return KH_OK;
}

int kh_pages_reserve(int32_t* page_table, int64_t table_stride, int32_t* kv_lens, int32_t* page_refs,
                     const int32_t* counts, int64_t rows, int64_t table_width, int64_t num_pages, int64_t page_size,
                     int32_t* moves, int32_t* info) {
  KH_REQUIRE_INIT();
  KH_REQUIRE(rows_ok(rows, table_width, table_stride, num_pages), "kh_pages_reserve: bad extents");
  KH_REQUIRE(rows <= kMaxRows, "kh_pages_reserve: %lld rows, at most %d", (long long)rows, kMaxRows);
  KH_REQUIRE(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
             "kh_pages_reserve: page size %lld is not a power of two from 16 to 4096", (long long)page_size);
  // (the pages that a call may need are counted in 32 bits)
  KH_REQUIRE(table_width <= (1 << 30) && table_width * page_size <= (1 << 30) && rows * table_width <= INT32_MAX,
             "kh_pages_reserve: the page table passes 2^30 rows, or 2^31 entries");
  KH_REQUIRE(info && (rows == 0 || (kv_lens && counts && moves)) && (rows == 0 || table_width == 0 || page_table) &&
                 (num_pages == 0 || page_refs),
             "kh_pages_reserve: null pointer");
  KH_REQUIRE(!overlap({table_span(page_table, table_stride, rows, table_width), ints(kv_lens, rows), ints(page_refs, num_pages),
                       ints(moves, 2 * rows), ints(info, 3)},
                      {ints(counts, rows)}),
             "kh_pages_reserve: the operands must not share memory with each other");
  pages_reserve_kernel<<<1, kOne, 0, stream()>>>(page_table, table_stride, kv_lens, page_refs, counts, (int)rows,
                                                 (int)table_width, (int)num_pages, log2_of(page_size), moves, info);
  KH_CHECK_LAUNCH();
  return KH_OK;
}

int kh_pages_compact(const int32_t* page_table, int64_t table_stride, const int32_t* page_refs, int64_t rows,
                     int64_t table_width, int64_t num_pages, int32_t* new_table, int32_t* new_refs, int32_t* moves,
                     int64_t max_moves, int32_t* info) {
  KH_REQUIRE_INIT();
  KH_REQUIRE(rows_ok(rows, table_width, table_stride, num_pages), "kh_pages_compact: bad extents");
  KH_REQUIRE(max_moves >= num_pages / 2 && max_moves <= INT32_MAX, "kh_pages_compact: room for %lld moves, %lld pages may need %lld",
             (long long)max_moves, (long long)num_pages, (long long)(num_pages / 2));
  KH_REQUIRE(info && (max_moves == 0 || moves) && (num_pages == 0 || (page_refs && new_refs)) &&
                 (rows == 0 || table_width == 0 || (page_table && new_table)),
             "kh_pages_compact: null pointer");
  KH_REQUIRE(!overlap({ints(new_table, rows * table_width), ints(new_refs, num_pages), ints(moves, 2 * max_moves), ints(info, 2)},
                      {table_span(page_table, table_stride, rows, table_width), ints(page_refs, num_pages)}),
             "kh_pages_compact: the results must not share memory with the inputs or each other");
  int32_t* to = nullptr;
  if (num_pages > 0) {
    to = (int32_t*)scratch_alloc((size_t)num_pages * 4);
    if (to == nullptr) return KH_ERR_OOM;
  }
  pages_compact_kernel<<<1, kOne, 0, stream()>>>(page_refs, (int)num_pages, new_refs, to, moves, (int)max_moves, info);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && rows > 0 && table_width > 0) {
    pages_rename_kernel<<<blocks_for(rows * table_width), 256, 0, stream()>>>(page_table, table_stride, (int)rows,
                                                                              (int)table_width, (int)num_pages, to, new_table);
    e = hipGetLastError();
  }
  if (to) scratch_free(to);
  if (e != hipSuccess) {
    set_error("kh_pages_compact: launch failed: %s", hipGetErrorString(e));
    return KH_ERR_HIP;
  }
  KH_DEBUG_SYNC();
  return KH_OK;
}

int kh_pages_copy(void* pages, int64_t planes, int64_t num_pages, int64_t page_bytes, const int32_t* moves,
                  int64_t max_moves, const int32_t* info) {
  KH_REQUIRE_INIT();
  KH_REQUIRE(planes >= 0 && num_pages >= 0 && num_pages <= INT32_MAX && page_bytes >= 0 && page_bytes <= INT32_MAX &&
                 max_moves >= 0 && max_moves <= INT32_MAX,
             "kh_pages_copy: bad extents");
  KH_REQUIRE(page_bytes % 16 == 0 && aligned16(pages), "kh_pages_copy: pages must be 16-byte aligned, of a multiple of 16 bytes");
  if (planes == 0 || num_pages == 0 || page_bytes == 0 || max_moves == 0) return KH_OK;
  KH_REQUIRE(pages && moves && info, "kh_pages_copy: null pointer");
  KH_REQUIRE(!overlap({Span(pages, page_bytes, num_pages, page_bytes, planes, num_pages * page_bytes)},
                      {ints(moves, 2 * max_moves), ints(info, 1)}),
             "kh_pages_copy: the pages must not share memory with the moves");
  const int64_t items = max_moves * planes * ((page_bytes + kPiece - 1) / kPiece), most = 8 * (int64_t)cu_count();
  pages_copy_kernel<<<(unsigned)(items < most ? items : most), 256, 0, stream()>>>(
      (uint8_t*)pages, planes, num_pages * page_bytes, page_bytes, (int)num_pages, moves, (int)max_moves, info);
  KH_CHECK_LAUNCH();
  return KH_OK;
}

}  // extern "C"
