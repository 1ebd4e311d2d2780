// Attention of new tokens over a paged KV cache (kh_paged_attention).
//
// With n new tokens of L cached rows, token j of a sequence sees the rows p <= L - n + j (causal) or p < L
// that lie in a page of the pool:  o = sum_p softmax_p(scale q . k_p) v_p.
//
// The query rows of one kv head are packed: packed row x = token * G + g holds query head hk * G + g of the
// token (G = hq / hkv), so the G heads that read a kv head share every K and V row that is loaded, and one
// token of G heads is as good a tile as G tokens.
//
// Work is split over tiles of packed rows and over chunks of `chunk` keys; where a tile's keys make more
// than one chunk, each chunk leaves (O, m, l) partials and paged_merge_kernel joins them in chunk order, so
// a result does not depend on timing.
#include <cmath>

#include "paged_rows.h"

using namespace kh;

namespace {

template <typename T, int D, int RT>
__global__ __launch_bounds__(kRowWaves * 64, sizeof(T) == 4 && D == 128 ? 1 : 2) void paged_rows_kernel(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, T* __restrict__ O, PagedBatch pb, int hq,
    int hkv, int G, PagedStrides st, float c2, float sign, int causal, int max_new, int most_rows, int chunk, int chunks,
    float* __restrict__ part) {
  __shared__ float join[RowLds<T, D, RT>::FLOATS];
  paged_rows<T, D, RT>(join, blockIdx.x, blockIdx.z, Q, K, V, O, pb, hq, hkv, G, st, c2, sign, causal, max_new, most_rows,
                       chunk, chunks, part);
}

// Joins the chunks of a token's query heads, relative to each row's maximum.  Chunks hold few_chunk keys in sequences
// of at most most_rows packed rows and many_chunk in others (0: these have none to join).
// Where a row lies and how many chunks it has: of them 0, nothing to do.
struct MergeArgs {
  int hq, causal, max_new, G, most_rows, few_chunk, many_chunk, chunks;
};
__device__ __forceinline__ int chunks_of(const PagedBatch& pb, const MergeArgs& a, int tok, bool* stored) {
  Tile t;
  t.b = pb.sequence_of(tok);
  *stored = false;
  if (t.b < 0) return 0;
  t.n = pb.count(t.b);
  t.len = pb.len(t.b);
  const int j = tok - pb.first(t.b), chunk = min(t.n, a.max_new) * a.G <= a.most_rows ? a.few_chunk : a.many_chunk;
  if (j >= a.max_new || chunk == 0) return 0;
  *stored = true;
  const int seen = seen_by(t, j, a.causal, pb.max_len);
  return min(a.chunks, (seen + chunk - 1) / chunk);
}
__device__ __forceinline__ float weight_of(float2 ml, float m, float c2) {
  return ml.x == -INFINITY && ml.y == 0.f ? 0.f : fast_exp2((ml.x - m) * c2);
}

// Many rows (at least as many tokens as CUs: 2048 tokens of 16 heads in two chunks 9 us, bound by the partials' reads):
// a workgroup per token, D / 4 lanes per row (query head), so that the token's place is looked up once
// and several rows' loads are in flight.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(const float* __restrict__ part, T* __restrict__ O, PagedBatch pb,
                                                          PagedStrides st, float c2, MergeArgs a) {
  constexpr int LPR = D / 4, ROWS = 256 / LPR;
  const int tok = blockIdx.x, lane = threadIdx.x % LPR;
  bool stored;
  const int ns = chunks_of(pb, a, tok, &stored);
  if (!stored) return;
  const int64_t all = (int64_t)pb.tokens * a.hq;
  for (int h = threadIdx.x / LPR; h < a.hq; h += ROWS) {
    const int64_t row = (int64_t)tok * a.hq + h;
    const float2* ml = part_ml<D>(part, all, a.chunks, row);
    const float* po = part + row * a.chunks * D + 4 * lane;
    float m = -INFINITY, l = 0.f;
    for (int s = 0; s < ns; ++s) m = fmaxf(m, ml[s].x);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int s = 0; s < ns; ++s) {
      const float2 u = ml[s];
      const float w = weight_of(u, m, c2);
      l += w * u.y;
      o += *reinterpret_cast<const f32x4*>(po + (int64_t)s * D) * w;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    T* to = O + (int64_t)tok * st.ot + (int64_t)h * st.oh + 4 * lane;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
    else
      *reinterpret_cast<f32x4*>(to) = o * inv;
  }
}

// Few rows (latency: 3.7 to 4.8 us): a workgroup per (token, query head); wave w sums chunks w, w + 4, ..., several
// loads in flight, and the four sums are added in wave order.
constexpr int kMergeWaves = 4;
template <typename T, int D>
__global__ __launch_bounds__(kMergeWaves * 64) void paged_merge_row_kernel(const float* __restrict__ part,
                                                                           T* __restrict__ O, PagedBatch pb,
                                                                           PagedStrides st, float c2, MergeArgs a) {
  constexpr int E = D / 64;
  __shared__ float join[kMergeWaves - 1][64][E + 1];
  const int tok = blockIdx.x / a.hq, h = blockIdx.x - tok * a.hq, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t row = (int64_t)tok * a.hq + h;
  bool stored;
  const int ns = chunks_of(pb, a, tok, &stored);
  if (!stored) return;
  const float2* ml = part_ml<D>(part, (int64_t)pb.tokens * a.hq, a.chunks, row);
  const float* po = part + row * a.chunks * D + E * lane;
  float m = -INFINITY;
  for (int s = lane; s < ns; s += 64) m = fmaxf(m, ml[s].x);
  m = wave_max(m);
  float o[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int s = w; s < ns; s += kMergeWaves) {
    const float2 u = ml[s];
    const float f = weight_of(u, m, c2);
    l += f * u.y;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += f * po[(int64_t)s * D + e];
  }
  if (w > 0) {
    join[w - 1][lane][E] = l;
#pragma unroll
    for (int e = 0; e < E; ++e) join[w - 1][lane][e] = o[e];
  }
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int i = 0; i < kMergeWaves - 1; ++i) {
    l += join[i][lane][E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += join[i][lane][e];
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) Elem<T>::store(O + (int64_t)tok * st.ot + (int64_t)h * st.oh, E * lane + e, o[e] * inv);
}

// A part of a launch of `tiles` tiles per kv head, of which `there` hold rows as far as can be told here: its keys in as
// many equal chunks (multiples of 128 keys, `least` at least; up to `whole` keys in one) as make no more than `most`
// workgroups with keys, and partials (one per row and chunk) of no more than most_parts rows.  With f the part of the
// keys that the tiles do not see on average, n chunks leave there (n (1 - f) + f) workgroups with keys.  Where that
// gives one chunk and a part of another (`uneven`), a second, shorter one shares the places that one each would leave
// empty: 3000 tokens of 9000 keys 269 -> 230 us, six chunks of up to 300 of 2600 91 -> 75; beside many workgroups of
// the other kind it loses (three of up to 300 and 20 tokens 63 -> 76), and so do a third and later chunk like it.
// A second chunk of less than 0.3 of the first is level in the mean of 24 batches (3400 tokens of 9000 keys 270 -> 246,
// 1658 tokens of 32 / 8 heads of 23335 686 -> 733) and costs partials: none then.
PagedPart part_of(const PagedCall& c, int64_t tiles, int64_t there, int least, int whole, int64_t most, int64_t most_parts,
                  bool uneven) {
  const int64_t len = c.pb.max_len, rows = (int64_t)c.pb.tokens * c.hq;
  if (there < 1) there = 1;
  if (len <= whole) return PagedPart{(int)(tiles * c.hkv), whole, 1};
  const double f = c.causal ? 0.5 * (c.max_new < len ? c.max_new : len) / len : 0.0;
  double n = ((double)most / ((double)there * c.hkv) - f) / (1.0 - f);
  if (!uneven || n < 1.3 || n >= 2.0) n = (double)(int64_t)n;
  if (n > (double)(most_parts / rows)) n = (double)(most_parts / rows);
  if (n < 1.0) n = 1.0;
  int64_t chunk = ((int64_t)std::ceil(len / n) + 127) / 128 * 128;
  if (chunk < least) chunk = least;
  return PagedPart{(int)(tiles * c.hkv), (int)chunk, (int)((len + chunk - 1) / chunk)};
}

template <typename T, int D, int RT>
void launch_rows(const PagedCall& c, const PagedPart& p, float* part) {
  paged_rows_kernel<T, D, RT><<<dim3(p.columns, 1, p.used), kRowWaves * 64, 0, stream()>>>(
      (const T*)c.q, (const T*)c.k, (const T*)c.v, (T*)c.o, c.pb, c.hq, c.hkv, c.G, c.st, c.c2, c.sign, c.causal, c.max_new,
      INT32_MAX, p.chunk, p.used, p.used > 1 ? part : nullptr);
}

// Packed rows of a sequence up to which tiles of 32 rows take it rather than those of paged_tiles.hip.  Where the two meet
// depends on the keys more than on the rows, and this is the middle.  Tiles of 32 rows against the others, us a call, of
// chunks of as many tokens of 16 / 8 heads: over 2000 keys and fewer the small ones win on both sides of the limit (four
// of 48: 27 against 29; of up to 132: 32 against 38; of up to 256: 34 against 36; sixteen of up to 132 of 500:
// 26 against 47), over 8000 and more the large ones do (four of 80 of 8000: 65 against 57; of 100: 88 against 61; of
// up to 256: 126 against 88; one of 256 of 16384: 89 against 60).
constexpr int kFewRows = 256;

template <typename T, int D>
int launch(const PagedCall& c) {
  const int64_t most = (int64_t)c.max_new * c.G, cus = cu_count();
  // (the tiles take pools of equal strides only)
  const bool many_too =
      sizeof(T) == 2 && most > kFewRows && c.st.kp == c.st.vp && c.st.kh == c.st.vh && c.st.kr == c.st.vr;
  const bool few_too = !many_too || c.pb.batch > 1;  // (a sequence alone is one or the other's)
  // Tiles of 256 rows read K and V half as often as those of 128, of which a CU holds two: better where one
  // workgroup per CU is all there is and its keys are many (2048 tokens of 16384, 16 / 8 heads: 285 us against
  // 318), worse with ragged or short ones (four chunks of 512 of 8192: 196 against 179).
  const int64_t tiles8 = many_too && !few_too ? tiles_of(c, 256) : 0;
  const int waves = tiles8 > 0 && tiles8 * c.hkv <= cus && c.pb.max_len >= 6144 ? 8 : 4;
  const int rt = most <= 16 ? 1 : 2;
  const int64_t few_tiles = !few_too ? 0 : tiles_of(c, 16 * rt, 0, many_too ? kFewRows : INT32_MAX);
  const int64_t many_tiles = !many_too ? 0 : (waves == 8 ? tiles8 : tiles_of(c, 128, few_too ? kFewRows : 0));
  KH_REQUIRE((few_tiles + many_tiles) * c.hkv <= (1 << 28) && (int64_t)c.pb.tokens * c.hq <= INT32_MAX,
             "kh_paged_attention: too many query rows");
  // Where both are there, the tiles of few rows are those of a batch in which as many sequences as can be have max_new
  // tokens: it is only the chunks' length that depends on the guess.
  int64_t few_there = few_tiles;
  if (many_too && few_too) {
    const int64_t full = c.pb.tokens / c.max_new < c.pb.batch ? c.pb.tokens / c.max_new : c.pb.batch;
    const int64_t guess = (c.pb.tokens - full * c.max_new) * c.G / 32 + c.pb.batch - full;
    few_there = guess < few_tiles ? guess : few_tiles;
  }
  // Chunks of keys: as many workgroups as the chip holds at once (two per CU, one of 256 rows, one of the rows kernel
  // in fp32 at d 128).  Over 32 batches of single tokens, prompts' chunks and both: 81.7 us in the geometric mean,
  // with a quarter or a half more of them 86.3, with twice as many 88.1, with chunk lengths of powers of two 82.9.
  // 512 keys of a tile at least: partials cost more than shorter chunks gain.  Beside a prompt's many rows, whose
  // workgroups take as long, few rows need no short chunks: partials of 2^18 rows at most.
  const int64_t places = cus * (waves == 8 ? 1 : 2);
  // Few rows of up to 384 bf16 keys stay in one chunk: its third step costs less than the merge's launch (300 keys 7.9 us
  // against 8.1, 200 keys 7.0 against 8.4; 450 keys 9.0 against 8.4; fp32 steps cost more: 200 keys 11.7 against 11.0).
  const PagedPart few =
      part_of(c, few_tiles, few_there, 128, sizeof(T) == 2 ? 384 : 128, cus * (sizeof(T) == 4 && D == 128 ? 1 : 2),
              many_too ? 1 << 18 : INT64_MAX, !many_too);
  const PagedPart many =
      part_of(c, many_tiles, many_tiles, 512, 512, places, INT64_MAX, !few_too || few_there * c.hkv < places / 2);
  const int few_chunks = few_too ? few.used : 1, many_chunks = many_too ? many.used : 1;
  const int chunks = few_chunks > many_chunks ? few_chunks : many_chunks;
  KH_REQUIRE(chunks <= 65535 && (int64_t)few.columns * few_chunks + (int64_t)many.columns * many_chunks <= INT32_MAX,
             "kh_paged_attention: too many chunks of keys");
  float* part = nullptr;
  const int64_t rows = (int64_t)c.pb.tokens * c.hq;
  if (chunks > 1) {
    part = (float*)scratch_alloc((size_t)rows * chunks * (D + 2) * 4);
    if (part == nullptr) return KH_ERR_OOM;
  }
  if (many_too && few_too)
    launch_paged_mixed(c, D, kFewRows, many, few, chunks, part);
  else if (many_too)
    launch_paged_tiles(c, D, waves, many, chunks, part);
  else if (rt == 1)
    launch_rows<T, D, 1>(c, few, part);
  else
    launch_rows<T, D, 2>(c, few, part);
  hipError_t e = hipGetLastError();
  if (part && e == hipSuccess) {
    const MergeArgs a{c.hq, c.causal, c.max_new, c.G, !many_too ? INT32_MAX : (few_too ? kFewRows : 0),
                      few_chunks > 1 ? few.chunk : 0, many_chunks > 1 ? many.chunk : 0, chunks};
    if (c.pb.tokens >= cu_count())
      paged_merge_kernel<T, D><<<c.pb.tokens, 256, 0, stream()>>>(part, (T*)c.o, c.pb, c.st, c.c2, a);
    else
      paged_merge_row_kernel<T, D><<<(unsigned)rows, kMergeWaves * 64, 0, stream()>>>(part, (T*)c.o, c.pb, c.st, c.c2, a);
    e = hipGetLastError();
  }
  if (part) scratch_free(part);
  if (e != hipSuccess) {
    set_error("kh_paged_attention: launch failed: %s", hipGetErrorString(e));
    return KH_ERR_HIP;
  }
  KH_DEBUG_SYNC();
  return KH_OK;
}

}  // namespace

namespace kh {

int paged_batch(const char* who, const int32_t* table, const int32_t* lens, const int32_t* starts, int64_t tokens,
                int64_t batch, int64_t num_pages, int64_t page_size, int64_t table_width, int64_t table_stride,
                int64_t max_kv_len, PagedBatch* pb) {
  KH_REQUIRE(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
             "%s: page size %lld is not a power of two from 16 to 4096", who, (long long)page_size);
  KH_REQUIRE(tokens >= 0 && tokens <= INT32_MAX && batch >= 0 && batch <= 65535, "%s: bad token or sequence count", who);
  KH_REQUIRE(num_pages >= 0 && num_pages <= INT32_MAX && table_width >= 0 && table_stride >= table_width,
             "%s: bad page table", who);
  KH_REQUIRE(table_width <= (1 << 30) && table_width * page_size <= (1 << 30),
             "%s: a page table of %lld pages of %lld rows passes 2^30 rows", who, (long long)table_width, (long long)page_size);
  KH_REQUIRE(starts != nullptr || tokens == batch, "%s: without query starts every sequence has one token (%lld tokens, "
             "%lld sequences)", who, (long long)tokens, (long long)batch);
  KH_REQUIRE(max_kv_len >= 0, "%s: negative max_kv_len", who);
  pb->table = table;
  pb->lens = lens;
  pb->starts = starts;
  pb->table_stride = table_stride;
  pb->batch = (int32_t)batch;
  pb->tokens = (int32_t)tokens;
  pb->num_pages = (int32_t)num_pages;
  pb->page_log = log2_of(page_size);
  pb->table_width = (int32_t)table_width;
  const int64_t most = table_width * page_size;
  pb->max_len = (int32_t)(max_kv_len < most ? max_kv_len : most);
  return KH_OK;
}

}  // namespace kh

extern "C" {

int kh_paged_attention(const void* q, const void* k_pages, const void* v_pages, void* o, const int32_t* page_table,
                       const int32_t* kv_lens, const int32_t* query_starts, int64_t tokens, int64_t batch, int hq,
                       int hkv, int d, int64_t num_pages, int64_t page_size, int64_t table_width,
                       int64_t table_stride, const int64_t* strides, float scale, int causal, int64_t max_query_len,
                       int64_t max_kv_len, int dtype) {
  KH_REQUIRE_INIT();
  KH_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, "kh_paged_attention: numHeadsQ (%d) must be divisible by numHeadsKV (%d)",
             hq, hkv);
  KH_REQUIRE(hq <= 65535, "kh_paged_attention: %d query heads are too many", hq);
  KH_REQUIRE(d == 64 || d == 128, "kh_paged_attention: head_dim %d not supported (64 or 128)", d);
  KH_REQUIRE(dtype == KH_BF16 || dtype == KH_F32, "kh_paged_attention: unsupported dtype %d", dtype);
  KH_REQUIRE(max_query_len >= 0, "kh_paged_attention: negative max_query_len");
  KH_REQUIRE(scale - scale == 0.f, "kh_paged_attention: the scale is not finite");
  PagedCall c;
  const int rc = paged_batch("kh_paged_attention", page_table, kv_lens, query_starts, tokens, batch, num_pages, page_size,
                             table_width, table_stride, max_kv_len, &c.pb);
  if (rc != KH_OK) return rc;
  if (tokens == 0 || batch == 0 || max_query_len == 0) return KH_OK;
  KH_REQUIRE(q && o && kv_lens && strides && (num_pages == 0 || (k_pages && v_pages)) && (table_width == 0 || page_table),
             "kh_paged_attention: null pointer");
  KH_REQUIRE(tokens * (hq / hkv) <= INT32_MAX - 1024, "kh_paged_attention: too many query rows");
  const int per = dtype == KH_BF16 ? 8 : 4;
  bool wide = aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(o);
  for (int i = 0; i < 10; ++i) wide = wide && strides[i] % per == 0;
  KH_REQUIRE(wide, "kh_paged_attention: operands must be 16-byte aligned with 16-byte aligned strides");
  // sixteen rows of a page are addressed with 32-bit byte offsets
  KH_REQUIRE(strides[4] >= 0 && strides[4] <= (1 << 24) && strides[7] >= 0 && strides[7] <= (1 << 24),
             "kh_paged_attention: the pages' row strides must be from 0 to 2^24");
  const int64_t size = dtype == KH_BF16 ? 2 : 4, run = size * d;
  auto rows = [&](const void* at, const int64_t* st) { return Span(at, run, tokens, size * st[0], hq, size * st[1]); };
  auto pool = [&](const void* at, const int64_t* st) {
    return Span(at, run, num_pages, size * st[0], hkv, size * st[1], page_size, size * st[2]);
  };
  KH_REQUIRE(!overlap({rows(o, strides + 8)},
                      {rows(q, strides), pool(k_pages, strides + 2), pool(v_pages, strides + 5),
                       table_span(page_table, table_stride, batch, table_width), ints(kv_lens, batch), ints(query_starts, batch + 1)}),
             "kh_paged_attention: the output must not share memory with the inputs");
  c.q = q;
  c.k = k_pages;
  c.v = v_pages;
  c.o = o;
  c.hq = hq;
  c.hkv = hkv;
  c.G = hq / hkv;
  c.st = PagedStrides{strides[0], strides[1], strides[2], strides[3], strides[4],
                      strides[5], strides[6], strides[7], strides[8], strides[9]};
  c.sign = scale > 0.f ? 1.f : (scale < 0.f ? -1.f : 0.f);
  c.c2 = scale == 0.f ? 1.f : fabsf(scale) * kLog2e;
  c.causal = causal;
  c.max_new = query_starts == nullptr ? 1 : (int)(max_query_len < tokens ? max_query_len : tokens);
  if (dtype == KH_BF16) return d == 64 ? launch<uint16_t, 64>(c) : launch<uint16_t, 128>(c);
  return d == 64 ? launch<float, 64>(c) : launch<float, 128>(c);
}

}  // extern "C"
