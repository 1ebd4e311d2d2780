// Attention of new tokens over a paged KV cache (kh_paged_attention).
#include "paged.h"

using namespace kh;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct PagedStrides {
  int64_t qt, qh, kp, kh, kr, vp, vh, vr, ot, oh;
};

// One wave per (token, query head): 64 keys at a time, a key per lane for the scores and a group of
// columns per lane for the sum.
template <typename T, int D>
__global__ __launch_bounds__(64) void paged_rows_kernel(const T* __restrict__ Q, const T* __restrict__ K,
                                                        const T* __restrict__ V, T* __restrict__ O, PagedBatch pb,
                                                        int hq, int ratio, PagedStrides st, float scale, int causal,
                                                        int max_new) {
  constexpr int C = D / 64;
  const int t = blockIdx.x, h = blockIdx.y, hk = h / ratio, lane = threadIdx.x;
  const int b = pb.sequence_of(t);
  if (b < 0) return;
  const int len = pb.len(b), n = pb.count(b), j = t - pb.first(b);
  if (j >= max_new) return;
  const int seen = min(pb.max_len, causal ? max(0, len - n + j + 1) : len);
  const T* q = Q + t * st.qt + h * st.qh;
  float m = -INFINITY, l = 0.f, o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = 0.f;
  for (int k0 = 0; k0 < seen; k0 += 64) {
    const int key = k0 + lane;
    int id = -1;
    if (key < seen) id = pb.table[b * pb.table_stride + (key >> pb.page_log)];
    const bool there = pb.is_page(id);
    const int64_t slot = key & ((1 << pb.page_log) - 1);
    float s = -INFINITY;
    if (there) {
      const T* k = K + id * st.kp + hk * st.kh + slot * st.kr;
      float d = 0.f;
      for (int i = 0; i < D; ++i) d += Elem<T>::load(q, i) * Elem<T>::load(k, i);
      s = d * scale;
    }
    const float mn = fmaxf(m, wave_max(s)), mu = mn == -INFINITY ? 0.f : mn;
    const float a = m == -INFINITY ? 0.f : exp2f((m - mu) * kLog2e), p = exp2f((s - mu) * kLog2e);
    l = l * a + wave_sum(p);
    m = mn;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] *= a;
    for (int i = 0; i < 64; ++i) {
      const int idi = __shfl(id, i, 64);
      const float pi = __shfl(p, i, 64);
      if (!pb.is_page(idi)) continue;
      const T* v = V + idi * st.vp + hk * st.vh + ((k0 + i) & ((1 << pb.page_log) - 1)) * st.vr;
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] += pi * Elem<T>::load(v, lane * C + c);
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) Elem<T>::store(O + t * st.ot + h * st.oh, lane * C + c, l > 0.f || l != l ? o[c] / l : 0.f);
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
  KH_REQUIRE(table_width * page_size <= INT32_MAX, "%s: a page table of %lld pages of %lld rows passes 2^31 rows", who,
             (long long)table_width, (long long)page_size);
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
  PagedBatch pb;
  const int rc = paged_batch("kh_paged_attention", page_table, kv_lens, query_starts, tokens, batch, num_pages, page_size,
                             table_width, table_stride, max_kv_len, &pb);
  if (rc != KH_OK) return rc;
  if (tokens == 0 || batch == 0 || max_query_len == 0) return KH_OK;
  KH_REQUIRE(q && o && kv_lens && strides && (num_pages == 0 || (k_pages && v_pages)) && (table_width == 0 || page_table),
             "kh_paged_attention: null pointer");
  const int per = dtype == KH_BF16 ? 8 : 4;
  bool wide = aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(o);
  for (int i = 0; i < 10; ++i) wide = wide && strides[i] % per == 0;
  KH_REQUIRE(wide, "kh_paged_attention: operands must be 16-byte aligned with 16-byte aligned strides");
  const PagedStrides st{strides[0], strides[1], strides[2], strides[3], strides[4],
                        strides[5], strides[6], strides[7], strides[8], strides[9]};
  const int max_new = (int)(max_query_len < tokens ? max_query_len : tokens);
  const dim3 grid((unsigned)tokens, hq);
#define KH_PAGED_ROWS(T, DD)                                                                                        \
  paged_rows_kernel<T, DD><<<grid, 64, 0, stream()>>>((const T*)q, (const T*)k_pages, (const T*)v_pages, (T*)o, pb, \
                                                      hq, hq / hkv, st, scale, causal, max_new)
  if (dtype == KH_BF16) {
    if (d == 64)
      KH_PAGED_ROWS(uint16_t, 64);
    else
      KH_PAGED_ROWS(uint16_t, 128);
  } else {
    if (d == 64)
      KH_PAGED_ROWS(float, 64);
    else
      KH_PAGED_ROWS(float, 128);
  }
#undef KH_PAGED_ROWS
  KH_CHECK_LAUNCH();
  return KH_OK;
}

}  // extern "C"
