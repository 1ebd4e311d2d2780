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
#include <type_traits>

#include "flash_tiles.h"
#include "paged.h"

using namespace kh;

namespace {

// ---- few rows: K and V straight from the pages into MFMA operands --------------------------------
//
// A workgroup of four waves takes one tile of 16 RT packed rows of one kv head and one chunk of keys; wave
// w takes the chunk's 32-key blocks w, w + 4, ...  A 32-key block is two 16-key halves, each inside one
// page (pages are multiples of 16 rows), so its page id and base address are wave-uniform.
//
//   S^T (16 keys x 16 rows) = K Q^T with v_mfma_f32_16x16x32_bf16 (or _16x16x4_f32): lane (r, q), r =
//     lane % 16, q = lane / 16, loads K row r of the half, columns 32 c + 8 q .. + 7 (fp32: 16 c + 4 q .. + 3)
//     and gets the scores of packed row r with keys 4 q + i.
//   O^T += V^T P^T: the k slots of the product may hold the keys in any order that P and V share, so lane
//     (r, q) keeps the P values it has (keys 4 q + i of both halves) and loads the V rows of those keys, D/16
//     consecutive columns EPL r ..: 16 lanes read a whole row.  Tile dt of O^T has the columns EPL r + dt.
// Nothing passes through LDS until the waves' (m, l, O) are joined at the end.
//
// Softmax relative to a reference maximum m (raw q . k units) that the accumulators start from, raised
// only when a lane's sum of P exceeds kSumMax, as in the contiguous prefill kernel: O / l does not depend on
// it, and P <= kSumMax holds whatever the scores are.
constexpr int kRowWaves = 4;

template <typename T, int D>
struct RowOps;

// bfloat16
template <int D>
struct RowOps<uint16_t, D> {
  static constexpr int NK = D / 32, EPL = D / 16;
  struct K {
    uint4 v[NK];
  };
  using VRow = std::conditional_t<EPL == 8, uint4, uint2>;
  struct Q {
    bf16x8 v[NK];
  };
  // A query row, and the row times sign (0: zeros whatever it holds).
  static __device__ __forceinline__ void load_q(Q& q, const uint16_t* row, int lq) {
#pragma unroll
    for (int c = 0; c < NK; ++c)
      q.v[c] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(row + 32 * c + 8 * lq));
  }
  static __device__ __forceinline__ void sign_q(Q& q, float sign) {
    const uint32_t flip = sign < 0.f ? 0x80008000u : 0u, keep = sign != 0.f ? ~0u : 0u;
#pragma unroll
    for (int c = 0; c < NK; ++c) {
      uint4 u = __builtin_bit_cast(uint4, q.v[c]);
      u.x = (u.x ^ flip) & keep;
      u.y = (u.y ^ flip) & keep;
      u.z = (u.z ^ flip) & keep;
      u.w = (u.w ^ flip) & keep;
      q.v[c] = __builtin_bit_cast(bf16x8, u);
    }
  }
  static __device__ __forceinline__ void load_k(K& k, __amdgpu_buffer_rsrc_t r, uint32_t off, int lq) {
#pragma unroll
    for (int c = 0; c < NK; ++c) k.v[c] = buf_load16(r, off + 64 * c + 16 * lq);
  }
  static __device__ __forceinline__ void load_v(VRow& v, __amdgpu_buffer_rsrc_t r, uint32_t off) {
    if constexpr (EPL == 8)
      v = buf_load16(r, off);
    else
      v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
  }
  static __device__ __forceinline__ f32x4 qk(const K& k, const Q& q, f32x4 s) {
#pragma unroll
    for (int c = 0; c < NK; ++c)
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k.v[c]), q.v[c], s, 0, 0, 0);
    return s;
  }
  static __device__ __forceinline__ uint32_t word(const VRow& v, int w) {
    if constexpr (EPL == 8)
      return w == 0 ? v.x : (w == 1 ? v.y : (w == 2 ? v.z : v.w));
    else
      return w == 0 ? v.x : v.y;
  }
  // P of one row tile as the products take it, and the lane's sum of those values.
  struct P {
    bf16x8 v;
  };
  static __device__ __forceinline__ float exponentiate(const f32x4 (&s)[2], float c2, P& p) {
    float sum = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __bf16 b = (__bf16)fast_exp2(s[h][i] * c2);
        p.v[4 * h + i] = b;
        sum += (float)b;
      }
    return sum;
  }
  template <int RT>
  static __device__ __forceinline__ void pv(const VRow (&v)[8], const P (&p)[RT], f32x4 (&o)[RT][EPL]) {
#pragma unroll
    for (int dt = 0; dt < EPL; ++dt) {
      const uint32_t sel = (dt & 1) ? 0x07060302u : 0x05040100u;  // the high or low halves of two words
      uint4 a;
      a.x = __builtin_amdgcn_perm(word(v[1], dt >> 1), word(v[0], dt >> 1), sel);
      a.y = __builtin_amdgcn_perm(word(v[3], dt >> 1), word(v[2], dt >> 1), sel);
      a.z = __builtin_amdgcn_perm(word(v[5], dt >> 1), word(v[4], dt >> 1), sel);
      a.w = __builtin_amdgcn_perm(word(v[7], dt >> 1), word(v[6], dt >> 1), sel);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), p[rt].v, o[rt][dt], 0, 0, 0);
    }
  }
  // Whether a V row's values are all finite; and value dt of it.
  static __device__ __forceinline__ bool odd(const VRow& v) {
    bool any = false;
#pragma unroll
    for (int w = 0; w < EPL / 2; ++w) {
      const uint32_t u = word(v, w);
      any = any || (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
    }
    return any;
  }
  static __device__ __forceinline__ void clear(VRow& v) {
    if constexpr (EPL == 8)
      v = make_uint4(0, 0, 0, 0);
    else
      v = make_uint2(0, 0);
  }
  static __device__ __forceinline__ float p_of(const P& p, int e) { return (float)p.v[e]; }
  static __device__ __forceinline__ void store(uint16_t* o, const float (&f)[4 * EPL]) {
#pragma unroll
    for (int i = 0; i < 4 * EPL; i += 8) {
      float g[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = f[i + j];
      *reinterpret_cast<uint4*>(o + i) = pack_bf16x8(g);
    }
  }
};

// float32
template <int D>
struct RowOps<float, D> {
  static constexpr int NK = D / 16, EPL = D / 16;
  struct K {
    f32x4 v[NK];
  };
  struct VRow {
    f32x4 v[EPL / 4];
  };
  struct Q {
    f32x4 v[NK];
  };
  static __device__ __forceinline__ void load_q(Q& q, const float* row, int lq) {
#pragma unroll
    for (int c = 0; c < NK; ++c) q.v[c] = *reinterpret_cast<const f32x4*>(row + 16 * c + 4 * lq);
  }
  static __device__ __forceinline__ void sign_q(Q& q, float sign) {
#pragma unroll
    for (int c = 0; c < NK; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) q.v[c][i] = sign == 0.f ? 0.f : q.v[c][i] * sign;
  }
  static __device__ __forceinline__ void load_k(K& k, __amdgpu_buffer_rsrc_t r, uint32_t off, int lq) {
#pragma unroll
    for (int c = 0; c < NK; ++c) k.v[c] = __builtin_bit_cast(f32x4, buf_load16(r, off + 64 * c + 16 * lq));
  }
  static __device__ __forceinline__ void load_v(VRow& v, __amdgpu_buffer_rsrc_t r, uint32_t off) {
#pragma unroll
    for (int i = 0; i < EPL / 4; ++i) v.v[i] = __builtin_bit_cast(f32x4, buf_load16(r, off + 16 * i));
  }
  static __device__ __forceinline__ f32x4 qk(const K& k, const Q& q, f32x4 s) {
#pragma unroll
    for (int c = 0; c < NK; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k.v[c][i], q.v[c][i], s, 0, 0, 0);
    return s;
  }
  struct P {
    float v[8];
  };
  static __device__ __forceinline__ float exponentiate(const f32x4 (&s)[2], float c2, P& p) {
    float sum = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p.v[4 * h + i] = fast_exp2(s[h][i] * c2);
        sum += p.v[4 * h + i];
      }
    return sum;
  }
  template <int RT>
  static __device__ __forceinline__ void pv(const VRow (&v)[8], const P (&p)[RT], f32x4 (&o)[RT][EPL]) {
#pragma unroll
    for (int dt = 0; dt < EPL; ++dt)
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e].v[dt / 4][dt % 4], p[rt].v[e], o[rt][dt], 0, 0, 0);
  }
  static __device__ __forceinline__ bool odd(const VRow& v) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < EPL; ++i) any = any || (__float_as_uint(v.v[i / 4][i % 4]) & 0x7f800000u) == 0x7f800000u;
    return any;
  }
  static __device__ __forceinline__ void clear(VRow& v) {
#pragma unroll
    for (int i = 0; i < EPL / 4; ++i) v.v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  static __device__ __forceinline__ float p_of(const P& p, int e) { return p.v[e]; }
  static __device__ __forceinline__ void store(float* o, const float (&f)[4 * EPL]) {
#pragma unroll
    for (int i = 0; i < 4 * EPL; i += 4) *reinterpret_cast<f32x4*>(o + i) = f32x4{f[i], f[i + 1], f[i + 2], f[i + 3]};
  }
};

template <typename T, int D, int RT>
__global__ __launch_bounds__(kRowWaves * 64, sizeof(T) == 4 && D == 128 ? 1 : 2) void paged_rows_kernel(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, T* __restrict__ O, PagedBatch pb, int hq,
    int hkv, int G, PagedStrides st, float c2, float sign, int causal, int max_new, int most_rows, int chunk, int chunks, float* __restrict__ part) {
  using R = RowOps<T, D>;
  constexpr int EPL = R::EPL;
  constexpr int MS = 2 + 4 * EPL;  // floats per lane and row tile that the waves exchange
  __shared__ float join[(kRowWaves - 1) * RT * MS * 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, lq = lane >> 4;
  // Workgroups go to the eight XCDs in turn: with the kv head innermost an XCD's L2 holds the rows of one or a few
  // heads, which sequences that share pages (beams of one prompt) read at about the same time.
  const int hk = blockIdx.x % hkv, split = blockIdx.z;
  const Tile t = find_tile(pb, blockIdx.x / hkv, G, 16 * RT, max_new, 0, most_rows);
  if (t.b < 0) return;
  // the keys that the tile's last row sees bound the tile's
  const int last = min(t.row0 + 16 * RT, t.rows) - 1;
  const int end = seen_by(t, last / G, causal, pb.max_len);
  const int k0 = split * chunk, k1 = min(end, k0 + chunk);
  if (split > 0 && k0 >= end) return;  // (the first chunk of a tile without keys stores zeros)

  typename R::Q q[RT];
  int sees[RT];  // keys that this lane's packed row sees
  int64_t at[RT];
  bool there[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int xr = t.row0 + 16 * rt + r, x = min(xr, t.rows - 1), j = x / G, h = hk * G + x - j * G;
    there[rt] = xr < t.rows;  // (a row that is not there reads the last one's query, and leaves nothing)
    sees[rt] = there[rt] ? seen_by(t, j, causal, pb.max_len) : 0;
    at[rt] = (int64_t)(t.t0 + j) * hq + h;
    R::load_q(q[rt], Q + (int64_t)(t.t0 + j) * st.qt + (int64_t)h * st.qh, lq);
  }
  const int first_sees = seen_by(t, t.row0 / G, causal, pb.max_len);  // the fewest keys that a row of the tile sees

  f32x4 o[RT][EPL];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = there[rt] ? -INFINITY : 0.f;  // (a row that is not there never asks for a raise)
    l[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < EPL; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int32_t* table = pb.table + t.b * pb.table_stride;
  const int page_mask = (1 << pb.page_log) - 1;
  typename R::K kr[2];
  typename R::VRow vr[8];
  bool held[2];
  // Page ids of the wave's next 32 blocks, one half per lane (-1: none, or behind `end`): one load ahead of
  // the rows' own, which wait for nothing then.
  int ids = -1;
  auto load_ids = [&](int kb) {
    const int key = kb + 32 * kRowWaves * (lane >> 1) + 16 * (lane & 1);
    ids = key < min(pb.max_len, k0 + chunk) ? table[key >> pb.page_log] : -1;
  };
  // Half h of the wave's block n (at key kb): its page's rows as far as keys below `end` go; a half in no
  // page, or behind `end`, reads as zeros.
  auto rsrc = [&](const T* base, int64_t sp, int64_t sh, int64_t sr, int kb, int n, int h, bool* in) {
    const int key = kb + 16 * h;
    const int id = __builtin_amdgcn_readlane(ids, 2 * (n & 31) + h);
    const bool ok = pb.is_page(id);
    *in = ok;
    const int rows = ok ? min(16, end - key) : 0;
    const T* p = base + (int64_t)(ok ? id : 0) * sp + (int64_t)hk * sh + (int64_t)(key & page_mask) * sr;
    return make_rsrc(p, rows > 0 ? (uint32_t)(((int64_t)(rows - 1) * sr + D) * sizeof(T)) : 0u);
  };
  auto load_k = [&](int kb, int n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto rk = rsrc(K, st.kp, st.kh, st.kr, kb, n, h, &held[h]);
      R::load_k(kr[h], rk, (uint32_t)(r * st.kr * sizeof(T)), lq);
    }
  };
  auto load_v = [&](int kb, int n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bool in;
      const auto rv = rsrc(V, st.vp, st.vh, st.vr, kb, n, h, &in);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        R::load_v(vr[4 * h + i], rv, (uint32_t)(((4 * lq + i) * st.vr + EPL * r) * sizeof(T)));
    }
  };
  int kb = k0 + 32 * wave;
  load_ids(kb);
  if (kb < k1) {
    load_k(kb, 0);
    load_v(kb, 0);
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) R::sign_q(q[rt], there[rt] ? sign : 0.f);
#pragma unroll 1
  for (int n = 1; kb < k1; kb += 32 * kRowWaves, ++n) {
    f32x4 s[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float mn = m[rt] == -INFINITY ? 0.f : -m[rt];
#pragma unroll
      for (int h = 0; h < 2; ++h) s[rt][h] = R::qk(kr[h], q[rt], f32x4{mn, mn, mn, mn});
    }
    const bool hole0 = !held[0], hole1 = !held[1];
    const bool more = kb + 32 * kRowWaves < k1;
    if (more) {
      if ((n & 31) == 0) load_ids(kb + 32 * kRowWaves);
      load_k(kb + 32 * kRowWaves, n);
    }
    const bool cut = kb + 32 > first_sees;  // some row of the tile does not see all 32 keys
    if (cut || hole0 || hole1)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (kb + 16 * h + 4 * lq + i >= sees[rt] || (h == 0 ? hole0 : hole1)) s[rt][h][i] = -INFINITY;
    typename R::P p[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float ps = R::exponentiate(s[rt], c2, p[rt]);
      if (__any(m[rt] == -INFINITY || !(ps <= kSumMax))) {
        // raise the rows' reference to their maximum over the block: lanes r, r + 16, .. hold one row
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rt][h][i]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        float d, alpha;
        if (m[rt] == -INFINITY) {
          d = mx == -INFINITY ? 0.f : mx;
          alpha = 0.f;
          m[rt] = mx;
        } else {
          d = fmaxf(mx, 0.f);
          alpha = fast_exp2(-d * c2);
          m[rt] += d;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[rt][h][i] -= d;
        l[rt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < EPL; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[rt][dt][i] *= alpha;
        ps = R::exponentiate(s[rt], c2, p[rt]);
      }
      l[rt] += ps;
    }
    if (cut) {
      // A row that some packed rows see and others do not may hold infinities or NaN, and 0 times those is
      // not 0: such V rows are taken out of the products and added key by key to the rows that see them.
      bool any = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) any = any || R::odd(vr[e]);
      if (__any(any)) {
        for (int e = 0; e < 8; ++e)
          for (int qq = 0; qq < 4; ++qq) {
            const int key = kb + 16 * (e >> 2) + 4 * qq + (e & 3);
            if (key >= end) continue;
            const int id = table[key >> pb.page_log];
            if (!pb.is_page(id)) continue;
            const T* v = V + (int64_t)id * st.vp + (int64_t)hk * st.vh + (int64_t)(key & page_mask) * st.vr;
            bool bad = false;
            for (int d = lane; d < D; d += 64) bad = bad || !(fabsf(Elem<T>::load(v, d)) < INFINITY);
            if (!__any(bad)) continue;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              float pe = 0.f;
#pragma unroll
              for (int ee = 0; ee < 8; ++ee)
                if (ee == e) pe = R::p_of(p[rt], ee);
              pe = __shfl(pe, 16 * qq + r, 64);
              if (key < sees[rt])
#pragma unroll
                for (int dt = 0; dt < EPL; ++dt)
#pragma unroll
                  for (int i = 0; i < 4; ++i) o[rt][dt][i] += pe * Elem<T>::load(v, EPL * (4 * lq + i) + dt);
            }
#pragma unroll
            for (int ee = 0; ee < 8; ++ee)
              if (ee == e && lq == qq) R::clear(vr[ee]);
          }
      }
    }
    R::template pv<RT>(vr, p, o);
    if (more) load_v(kb + 32 * kRowWaves, n);
  }

  // Join the waves in wave order.
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += __shfl_xor(l[rt], 16, 64);
    l[rt] += __shfl_xor(l[rt], 32, 64);
  }
  if (wave > 0) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float* p = join + ((wave - 1) * RT + rt) * MS * 64 + lane;
      p[0] = m[rt];
      p[64] = l[rt];
#pragma unroll
      for (int dt = 0; dt < EPL; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[(2 + 4 * dt + i) * 64] = o[rt][dt][i];
    }
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float mo[kRowWaves], mt = m[rt];
    mo[0] = m[rt];
#pragma unroll
    for (int w = 1; w < kRowWaves; ++w) {
      mo[w] = join[((w - 1) * RT + rt) * MS * 64 + lane];
      mt = fmaxf(mt, mo[w]);
    }
    float f[4 * EPL];  // columns 4 EPL lq ..: tile dt's column i is EPL (4 lq + i) + dt
    const float a0 = mo[0] == -INFINITY ? 0.f : fast_exp2((mo[0] - mt) * c2);
    float lt = l[rt] * a0;
#pragma unroll
    for (int dt = 0; dt < EPL; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) f[EPL * i + dt] = o[rt][dt][i] * a0;
#pragma unroll
    for (int w = 1; w < kRowWaves; ++w) {
      const float* p = join + ((w - 1) * RT + rt) * MS * 64 + lane;
      const float a = mo[w] == -INFINITY ? 0.f : fast_exp2((mo[w] - mt) * c2);
      lt += a * p[64];
#pragma unroll
      for (int dt = 0; dt < EPL; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) f[EPL * i + dt] += a * p[(2 + 4 * dt + i) * 64];
    }
    if (!there[rt]) continue;
    if (part == nullptr) {
      const float inv = lt > 0.f || lt != lt ? 1.f / lt : 0.f;
#pragma unroll
      for (int i = 0; i < 4 * EPL; ++i) f[i] *= inv;
      const int64_t tok = at[rt] / hq, h = at[rt] - tok * hq;
      R::store(O + tok * st.ot + h * st.oh + 4 * EPL * lq, f);
    } else {
      float* po = part_o<D>(part, at[rt], chunks, split) + 4 * EPL * lq;
#pragma unroll
      for (int i = 0; i < 4 * EPL; i += 4) *reinterpret_cast<f32x4*>(po + i) = f32x4{f[i], f[i + 1], f[i + 2], f[i + 3]};
      if (lq == 0) part_ml<D>(part, (int64_t)pb.tokens * hq, chunks, at[rt])[split] = make_float2(mt, lt);
    }
  }
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

// Many rows: a workgroup per token, D / 4 lanes per row (query head), so that the token's place is looked up once
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

// Few rows: a workgroup per (token, query head); wave w sums chunks w, w + 4, ..., several loads in flight, and the
// four sums are added in wave order.
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

// The length of a chunk of keys: the shortest of least, 2 least, 4 least ... that makes no more than `most` workgroups
// of `tiles` tiles per kv head, or the whole length.
int chunk_of(const PagedCall& c, int64_t tiles, int least, int64_t most) {
  int64_t chunk = least;
  while (chunk < c.pb.max_len && tiles * c.hkv * ((c.pb.max_len + chunk - 1) / chunk) > most) chunk *= 2;
  return (int)chunk;
}

template <typename T, int D, int RT>
void launch_rows(const PagedCall& c, int most_rows, int64_t tiles, int chunk, int used, int chunks, float* part) {
  paged_rows_kernel<T, D, RT><<<dim3((unsigned)(tiles * c.hkv), 1, used), kRowWaves * 64, 0, stream()>>>(
      (const T*)c.q, (const T*)c.k, (const T*)c.v, (T*)c.o, c.pb, c.hq, c.hkv, c.G, c.st, c.c2, c.sign, c.causal, c.max_new,
      most_rows, chunk, chunks, part);
}

// Packed rows of a sequence up to which paged_rows_kernel takes it beside paged_tiles.hip: with 160 rows of up to 8000
// keys (four sequences) it is at 55 us and the tiles at 80, with 96 of 2000 at 19 against 32; with 400 to 512
// rows the tiles come level (512 of 16384 keys: 59 us against 87).
constexpr int kFewRows = 256;

template <typename T, int D>
int launch(const PagedCall& c) {
  const int64_t most = (int64_t)c.max_new * c.G, cus = cu_count();
  // (the tiles take pools of equal strides only)
  const bool tiles_too =
      sizeof(T) == 2 && most > kFewRows && c.st.kp == c.st.vp && c.st.kh == c.st.vh && c.st.kr == c.st.vr;
  // rows up to which paged_rows_kernel takes a sequence; a sequence alone is one or the other's
  const int few = tiles_too ? (c.pb.batch > 1 ? kFewRows : 0) : INT32_MAX;
  const int rt = most <= 16 ? 1 : 2;
  const int64_t few_tiles = few == 0 ? 0 : tiles_of(c, 16 * rt);
  // Tiles of 256 rows read K and V half as often as those of 128, of which a CU holds two: better where one
  // workgroup per CU is all there is and its keys are many (2048 tokens of 16384, 16 / 8 heads: 281 us against
  // 317), worse with ragged or short ones (four chunks of 512 of 8192: 196 against 179).
  const int64_t tiles8 = tiles_too ? tiles_of(c, 256) : 0;
  const int waves = tiles8 * c.hkv <= cus && c.pb.max_len >= 6144 ? 8 : 4;
  const int64_t many_tiles = !tiles_too ? 0 : (waves == 8 ? tiles8 : tiles_of(c, 128));
  // Chunks of keys: more workgroups than the chip holds at once, and shorter chunks than 512 keys of a tile, cost
  // more in partials than they gain (2600 keys of six ragged chunks: 88 us, 98 in twice as many chunks).  The
  // rows kernel runs two workgroups per CU, one of fp32 at d 128.
  const int few_chunk = chunk_of(c, few_tiles, 128, 5 * cus * (sizeof(T) == 4 && D == 128 ? 1 : 2) / 4);
  const int many_chunk = chunk_of(c, many_tiles, 512, waves == 8 ? cus : 2 * cus);
  auto count = [&](int chunk) { return c.pb.max_len > chunk ? (c.pb.max_len + chunk - 1) / chunk : 1; };
  const int few_chunks = few ? count(few_chunk) : 1, many_chunks = tiles_too ? count(many_chunk) : 1;
  const int chunks = few_chunks > many_chunks ? few_chunks : many_chunks;
  KH_REQUIRE(few_tiles * c.hkv <= INT32_MAX && many_tiles * c.hkv <= INT32_MAX && chunks <= 65535,
             "kh_paged_attention: too many tiles");
  KH_REQUIRE((int64_t)c.pb.tokens * c.hq <= INT32_MAX, "kh_paged_attention: too many rows");
  float* part = nullptr;
  const int64_t rows = (int64_t)c.pb.tokens * c.hq;
  if (chunks > 1) {
    part = (float*)scratch_alloc((size_t)rows * chunks * (D + 2) * 4);
    if (part == nullptr) return KH_ERR_OOM;
  }
  hipError_t e = hipSuccess;
  if (tiles_too) {
    launch_paged_tiles(c, D, waves, few, many_tiles, many_chunk, many_chunks, chunks,
                       many_chunks > 1 ? part : nullptr);
    e = hipGetLastError();
  }
  if (few && e == hipSuccess) {
    float* p = few_chunks > 1 ? part : nullptr;
    if (rt == 1)
      launch_rows<T, D, 1>(c, few, few_tiles, few_chunk, few_chunks, chunks, p);
    else
      launch_rows<T, D, 2>(c, few, few_tiles, few_chunk, few_chunks, chunks, p);
    e = hipGetLastError();
  }
  if (part && e == hipSuccess) {
    const MergeArgs a{c.hq,      c.causal, c.max_new, c.G, few, few_chunks > 1 ? few_chunk : 0, many_chunks > 1 ? many_chunk : 0,
                      chunks};
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
