// Paged attention of few query rows (paged_attention.hip; beside many rows in one launch: paged_tiles.hip).
#pragma once

#include <type_traits>

#include "flash_tiles.h"
#include "paged.h"

namespace kh {

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
// Long caches: bound by the loads in flight and by uneven chunks (8 bf16 sequences of 8k to 32k keys: 127 us, 5.1 TB/s;
// a large copy moves 4.9, the contiguous decode kernel reads 6.2).  Pages that sequences share come from L2 (four
// prompts' eight beams, 1531 keys: 20 us, 200 MB at 10 TB/s).  Short caches: the chain of length, page id, rows, products
// and join (two fp32 sequences of 777 keys: 9 us, one 32-key block per wave).  32 rows in fp32: the fp32 MFMAs of the
// longest tile with one wave per SIMD (200 tokens of 1000: 49 us).  Cache hints on the loads gained nothing; 64 fp32 rows
// that share K and V through LDS gained 3 to 18 % on long caches and lost 10 % on short ones.
//
// Softmax relative to a reference maximum m (raw q . k units) that the accumulators start from, raised
// only when a lane's sum of P exceeds kSumMax, as in the contiguous prefill kernel: O / l does not depend on
// it, and P <= kSumMax holds whatever the scores are.
//
// In bf16 P goes through the second product in two parts (2^-16 of it is lost rather than 2^-8), so that only the
// result is rounded to 8 bits: 2-norm error 1.7e-3, with one part 2.5e-3.  The matrix cores have room for it beside
// the loads: 8 sequences of 8k to 32k keys 0.5 % slower, four of 120 tokens of 4000 keys, which the products bound, 1 %.
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
  // (the products of different sums take turns: one that waits for its own last result leaves the matrix core idle)
  template <int RT>
  static __device__ __forceinline__ void qk(const K (&k)[2], const Q (&q)[RT], f32x4 (&s)[RT][2]) {
#pragma unroll
    for (int c = 0; c < NK; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          s[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[h].v[c]), q[rt].v[c], s[rt][h], 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t word(const VRow& v, int w) {
    if constexpr (EPL == 8)
      return w == 0 ? v.x : (w == 1 ? v.y : (w == 2 ? v.z : v.w));
    else
      return w == 0 ? v.x : v.y;
  }
  // P of one row tile as the products take it, rounded and what is left of it, rounded; and the lane's sum of P.
  struct P {
    bf16x8 v, rest;
  };
  static __device__ __forceinline__ float exponentiate(const f32x4 (&s)[2], float c2, P& p) {
    float sum = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = fast_exp2(s[h][i] * c2);
        const __bf16 b = (__bf16)e;
        p.v[4 * h + i] = b;
        p.rest[4 * h + i] = (__bf16)(e - (float)b);
        sum += e;
      }
    return sum;
  }
  template <int RT>
  static __device__ __forceinline__ void pv(const VRow (&v)[8], const P (&p)[RT], f32x4 (&o)[RT][EPL], bool both) {
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
      if (both)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), p[rt].rest, o[rt][dt], 0, 0, 0);
    }
  }
  // Whether any of the V rows' values is infinite or NaN.
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ bool odd(const VRow (&v)[8]) {
    u16x2 most = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int w = 0; w < EPL / 2; ++w)
        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, word(v[e], w) & 0x7fff7fffu));
    return most[0] >= 0x7f80u || most[1] >= 0x7f80u;
  }
  static __device__ __forceinline__ void clear(VRow& v) {
    if constexpr (EPL == 8)
      v = make_uint4(0, 0, 0, 0);
    else
      v = make_uint2(0, 0);
  }
  static __device__ __forceinline__ float p_of(const P& p, int e) { return (float)p.v[e] + (float)p.rest[e]; }
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
  template <int RT>
  static __device__ __forceinline__ void qk(const K (&k)[2], const Q (&q)[RT], f32x4 (&s)[RT][2]) {
#pragma unroll
    for (int c = 0; c < NK; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            s[rt][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[h].v[c][i], q[rt].v[c][i], s[rt][h], 0, 0, 0);
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
  static __device__ __forceinline__ void pv(const VRow (&v)[8], const P (&p)[RT], f32x4 (&o)[RT][EPL], bool) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int dt = 0; dt < EPL; ++dt)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e].v[dt / 4][dt % 4], p[rt].v[e], o[rt][dt], 0, 0, 0);
  }
  static __device__ __forceinline__ bool odd(const VRow (&v)[8]) {
    bool any = false;
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < EPL; ++i) any = any || (__float_as_uint(v[e].v[i / 4][i % 4]) & 0x7f800000u) == 0x7f800000u;
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
struct RowLds {
  static constexpr int MS = 2 + 4 * RowOps<T, D>::EPL;  // floats per lane and row tile that the waves exchange
  static constexpr int FLOATS = (kRowWaves - 1) * RT * MS * 64;
};

// Tile `column` / hkv of kv head `column` % hkv and chunk `split`; join: RowLds::FLOATS of LDS.
template <typename T, int D, int RT>
__device__ __forceinline__ void paged_rows(float* join, int column, int split, const T* __restrict__ Q,
                                           const T* __restrict__ K, const T* __restrict__ V, T* __restrict__ O,
                                           const PagedBatch& pb, int hq, int hkv, int G, const PagedStrides& st, float c2,
                                           float sign, int causal, int max_new, int most_rows, int chunk, int chunks,
                                           float* __restrict__ part) {
  using R = RowOps<T, D>;
  constexpr int EPL = R::EPL;
  constexpr int MS = RowLds<T, D, RT>::MS;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, lq = lane >> 4;
  // Workgroups go to the eight XCDs in turn: with the kv head innermost an XCD's L2 holds the rows of one or a few
  // heads, which sequences that share pages (beams of one prompt) read at about the same time.
  const int hk = column % hkv;
  const Tile t = find_tile(pb, column / hkv, G, 16 * RT, max_new, 0, most_rows);
  if (t.b < 0) return;
  // Page ids of the wave's next 32 blocks, one half per lane (-1: none, or behind the chunk): one load ahead of
  // the rows' own, which wait for nothing then.  The first are under way beside the length's own load.
  const int32_t* table = pb.table + t.b * pb.table_stride;
  const int page_mask = (1 << pb.page_log) - 1, k0 = split * chunk;
  int ids = -1;
  auto load_ids = [&](int kb) {
    const int key = kb + 32 * kRowWaves * (lane >> 1) + 16 * (lane & 1);
    ids = key < min(pb.max_len, k0 + chunk) ? table[key >> pb.page_log] : -1;
  };
  load_ids(k0 + 32 * wave);
  typename R::Q q[RT];
  int at_j[RT];
  int64_t at[RT];
  bool there[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int xr = t.row0 + 16 * rt + r, x = min(xr, t.rows - 1), j = x / G, h = hk * G + x - j * G;
    there[rt] = xr < t.rows;  // (a row that is not there reads the last one's query, and leaves nothing)
    at_j[rt] = j;
    at[rt] = (int64_t)(t.t0 + j) * hq + h;
    R::load_q(q[rt], Q + (int64_t)(t.t0 + j) * st.qt + (int64_t)h * st.qh, lq);
  }
  // the keys that the tile's last row sees bound the tile's
  const int last = min(t.row0 + 16 * RT, t.rows) - 1;
  const int end = seen_by(t, last / G, causal, pb.max_len);
  const int k1 = min(end, k0 + chunk);
  if (split > 0 && k0 >= end) return;  // (the first chunk of a tile without keys stores zeros)

  int sees[RT];  // keys that this lane's packed row sees
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) sees[rt] = there[rt] ? seen_by(t, at_j[rt], causal, pb.max_len) : 0;
  const int first_sees = seen_by(t, t.row0 / G, causal, pb.max_len);  // the fewest keys that a row of the tile sees

  f32x4 o[RT][EPL];
  float m[RT], l[RT];
  typename R::K kr[2];
  typename R::VRow vr[8];
  bool held[2];
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
  if (kb < k1) {
    load_k(kb, 0);
    load_v(kb, 0);
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) R::sign_q(q[rt], there[rt] ? sign : 0.f);
  bool both = sizeof(T) == 2;  // both parts of P
again:
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = there[rt] ? -INFINITY : 0.f;  // (a row that is not there never asks for a raise)
    l[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < EPL; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll 1
  for (int n = 1; kb < k1; kb += 32 * kRowWaves, ++n) {
    f32x4 s[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float mn = m[rt] == -INFINITY ? 0.f : -m[rt];
      s[rt][0] = s[rt][1] = f32x4{mn, mn, mn, mn};
    }
    R::template qk<RT>(kr, q, s);
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
      if (__any(R::odd(vr))) {
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
    R::template pv<RT>(vr, p, o, both);
    if (more) load_v(kb + 32 * kRowWaves, n);
  }
  // Where V holds an infinity, the part of P that the first leaves is 0 or negative at times, and their sum is NaN: a wave
  // whose O is not finite throughout goes once more over its keys with the first part alone.
  if (both) {
    uint32_t most = 0;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int dt = 0; dt < EPL; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) most = max(most, __float_as_uint(o[rt][dt][i]) & 0x7fffffffu);
    if (__any(most >= 0x7f800000u)) {
      both = false;
      kb = k0 + 32 * wave;
      load_ids(kb);
      load_k(kb, 0);
      load_v(kb, 0);
      goto again;
    }
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

}  // namespace kh
