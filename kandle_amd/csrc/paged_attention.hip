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

#include "paged.h"

using namespace kh;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSumMax = 4096.f;  // a lane's sum of P above this raises the reference maximum

struct PagedStrides {
  int64_t qt, qh, kp, kh, kr, vp, vh, vr, ot, oh;
};

// The (sequence, tile) of workgroup column x of a grid over tiles of `rows` packed rows: sequence b has
// ceil(min(n_b, max_new) * G / rows) tiles.  Every wave of the workgroup computes it for itself.
struct Tile {
  int b = -1, row0 = 0, rows = 0;  // first packed row, packed rows of the sequence
  int t0 = 0, n = 0, len = 0;      // first token, new tokens, cached rows
};
__device__ __forceinline__ Tile find_tile(const PagedBatch& pb, int x, int G, int rows, int max_new) {
  Tile t;
  int at = x;
  if (pb.starts == nullptr) {
    const int per = (G + rows - 1) / rows;
    t.b = x / per;
    at = x - t.b * per;
    if (t.b >= pb.batch) t.b = -1;
  } else {
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < pb.batch; b0 += 64) {
      const int b = b0 + lane;
      const int n = b < pb.batch ? min(pb.count(b), max_new) : 0;
      const int tiles = (int)(((int64_t)n * G + rows - 1) / rows);
      int inc = tiles;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(inc, o, 64);
        if (lane >= o) inc += u;
      }
      const int all = __shfl(inc, 63, 64);
      if (at < all) {
        const int who = __ffsll((unsigned long long)__ballot(inc > at)) - 1;
        at -= __shfl(inc - tiles, who, 64);
        t.b = b0 + who;
        break;
      }
      at -= all;
    }
  }
  t.b = __builtin_amdgcn_readfirstlane(t.b);
  if (t.b < 0) return t;
  at = __builtin_amdgcn_readfirstlane(at);
  t.t0 = pb.first(t.b);
  t.n = pb.count(t.b);
  t.len = pb.len(t.b);
  t.row0 = at * rows;
  t.rows = min(t.n, max_new) * G;
  return t;
}

// Keys that token j of the tile's sequence sees: those below the result (holes apart).
__device__ __forceinline__ int seen_by(const Tile& t, int j, int causal, int max_len) {
  return min(max_len, causal ? max(0, t.len - t.n + j + 1) : t.len);
}

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
  static __device__ __forceinline__ void load_q(Q& q, const uint16_t* row, int lq, bool there, float sign) {
    const uint32_t flip = sign < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int c = 0; c < NK; ++c) {
      uint4 u = there ? *reinterpret_cast<const uint4*>(row + 32 * c + 8 * lq) : make_uint4(0, 0, 0, 0);
      u.x ^= flip;
      u.y ^= flip;
      u.z ^= flip;
      u.w ^= flip;
      q.v[c] = __builtin_bit_cast(bf16x8, u);
    }
  }
  static __device__ __forceinline__ void load_k(K& k, __amdgpu_buffer_rsrc_t r, uint32_t off, int lq) {
#pragma unroll
    for (int c = 0; c < NK; ++c) k.v[c] = buf_load16_nt(r, off + 64 * c + 16 * lq);
  }
  static __device__ __forceinline__ void load_v(VRow& v, __amdgpu_buffer_rsrc_t r, uint32_t off) {
    if constexpr (EPL == 8)
      v = buf_load16_nt(r, off);
    else
      v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 2));
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
  static __device__ __forceinline__ void load_q(Q& q, const float* row, int lq, bool there, float sign) {
#pragma unroll
    for (int c = 0; c < NK; ++c) {
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
      q.v[c] = there ? *reinterpret_cast<const f32x4*>(row + 16 * c + 4 * lq) * sign : z;
    }
  }
  static __device__ __forceinline__ void load_k(K& k, __amdgpu_buffer_rsrc_t r, uint32_t off, int lq) {
#pragma unroll
    for (int c = 0; c < NK; ++c) k.v[c] = __builtin_bit_cast(f32x4, buf_load16_nt(r, off + 64 * c + 16 * lq));
  }
  static __device__ __forceinline__ void load_v(VRow& v, __amdgpu_buffer_rsrc_t r, uint32_t off) {
#pragma unroll
    for (int i = 0; i < EPL / 4; ++i) v.v[i] = __builtin_bit_cast(f32x4, buf_load16_nt(r, off + 16 * i));
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

// Partials of chunk s of packed row x of sequence b: its (token, head) pair's row in `part`, chunk s.
// O relative to m (not divided by l), then m (raw units) and l.
template <int D>
__device__ __forceinline__ float* part_o(float* part, int64_t row, int chunks, int s) {
  return part + (row * chunks + s) * D;
}
template <int D>
__device__ __forceinline__ float2* part_ml(float* part, int64_t all_rows, int chunks, int64_t row, int s) {
  return reinterpret_cast<float2*>(part + all_rows * chunks * D) + row * chunks + s;
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(kRowWaves * 64, sizeof(T) == 4 && D == 128 ? 1 : 2) void paged_rows_kernel(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, T* __restrict__ O, PagedBatch pb, int hq,
    int G, PagedStrides st, float c2, float sign, int causal, int max_new, int chunk, int chunks, float* __restrict__ part) {
  using R = RowOps<T, D>;
  constexpr int EPL = R::EPL;
  constexpr int MS = 2 + 4 * EPL;  // floats per lane and row tile that the waves exchange
  __shared__ float join[(kRowWaves - 1) * RT * MS * 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, lq = lane >> 4;
  const int hk = blockIdx.y, split = blockIdx.z;
  const Tile t = find_tile(pb, blockIdx.x, G, 16 * RT, max_new);
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
    const int x = t.row0 + 16 * rt + r, j = x / G, h = hk * G + x - j * G;
    there[rt] = x < t.rows;
    sees[rt] = there[rt] ? seen_by(t, j, causal, pb.max_len) : 0;
    at[rt] = (int64_t)(t.t0 + j) * hq + h;
    R::load_q(q[rt], Q + (int64_t)(t.t0 + j) * st.qt + (int64_t)h * st.qh, lq, there[rt] && sign != 0.f, sign);
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
  // The two halves of the block at key kb: their page's rows as far as keys below `end` go; a half in no
  // page, or behind `end`, reads as zeros.
  auto rsrc = [&](const T* base, int64_t sp, int64_t sh, int64_t sr, int key, bool* in) {
    int id = -1;
    if (key < end) id = table[key >> pb.page_log];
    id = __builtin_amdgcn_readfirstlane(id);
    const bool ok = pb.is_page(id);
    *in = ok;
    const int rows = ok ? min(16, end - key) : 0;
    const T* p = base + (int64_t)(ok ? id : 0) * sp + (int64_t)hk * sh + (int64_t)(key & page_mask) * sr;
    return make_rsrc(p, rows > 0 ? (uint32_t)(((int64_t)(rows - 1) * sr + D) * sizeof(T)) : 0u);
  };
  auto load_k = [&](int kb) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto rk = rsrc(K, st.kp, st.kh, st.kr, kb + 16 * h, &held[h]);
      R::load_k(kr[h], rk, (uint32_t)(r * st.kr * sizeof(T)), lq);
    }
  };
  auto load_v = [&](int kb) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bool in;
      const auto rv = rsrc(V, st.vp, st.vh, st.vr, kb + 16 * h, &in);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        R::load_v(vr[4 * h + i], rv, (uint32_t)(((4 * lq + i) * st.vr + EPL * r) * sizeof(T)));
    }
  };
  int kb = k0 + 32 * wave;
  if (kb < k1) {
    load_k(kb);
    load_v(kb);
  }
#pragma unroll 1
  for (; kb < k1; kb += 32 * kRowWaves) {
    f32x4 s[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float mn = m[rt] == -INFINITY ? 0.f : -m[rt];
#pragma unroll
      for (int h = 0; h < 2; ++h) s[rt][h] = R::qk(kr[h], q[rt], f32x4{mn, mn, mn, mn});
    }
    const bool hole0 = !held[0], hole1 = !held[1];
    const bool more = kb + 32 * kRowWaves < k1;
    if (more) load_k(kb + 32 * kRowWaves);
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
    if (more) load_v(kb + 32 * kRowWaves);
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
      if (lq == 0) *part_ml<D>(part, (int64_t)pb.tokens * hq, chunks, at[rt], split) = make_float2(mt, lt);
    }
  }
}

// Joins a row's chunks in order: a wave per (token, query head).
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(float* __restrict__ part, T* __restrict__ O, PagedBatch pb,
                                                          int hq, PagedStrides st, float c2, int causal, int max_new,
                                                          int chunk, int chunks) {
  constexpr int E = D / 64;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= (int64_t)pb.tokens * hq) return;
  const int tok = (int)(row / hq), h = (int)(row - (int64_t)tok * hq);
  Tile t;
  t.b = pb.sequence_of(tok);
  if (t.b < 0) return;
  t.n = pb.count(t.b);
  t.len = pb.len(t.b);
  const int j = tok - pb.first(t.b);
  if (j >= max_new) return;
  const int seen = seen_by(t, j, causal, pb.max_len), ns = min(chunks, (seen + chunk - 1) / chunk);
  float m = -INFINITY;
  for (int s = lane; s < ns; s += 64) m = fmaxf(m, part_ml<D>(part, (int64_t)pb.tokens * hq, chunks, row, s)->x);
  m = wave_max(m);
  float o[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int s = 0; s < ns; ++s) {
    const float2 ml = *part_ml<D>(part, (int64_t)pb.tokens * hq, chunks, row, s);
    if (ml.x == -INFINITY && ml.y == 0.f) continue;
    const float a = fast_exp2((ml.x - m) * c2);
    const float* p = part_o<D>(part, row, chunks, s) + E * lane;
    l += a * ml.y;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += a * p[e];
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) Elem<T>::store(O + tok * st.ot + h * st.oh, E * lane + e, o[e] * inv);
}

struct Call {
  const void *q, *k, *v;
  void* o;
  PagedBatch pb;
  int hq, hkv, G;
  PagedStrides st;
  float c2, sign;  // |scale| log2 e, and the scale's sign, which goes to the queries; scale 0: 1 and queries of 0
  int causal, max_new;
};

// Workgroup columns that cover every tile of `rows` packed rows, whatever the starts hold.
int64_t tiles_of(const Call& c, int rows) {
  const int64_t per = ((int64_t)c.max_new * c.G + rows - 1) / rows;
  const int64_t all = (int64_t)c.pb.tokens * c.G / rows + c.pb.batch;
  return c.pb.starts == nullptr || per * c.pb.batch < all ? per * c.pb.batch : all;
}

template <typename T, int D, int RT>
int launch_rows(const Call& c) {
  const int64_t tiles = tiles_of(c, 16 * RT);
  // chunks of keys: enough workgroups for the chip, at least 128 keys (a block for each wave) in each
  int chunk = 128;
  const int64_t want = 8 * (int64_t)cu_count();
  while (chunk < c.pb.max_len && tiles * c.hkv * ((c.pb.max_len + chunk - 1) / chunk) > want) chunk *= 2;
  const int chunks = c.pb.max_len > chunk ? (c.pb.max_len + chunk - 1) / chunk : 1;
  KH_REQUIRE(tiles <= INT32_MAX && c.hkv <= 65535 && chunks <= 65535, "kh_paged_attention: too many tiles");
  float* part = nullptr;
  const int64_t rows = (int64_t)c.pb.tokens * c.hq;
  if (chunks > 1) {
    part = (float*)scratch_alloc((size_t)rows * chunks * (D + 2) * 4);
    if (part == nullptr) return KH_ERR_OOM;
  }
  paged_rows_kernel<T, D, RT><<<dim3((unsigned)tiles, c.hkv, chunks), kRowWaves * 64, 0, stream()>>>(
      (const T*)c.q, (const T*)c.k, (const T*)c.v, (T*)c.o, c.pb, c.hq, c.G, c.st, c.c2, c.sign, c.causal, c.max_new, chunk, chunks,
      part);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && part) {
    paged_merge_kernel<T, D><<<(unsigned)((rows + 3) / 4), 256, 0, stream()>>>(
        part, (T*)c.o, c.pb, c.hq, c.st, c.c2, c.causal, c.max_new, chunk, chunks);
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

template <typename T, int D>
int launch(const Call& c) {
  if ((int64_t)c.max_new * c.G <= 16) return launch_rows<T, D, 1>(c);
  return launch_rows<T, D, 2>(c);
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
  KH_REQUIRE(hkv <= 65535, "kh_paged_attention: %d kv heads are too many", hkv);
  KH_REQUIRE(d == 64 || d == 128, "kh_paged_attention: head_dim %d not supported (64 or 128)", d);
  KH_REQUIRE(dtype == KH_BF16 || dtype == KH_F32, "kh_paged_attention: unsupported dtype %d", dtype);
  KH_REQUIRE(max_query_len >= 0, "kh_paged_attention: negative max_query_len");
  KH_REQUIRE(scale - scale == 0.f, "kh_paged_attention: the scale is not finite");
  Call c;
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
