// Paged attention of many query rows in bfloat16: K and V tiles in LDS, shared by the waves of a workgroup.
//
// A workgroup of WAVES waves takes a tile of 32 WAVES packed rows (token x query head of one kv head, paged.h)
// and one chunk of keys, in LDS tiles of BN keys, double buffered with one barrier per tile; each wave owns 32
// rows, one per lane of a half wave, and works on 64 keys at a time:
//   S^T (64 keys x 32 rows) = K Q^T and O^T += V^T P^T with v_mfma_f32_32x32x16_bf16, K rows stored with bits 2
//   and 3 of the key swapped so that S^T leaves P in the operand layout of the second product, V read
//   transposed (ds_read_b64_tr_b16), the softmax relative to a reference that the accumulators start from
//   (flash_tiles.h) -- the products of the contiguous prefill kernel.
// P is rounded to bf16 once for the second product, as there: these tiles are bound by their products, of which a second
// part of P would make half as many again (2-norm error 2.3e-3, of which the result's rounding is 1.7e-3).
// What differs is where rows come from: 16 keys lie in one page, the threads of a wave that load together
// read inside one such block, so a block's place is a lane's value read as scalars (one lane per block, worked
// out for 1024 keys at once), and its buffer range ends with the page's rows that the tile sees (others, and
// blocks in no page, read as zeros).  K and V pools have equal strides here.
//
// Bound by the chain QK -> exp2 -> PV of each wave and by the uneven last tiles: 2048 tokens of 16384 keys (256-row
// tiles) 280 us a call, 9 of them the merge's = 940 TFLOP/s, 70 % of a large matrix product (a kernel trace, which
// slows it, has 296 to 306 us); 64 sequences' chunks of 300 tokens of 5000 (128-row tiles) 770 TFLOP/s.
#include "paged_rows.h"

using namespace kh;

namespace {

typedef uint32_t v4u32 __attribute__((ext_vector_type(4)));

template <int D, int WAVES, int BN>
struct TileCfg {
  static constexpr int THREADS = WAVES * 64;
  static constexpr int KSTR = D + 8, VSTR = D + 32;  // LDS row strides without bank conflicts (flash_prefill.hip)
  static constexpr int KTILE = BN * KSTR, VTILE = BN * VSTR, STAGE = KTILE + VTILE;
  static constexpr int CPR = D / 8;                  // 16-byte pieces of a row
  static constexpr int RPW = 64 / CPR;               // rows that a wave loads at once
  static constexpr int NK = BN * CPR / THREADS;      // pieces of K (and of V) per thread and tile
  static constexpr int NQ = D / 16, ND = D / 32, NCH = BN / 64;
  static_assert(NK >= 1 && BN % 64 == 0 && THREADS / CPR % 16 == 0, "whole 16-key blocks per load");
};

// Tile `column` / hkv of kv head `column` % hkv (innermost: an XCD's L2 holds few heads) and chunk `split`; smem: 2
// STAGE elements of LDS, odd: whether a wave's V pieces of a staged tile held infinities or NaN.
template <int D, int WAVES, int BN>
__device__ __forceinline__ void paged_tiles(uint16_t* smem, int (&odd)[2][WAVES], int column, int split,
                                            const uint16_t* __restrict__ Q, const uint16_t* __restrict__ K,
                                            const uint16_t* __restrict__ V, uint16_t* __restrict__ O,
                                            const PagedBatch& pb, int hq, int hkv, int G, const PagedStrides& st, float c2,
                                            float sign, int causal, int max_new, int min_rows, int chunk, int chunks,
                                            float* __restrict__ part) {
  using C = TileCfg<D, WAVES, BN>;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 31, g = lane >> 5;
  const int hk = column % hkv;
  const Tile t = find_tile(pb, column / hkv, G, 32 * WAVES, max_new, min_rows, INT32_MAX);
  if (t.b < 0) return;
  const int end = seen_by(t, (min(t.row0 + 32 * WAVES, t.rows) - 1) / G, causal, pb.max_len);
  const int k0 = split * chunk, k1 = min(end, k0 + chunk);
  if (split > 0 && k0 >= end) return;  // (the first chunk of a tile without keys stores zeros)

  // this lane's row, and the keys that the wave's rows see
  const int row0 = t.row0 + 32 * wave;
  const bool there = row0 + r < t.rows;
  const int x = min(row0 + r, t.rows - 1), j = x / G, h = hk * G + x - j * G;
  const int sees = there ? seen_by(t, j, causal, pb.max_len) : 0;
  const int wave_end = row0 < t.rows ? seen_by(t, (min(row0 + 32, t.rows) - 1) / G, causal, pb.max_len) : 0;
  const int all_see = row0 < t.rows ? seen_by(t, row0 / G, causal, pb.max_len) : 0;
  const int tile_sees = seen_by(t, t.row0 / G, causal, pb.max_len);  // what every row of the tile sees

  // A window of 64 blocks of 16 keys, from key k0 + 1024 w, one block per lane: the byte offset of its first row in
  // the pools (K and V alike: their strides are), the bytes from there that the tile may read, and which
  // blocks lie in a page at all; and the page id for the next window.
  const int32_t* table = pb.table + t.b * pb.table_stride;
  auto id_of = [&](int w) {
    const int key = k0 + 1024 * w + 16 * lane;
    return key < k1 ? table[key >> pb.page_log] : -1;
  };
  int64_t offs;
  uint32_t room;
  uint64_t held;
  auto window = [&](int w, int id) {
    const int key = k0 + 1024 * w + 16 * lane, rows = min(16, end - key);
    const bool ok = pb.is_page(id);
    offs = ok ? 2 * ((int64_t)id * st.kp + (int64_t)hk * st.kh + (int64_t)(key & ((1 << pb.page_log) - 1)) * st.kr) : 0;
    room = ok && rows > 0 ? 2u * (uint32_t)((rows - 1) * st.kr + D) : 0u;
    held = __ballot(ok);
  };
  window(0, id_of(0));
  int id_next = k0 + 1024 < k1 ? id_of(1) : -1;
  bf16x8 qreg[C::NQ];
  {
    const uint16_t* q = Q + (int64_t)(t.t0 + j) * st.qt + (int64_t)h * st.qh + 8 * g;
#pragma unroll
    for (int c = 0; c < C::NQ; ++c) qreg[c] = as_bf16x8(*reinterpret_cast<const uint4*>(q + 16 * c));
  }

  // Loads of a tile: piece i of this thread is row `krow` of block wblk + i BSTEP, columns dcol ..
  constexpr int BSTEP = C::THREADS / C::CPR / 16;
  const int wblk = wave * C::RPW / 16, krow = (tid / C::CPR) & 15, dcol = 8 * (tid % C::CPR);
  uint4 kst[C::NK], vst[C::NK];
  const uint32_t mine = 2u * (uint32_t)(krow * st.kr + dcol);
  auto load = [&](int tile) {
#pragma unroll
    for (int i = 0; i < C::NK; ++i) {
      const int blk = (tile * (BN / 16) + wblk + i * BSTEP) & 63;
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)offs, blk), hi = __builtin_amdgcn_readlane((int)(offs >> 32), blk);
      const uint32_t bytes = __builtin_amdgcn_readlane((int)room, blk);
      const int64_t o = (int64_t)(((uint64_t)hi << 32) | lo);
      kst[i] = buf_load16(make_rsrc((const uint8_t*)K + o, bytes), mine);
      vst[i] = buf_load16(make_rsrc((const uint8_t*)V + o, bytes), mine);
    }
  };
  auto swap23 = [](int k) { return (k & ~12) | ((k & 4) << 1) | ((k & 8) >> 1); };
  auto store = [&](int tile) {
    uint16_t* stage = smem + (tile & 1) * C::STAGE;
    if (k0 + (tile + 1) * BN > tile_sees) {  // rows of the tile see different keys of it: `cut` below
      bool any = false;
#pragma unroll
      for (int i = 0; i < C::NK; ++i) {
        const v4u32 u = __builtin_bit_cast(v4u32, vst[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) any = any || (u[k] & 0x7f80u) == 0x7f80u || (u[k] & 0x7f800000u) == 0x7f800000u;
      }
      const bool found = __any(any);
      if (lane == 0) odd[tile & 1][wave] = found;
    }
#pragma unroll
    for (int i = 0; i < C::NK; ++i) {
      const int key = 16 * (wblk + i * BSTEP) + krow;
      *reinterpret_cast<uint4*>(stage + swap23(key) * C::KSTR + dcol) = kst[i];
      *reinterpret_cast<uint4*>(stage + C::KTILE + key * C::VSTR + dcol) = vst[i];
    }
  };

  f32x16 oacc[C::ND];
#pragma unroll
  for (int dt = 0; dt < C::ND; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.f;
  SoftmaxLog2 sl;
  if (!there) sl.m = 0.f;  // (a row that is not there never asks for a raise)
  const int ntiles = (k1 - k0 + BN - 1) / BN;
  constexpr uint32_t kBits = BN == 128 ? 0xffu : 0xfu;
  uint32_t bits = 0;  // which blocks of the current tile lie in a page
  if (ntiles > 0) {
    load(0);
    bits = (uint32_t)held & kBits;
    store(0);
  }
  {
    const uint32_t flip = sign < 0.f ? 0x80008000u : 0u, keep = there && sign != 0.f ? ~0u : 0u;
#pragma unroll
    for (int c = 0; c < C::NQ; ++c) {
      uint4 u = __builtin_bit_cast(uint4, qreg[c]);
      qreg[c] = as_bf16x8(make_uint4((u.x ^ flip) & keep, (u.y ^ flip) & keep, (u.z ^ flip) & keep, (u.w ^ flip) & keep));
    }
  }
  // nothing outstanding before the loop, so that its waits only ever cover the next tile's loads
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();

#pragma unroll 1
  for (int tile = 0; tile < ntiles; ++tile) {
    const bool more = tile + 1 < ntiles;
    uint32_t bits_next = 0;
    if (more) {
      const int blk = (tile + 1) * (BN / 16);
      if ((blk & 63) == 0) {
        window(blk / 64, id_next);
        id_next = id_of(blk / 64 + 1);
      }
      load(tile + 1);
      bits_next = (uint32_t)(held >> (blk & 63)) & kBits;
    }
    const uint16_t* ks = smem + (tile & 1) * C::STAGE;
#pragma unroll
    for (int c = 0; c < C::NCH; ++c) {
      const int kt = k0 + tile * BN + 64 * c;
      if (kt >= wave_end) continue;
      const uint16_t* vs = ks + C::KTILE + 64 * c * C::VSTR;
      // S^T - m
      f32x16 sacc[2];
      mfma_block_begin();
      {
        bf16x8 kf[2 * C::NQ];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint16_t* kp = ks + (64 * c + 32 * s + r) * C::KSTR + 8 * g;
#pragma unroll
          for (int i = 0; i < C::NQ; ++i) kf[s * C::NQ + i] = as_bf16x8(*reinterpret_cast<const uint4*>(kp + 16 * i));
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          sacc[s] = sl.mneg;
#pragma unroll
          for (int i = 0; i < C::NQ; ++i)
            sacc[s] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s * C::NQ + i], qreg[i], sacc[s], 0, 0, 0);
        }
        sched_reads_ahead<2 * C::NQ, 1>();
      }
      mfma_block_end();
      // register i of half s holds key kt + 32 s + 16 (i >> 3) + 8 g + (i & 7)
      const uint32_t pages = (bits >> (4 * c)) & 15u;
      const bool cut = kt + 64 > all_see;  // some row of the wave does not see all 64 keys
      if (cut || pages != 15u) {
        const int lim = sees - kt - 8 * g;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * s + 16 * (i >> 3) + (i & 7) >= lim || !((pages >> (2 * s + (i >> 3))) & 1u)) sacc[s][i] = -INFINITY;
      }
      bf16x8 pk[4];
      float ps = SoftmaxLog2::exponentiate(sacc, c2, pk);
      if (sl.need_raise(ps)) {
        sl.raise(sacc, c2, oacc);
        ps = SoftmaxLog2::exponentiate(sacc, c2, pk);
      }
      sl.l += ps;
      if (cut) {
        // A V row that some of the wave's rows see and others do not may hold infinities or NaN, and 0 times
        // those is not 0: a chunk of a tile that holds any is summed key by key, by the rows that see the key.
        int any = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) any |= odd[tile & 1][i];
        if (__builtin_amdgcn_readfirstlane(any)) {
#pragma unroll 1
          for (int key = 0; key < 64; ++key) {
            uint32_t word = 0;  // the pair of P values that holds the key's
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (k == key >> 4 && e == ((key >> 1) & 3)) word = __builtin_bit_cast(v4u32, pk[k])[e];
            word = __shfl(word, r + 32 * ((key >> 3) & 1), 64);
            const float p = (key & 1) ? hi_bf16(word) : lo_bf16(word);
            if (kt + key < sees && ((pages >> (key >> 4)) & 1u)) {
              const uint16_t* v = vs + key * C::VSTR + 4 * g;
#pragma unroll
              for (int dt = 0; dt < C::ND; ++dt)
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                  const uint2 u = *reinterpret_cast<const uint2*>(v + 32 * dt + 8 * a);
                  oacc[dt][4 * a] += p * lo_bf16(u.x);
                  oacc[dt][4 * a + 1] += p * hi_bf16(u.x);
                  oacc[dt][4 * a + 2] += p * lo_bf16(u.y);
                  oacc[dt][4 * a + 3] += p * hi_bf16(u.y);
                  __builtin_amdgcn_sched_barrier(0);  // (few registers here: the loop's staged rows are live)
                }
            }
          }
          continue;
        }
      }
      // O^T += V^T P^T
      mfma_block_begin();
      {
        const int L = lane & 15, Gq = lane >> 4;
        const uint16_t* vbase = vs + (8 * (Gq >> 1) + (L >> 2)) * C::VSTR + 16 * (Gq & 1) + 4 * (L & 3);
        v8i16 af[C::ND * 4];
#pragma unroll
        for (int dt = 0; dt < C::ND; ++dt)
#pragma unroll
          for (int kc = 0; kc < 4; ++kc) {
            const uint16_t* p0 = vbase + 16 * kc * C::VSTR + 32 * dt;
            const v4i16 lo = lds_read_tr16(p0), hi = lds_read_tr16(p0 + 4 * C::VSTR);
            af[dt * 4 + kc] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          }
#pragma unroll
        for (int dt = 0; dt < C::ND; ++dt)
#pragma unroll
          for (int kc = 0; kc < 4; ++kc)
            oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, af[dt * 4 + kc]), pk[kc], oacc[dt],
                                                               0, 0, 0);
        sched_reads_ahead<C::ND * 4, 2>();
      }
      mfma_block_end();
    }
    if (more) store(tile + 1);
    bits = bits_next;
    __syncthreads();
  }

  const float l = sl.l + __shfl_xor(sl.l, 32, 64);
  if (!there) return;
  // lane: columns 32 dt + 8 a + 4 g + i from register 4 a + i of tile dt
  if (part == nullptr) {
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    uint16_t* o = O + (int64_t)(t.t0 + j) * st.ot + (int64_t)h * st.oh;
#pragma unroll
    for (int dt = 0; dt < C::ND; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        uint2 w;
        w.x = pack_bf16x2(oacc[dt][4 * a] * inv, oacc[dt][4 * a + 1] * inv);
        w.y = pack_bf16x2(oacc[dt][4 * a + 2] * inv, oacc[dt][4 * a + 3] * inv);
        *reinterpret_cast<uint2*>(o + 32 * dt + 8 * a + 4 * g) = w;
      }
  } else {
    const int64_t at = (int64_t)(t.t0 + j) * hq + h;
    float* po = part_o<D>(part, at, chunks, split);
#pragma unroll
    for (int dt = 0; dt < C::ND; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<f32x4*>(po + 32 * dt + 8 * a + 4 * g) =
            f32x4{oacc[dt][4 * a], oacc[dt][4 * a + 1], oacc[dt][4 * a + 2], oacc[dt][4 * a + 3]};
    if (g == 0) part_ml<D>(part, (int64_t)pb.tokens * hq, chunks, at)[split] = make_float2(sl.m, l);
  }
}

template <int D, int WAVES, int BN, int MINB>
__global__ __launch_bounds__(WAVES * 64, MINB) void paged_tiles_kernel(
    const uint16_t* __restrict__ Q, const uint16_t* __restrict__ K, const uint16_t* __restrict__ V,
    uint16_t* __restrict__ O, PagedBatch pb, int hq, int hkv, int G, PagedStrides st, float c2, float sign, int causal,
    int max_new, int min_rows, int chunk, int chunks, float* __restrict__ part) {
  __shared__ __attribute__((aligned(16))) uint16_t smem[2 * TileCfg<D, WAVES, BN>::STAGE];
  __shared__ int odd[2][WAVES];
  paged_tiles<D, WAVES, BN>(smem, odd, blockIdx.x, blockIdx.z, Q, K, V, O, pb, hq, hkv, G, st, c2, sign, causal, max_new,
                            min_rows, chunk, chunks, part);
}

// Sequences of many rows and of few (chunks of prompts beside single tokens) in one launch, so that they run beside
// each other: tiles of 128 rows and of 32.  As two launches one after the other six ragged chunks of up to 300 tokens take
// 91 us, a chunk of 2048 of 8192 beside 31 tokens of 8192 394; together 75 and 275.
template <int D>
__global__ __launch_bounds__(256, 2) void paged_mixed_kernel(const uint16_t* __restrict__ Q,
                                                             const uint16_t* __restrict__ K,
                                                             const uint16_t* __restrict__ V, uint16_t* __restrict__ O,
                                                             PagedBatch pb, int hq, int hkv, int G, PagedStrides st,
                                                             float c2, float sign, int causal, int max_new, int few_rows,
                                                             PagedPart many, PagedPart few, int turn, int chunks,
                                                             float* __restrict__ part) {
  constexpr int TILE = 4 * TileCfg<D, 4, 64>::STAGE, ROWS = 4 * RowLds<uint16_t, D, 2>::FLOATS;
  __shared__ __attribute__((aligned(16))) uint8_t lds[TILE > ROWS ? TILE : ROWS];
  __shared__ int odd[2][4];
  // The two kinds take turns, one of each per CU, as long as both last.  (Chunk of 2048 tokens of 8192 and 31 single
  // tokens of 8192: 263 us, one kind after the other 268, turns of 64 workgroups 293, of 8 303.)
  const int of_many = many.columns * many.used, of_few = few.columns * few.used;
  const int both = min(of_many, of_few) / turn * turn;
  int x = blockIdx.x;
  bool is_many;
  if (x < 2 * both) {
    is_many = (x / turn & 1) == 0;
    x = x / (2 * turn) * turn + x % turn;
  } else {
    is_many = x - both < of_many;
    x -= is_many ? both : of_many;
  }
  if (is_many)
    paged_tiles<D, 4, 64>(reinterpret_cast<uint16_t*>(lds), odd, x % many.columns, x / many.columns, Q, K, V, O, pb, hq, hkv,
                          G, st, c2, sign, causal, max_new, few_rows, many.chunk, chunks, many.used > 1 ? part : nullptr);
  else {
    // (few.columns is a bound: the chunks of a tile side by side leave the workgroups without one to the end)
    const int hk = x % hkv, at = x / hkv;
    paged_rows<uint16_t, D, 2>(reinterpret_cast<float*>(lds), at / few.used * hkv + hk, at % few.used, Q, K, V, O, pb, hq,
                               hkv, G, st, c2, sign, causal, max_new, few_rows, few.chunk, chunks,
                               few.used > 1 ? part : nullptr);
  }
}

template <int D, int WAVES, int BN, int MINB>
void launch_tiles(const PagedCall& c, const PagedPart& many, int chunks, float* part) {
  paged_tiles_kernel<D, WAVES, BN, MINB><<<dim3(many.columns, 1, many.used), WAVES * 64, 0, stream()>>>(
      (const uint16_t*)c.q, (const uint16_t*)c.k, (const uint16_t*)c.v, (uint16_t*)c.o, c.pb, c.hq, c.hkv, c.G, c.st, c.c2,
      c.sign, c.causal, c.max_new, 0, many.chunk, chunks, many.used > 1 ? part : nullptr);
}

template <int D>
void launch_mixed(const PagedCall& c, int few_rows, const PagedPart& many, const PagedPart& few, int chunks, float* part) {
  paged_mixed_kernel<D><<<(unsigned)(many.columns * many.used + few.columns * few.used), 256, 0, stream()>>>(
      (const uint16_t*)c.q, (const uint16_t*)c.k, (const uint16_t*)c.v, (uint16_t*)c.o, c.pb, c.hq, c.hkv, c.G, c.st, c.c2,
      c.sign, c.causal, c.max_new, few_rows, many, few, cu_count(), chunks, part);
}

}  // namespace

namespace kh {

void launch_paged_tiles(const PagedCall& c, int d, int waves, const PagedPart& many, int chunks, float* part) {
  if (d == 128 && waves == 8)
    launch_tiles<128, 8, 128, 1>(c, many, chunks, part);
  else if (d == 128)
    launch_tiles<128, 4, 64, 2>(c, many, chunks, part);
  else if (waves == 8)
    launch_tiles<64, 8, 128, 1>(c, many, chunks, part);
  else
    launch_tiles<64, 4, 64, 2>(c, many, chunks, part);
}

void launch_paged_mixed(const PagedCall& c, int d, int few_rows, const PagedPart& many, const PagedPart& few, int chunks,
                        float* part) {
  if (d == 128)
    launch_mixed<128>(c, few_rows, many, few, chunks, part);
  else
    launch_mixed<64>(c, few_rows, many, few, chunks, part);
}

}  // namespace kh
