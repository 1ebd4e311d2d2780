// What the bf16 MFMA attention kernels share (flash_prefill.hip, paged_tiles.hip): the operand reads of
// v_mfma_f32_32x32x16_bf16 products of key-major LDS tiles, and the online softmax of their scores.
#pragma once

#include "common.h"

namespace kh {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kXcds = 8;  // MI355X: accelerator complex dies, one L2 each

__device__ __forceinline__ bf16x8 as_bf16x8(uint4 v) { return __builtin_bit_cast(bf16x8, v); }

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef short v8i16 __attribute__((ext_vector_type(8)));

// gfx950 ds_read_b64_tr_b16: within each 16-lane group, element k of lane j is element (j & 3)
// of the four bf16 at the address of lane 4k + (j >> 2).
__device__ __forceinline__ v4i16 lds_read_tr16(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(p));
}

// Operand reads of a block of NM MFMAs (RPM LDS reads each): the reads of the first kReadsAhead
// MFMAs are issued first and each MFMA is followed by the reads of the one kReadsAhead places later,
// so several operands are in flight while the matrix core works (the default schedule keeps one or
// two).  Placed after the block's code; it orders the DS reads and MFMAs of the basic block.
constexpr int kReadsAhead = 4;
template <int NM, int RPM>
__device__ __forceinline__ void sched_reads_ahead() {
  constexpr int AHEAD = kReadsAhead < NM ? kReadsAhead : NM;
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * RPM, 0);  // DS reads
#pragma unroll
  for (int i = 0; i < NM - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);          // one MFMA
    __builtin_amdgcn_sched_group_barrier(0x100, RPM, 0);        // the reads of a later one
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// The two waves of a SIMD alternate between MFMA blocks (QK^T, PV) and softmax VALU work; a wave
// raises its issue priority for its MFMA blocks, so the arbiter keeps the matrix core fed while the
// other wave's VALU work fills the issue slots in between (C3: +0.5-1 %; priority on the QK^T
// block alone -0.4 %, on PV alone -3 %).
__device__ __forceinline__ void mfma_block_begin() { __builtin_amdgcn_s_setprio(1); }
__device__ __forceinline__ void mfma_block_end() { __builtin_amdgcn_s_setprio(0); }

// Row maximum of a chunk's scores: this lane's 32, then the partner lane (lane ^ 32) that holds
// the other 32 keys of the same query row.
template <int NSUB>
__device__ __forceinline__ float chunk_row_max(const f32x16 (&sc)[NSUB]) {
  float m4[NSUB * 4];
#pragma unroll
  for (int s = 0; s < NSUB; ++s)
#pragma unroll
    for (int j = 0; j < 16; j += 4)
      m4[s * 4 + j / 4] = fmaxf(fmaxf(sc[s][j], sc[s][j + 1]), fmaxf(sc[s][j + 2], sc[s][j + 3]));
  float mx = m4[0];
#pragma unroll
  for (int i = 1; i < NSUB * 4; ++i) mx = fmaxf(mx, m4[i]);
  return fmaxf(mx, __shfl_xor(mx, 32, 64));
}

// Online softmax of the causal / unmasked route: raw q.k scores relative to the reference maximum m
// (the QK^T accumulators start at mneg = -m, 0 before the first raise); P = 2^(c (s - m)) with
// c = scale log2 e.
constexpr float kSumMax = 4096.f;  // a lane's chunk sum of P above this raises the reference

struct SoftmaxLog2 {
  float m = -INFINITY;  // reference maximum of this row (raw q.k units); -inf before the first raise
  float l = 0.f;        // partial denominator of this lane's keys, relative to m
  f32x16 mneg;          // -m in every register (0 while m = -inf)

  __device__ __forceinline__ SoftmaxLog2() {
#pragma unroll
    for (int j = 0; j < 16; ++j) mneg[j] = 0.f;
  }
  // P = 2^(c sc) as bf16 operands; returns this lane's sum of those bf16 values (two per
  // v_dot2c_f32_bf16 against (1, 1)): l then sums exactly the weights the PV product applies.
  template <int NSUB>
  static __device__ __forceinline__ float exponentiate(const f32x16 (&sc)[NSUB], float c, bf16x8 (&pk)[2 * NSUB]) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
    float ps[2 * NSUB];
#pragma unroll
    for (int s = 0; s < NSUB; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bf16x8 pv;
#pragma unroll
        for (int e = 0; e < 8; ++e) pv[e] = (__bf16)fast_exp2(sc[s][8 * h + e] * c);
        pk[2 * s + h] = pv;
        const bf16x2 p01 = __builtin_shufflevector(pv, pv, 0, 1), p23 = __builtin_shufflevector(pv, pv, 2, 3);
        const bf16x2 p45 = __builtin_shufflevector(pv, pv, 4, 5), p67 = __builtin_shufflevector(pv, pv, 6, 7);
        float sum = __builtin_amdgcn_fdot2_f32_bf16(p01, one, 0.f, false);
        sum = __builtin_amdgcn_fdot2_f32_bf16(p23, one, sum, false);
        sum = __builtin_amdgcn_fdot2_f32_bf16(p45, one, sum, false);
        ps[2 * s + h] = __builtin_amdgcn_fdot2_f32_bf16(p67, one, sum, false);
      }
    float t = ps[0];
#pragma unroll
    for (int i = 1; i < 2 * NSUB; ++i) t += ps[i];
    return t;
  }
  // True (wave-uniform) if some row of the wave must raise its reference: the first chunk, or a
  // lane sum above kSumMax (inf included).
  __device__ __forceinline__ bool need_raise(float ps) const {
    return __any(m == -INFINITY || !(ps <= kSumMax));
  }
  // Raises every row's reference to its exact maximum over the chunk (when higher), shifts the
  // chunk's scores to the new reference and rescales O and l.  A row with nothing unmasked so far
  // keeps m = -inf (and P = 0).
  template <int NSUB, int ND>
  __device__ __forceinline__ void raise(f32x16 (&sc)[NSUB], float c, f32x16 (&oacc)[ND]) {
    const float mx = chunk_row_max(sc);  // relative to m (absolute while m = -inf)
    float d, alpha;
    if (m == -INFINITY) {
      d = mx == -INFINITY ? 0.f : mx;
      alpha = 0.f;  // O and l are still empty
      m = mx;
    } else {
      d = fmaxf(mx, 0.f);
      alpha = fast_exp2(-d * c);
      m += d;
    }
#pragma unroll
    for (int s = 0; s < NSUB; ++s)
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[s][j] -= d;
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int j = 0; j < 16; ++j) oacc[dt][j] *= alpha;
    const float mn = m == -INFINITY ? 0.f : -m;
#pragma unroll
    for (int j = 0; j < 16; ++j) mneg[j] = mn;
  }
};

}  // namespace kh
