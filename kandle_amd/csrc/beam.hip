// The selection of a beam search step (kh_beam_select): the k best continuations of every group of beams
// over beams x vocabulary.
//
//   score(beam, token) = logits[beam, token] - log sum exp(logits[beam, :]) + scores[beam]
// A finished beam has one continuation: itself, with the end token.  NaN, as a logit or a score, counts
// as -inf.  Order: the larger score in float64, then the lower beam, then the larger logit, then the lower token.  A
// beam's scores never fall as its logits grow (where its score so far is large, different logits make one score),
// so inside a beam the logits decide, and only the k largest of each are scored.
#include "paged.h"

using namespace kh;

namespace {

constexpr int kMaxK = 64;
constexpr int kMaxBeams = 64;
constexpr float kLog2e = 1.4426950408889634f;

// Order-preserving bits (-0 as +0), above 0 for every number: 0 stands for no candidate.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ uint64_t order_bits(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x == 0.0 ? 0.0 : x);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double order_value(uint64_t u) {
  return __longlong_as_double((long long)((u >> 63) ? (u & 0x7fffffffffffffffull) : ~u));
}
__device__ __forceinline__ float no_nan(float x) { return fmaxf(x, -INFINITY); }

// A logit's key inside its beam: the larger logit first, then the lower id.
__device__ __forceinline__ uint64_t order_key(float x, int id) {
  return ((uint64_t)order_bits(x) << 32) | (uint64_t)(0xffffffffu - (uint32_t)id);
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor(v, o, 64);
    v = u > v ? u : v;
  }
  return v;
}
__device__ __forceinline__ float wave_max_dpp(float v) {
  v = fmaxf(v, dpp_f<0xB1>(v));
  v = fmaxf(v, dpp_f<0x4E>(v));
  v = fmaxf(v, dpp_f<0x141>(v));
  v = fmaxf(v, dpp_f<0x140>(v));
  const int b = __builtin_bit_cast(int, v);
  return fmaxf(fmaxf(__builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 0)), __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 16))),
               fmaxf(__builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 32)), __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 48))));
}
// Place of this lane among those whose bit is set in `who`.
__device__ __forceinline__ int place_in(uint64_t who) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
}

// The selections below start from the k-th largest of the 64 lanes' maxima: k candidates are at least as large, so
// nothing below it is among the k largest, and a handful above it are left, which are ranked by counting.
// It is found bit by bit with ballots, and may be left lower as soon as exactly k lanes are above.  Where more
// than kRoom candidates are left (many equal values), k rounds of a wave-wide maximum do the same.
constexpr int kRoom = 128;
__device__ __forceinline__ uint32_t kth_lane(uint32_t top, int k) {
  uint32_t floor = 0;
  for (int b = 31; b >= 0; --b) {
    const uint32_t t = floor | (1u << b);
    const int n = __popcll(__ballot(top >= t));
    if (n >= k) floor = t;
    if (n == k) break;
  }
  return floor;
}

// A candidate of the merge: the larger `hi` (order bits of a float64 score) first, then the lower `at`: beam, inverted
// order bits of the logit, and place among the beam's candidates, of which those of equal logits lie in the order of
// their tokens (6, 32 and 24 bits: 64 beams of 2^18 runs of 64 candidates).  hi 0: none.
struct Cand {
  uint64_t hi, at;
};
__device__ __forceinline__ uint64_t cand_at(int beam, uint32_t logit_bits, int place) {
  return (uint64_t)beam << 56 | (uint64_t)~logit_bits << 24 | (uint64_t)place;
}
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.hi > b.hi || (a.hi == b.hi && a.at < b.at); }

// The k best of a wave's candidates, N per lane in registers, in order to out[0 .. k) (LDS; none behind the
// last); `room` is the wave's own LDS for kRoom candidates.
template <int N>
__device__ __forceinline__ void wave_best(Cand (&c)[N], int k, Cand* room, Cand* out) {
  const int lane = threadIdx.x & 63;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, (uint32_t)(c[i].hi >> 32));
  const uint32_t floor = kth_lane(top, k);
  int count = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool keep = c[i].hi != 0 && (uint32_t)(c[i].hi >> 32) >= floor;
    const uint64_t who = __ballot(keep);
    if (who != 0) {
      const int at = count + place_in(who);
      if (keep && at < kRoom) room[at] = c[i];
      count += __popcll(who);
    }
  }
  __builtin_amdgcn_wave_barrier();
  if (count <= kRoom) {
    for (int j = lane; j < k; j += 64) out[j] = Cand{0, 0};
    __builtin_amdgcn_wave_barrier();
    for (int j = lane; j < count; j += 64) {
      const Cand mine = room[j];
      int rank = 0;
#pragma unroll 8
      for (int i = 0; i < count; ++i) rank += before(room[i], mine);
      if (rank < k) out[rank] = mine;
    }
  } else {
    for (int j = 0; j < k; ++j) {
      Cand best{0, 0};
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c[i].hi != 0 && (best.hi == 0 || before(c[i], best))) best = c[i];
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const Cand u{__shfl_xor(best.hi, o, 64), __shfl_xor(best.at, o, 64)};
        if (u.hi != 0 && (best.hi == 0 || before(u, best))) best = u;
      }
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c[i].hi == best.hi && c[i].at == best.at) c[i].hi = 0;
      if (lane == 0) out[j] = best;
    }
  }
  __builtin_amdgcn_wave_barrier();
}

// A workgroup takes a run of 8192 logits of one row, 32 per lane in registers: their maximum, the sum of
// exponentials relative to it, and the k largest in order.  Rows may start anywhere: the lanes' 16-byte loads
// lie on the 16-byte grid of the memory, and those that cross a row's ends are made value by value.
//
// Bound by the chain load -> maximum -> threshold -> ranking of waves that all start together: 128 rows of 151936 bf16
// logits, of which a quarter have finished, 16 us (29 MB), in which a wave waits 60 % of its time and the vector ALU (13.5
// instructions per logit, four of them the exponential's) is busy for half; four fp32 rows, 76 workgroups, 7.8.  Runs of
// twice the length in as many registers are slower (22.4 -> 25.3 us a call): fewer waves hide the chain.
constexpr int kPer = 32, kRunWaves = 4, kRun = kPer * 64 * kRunWaves;
template <typename T>
__global__ __launch_bounds__(kRunWaves * 64) void beam_runs_kernel(const T* __restrict__ logits, int64_t sg, int64_t sb,
                                                                   int beams, int vocab,
                                                                   const int32_t* __restrict__ finished, int k, int runs,
                                                                   float2* __restrict__ sums, uint64_t* __restrict__ keys) {
  constexpr int E = 16 / sizeof(T);
  __shared__ uint64_t room[kRunWaves][kRoom];
  __shared__ uint64_t best[kRunWaves * kMaxK];
  __shared__ float2 part[kRunWaves];
  const int row = blockIdx.y, run = blockIdx.x, lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (finished && finished[row] != 0) return;
  const T* x = logits + (int64_t)(row / beams) * sg + (int64_t)(row % beams) * sb;
  const int shift = (int)(((uintptr_t)x & 15) / sizeof(T));
  const int start = run * kRun + w * (kRun / kRunWaves) + lane * E - shift;  // id of the lane's first value
  float v[kPer];
#pragma unroll
  for (int j = 0; j < kPer / E; ++j) {
    const int id = start + j * 64 * E;
    if (id >= 0 && id + E <= vocab) {
      const uint4 u = *reinterpret_cast<const uint4*>(x + id);
      if constexpr (E == 4) {
        v[4 * j] = __uint_as_float(u.x);
        v[4 * j + 1] = __uint_as_float(u.y);
        v[4 * j + 2] = __uint_as_float(u.z);
        v[4 * j + 3] = __uint_as_float(u.w);
      } else {
        float f[8];
        unpack_bf16x8(u, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * j + e] = f[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[E * j + e] = id + e >= 0 && id + e < vocab ? Elem<T>::load(x, id + e) : -INFINITY;
    }
  }
  // id of value i; values behind the row's end are -inf like some inside it, and told apart by it
  auto id_of = [&](int i) { return start + (i / E) * 64 * E + i % E; };
  float mine = -INFINITY;  // (a maximum passes over NaN)
#pragma unroll
  for (int i = 0; i < kPer; ++i) mine = __builtin_fmaxf(mine, v[i]);
  const float m = wave_max_dpp(mine);
  // (-inf at least: what kth_lane leaves may lie below it, where the bits are a NaN's)
  const float floor = order_value(max(kth_lane(order_bits(mine), k), order_bits(-INFINITY)));
  auto sum = [&] {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) s += fast_exp2((v[i] - m) * kLog2e);
    return wave_sum(s);
  };
  float s = m > -INFINITY ? sum() : 0.f;
  // NaN counts as -inf, which matters where the sum has found one or -inf is among the k largest
  if (s != s || floor == -INFINITY) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = no_nan(v[i]);
    s = m > -INFINITY ? sum() : 0.f;
  }
  if (lane == 0) part[w] = make_float2(m, s);
  // the wave's k best as order keys, in order
  uint64_t* out = best + w * k;
  int count = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    bool keep = v[i] >= floor;
    if (__ballot(keep) != 0) {
      const int id = id_of(i);
      keep = keep && id >= 0 && id < vocab;
      const uint64_t who = __ballot(keep);
      const int at = count + place_in(who);
      if (keep && at < kRoom) room[w][at] = order_key(v[i], id);
      count += __popcll(who);
    }
  }
  for (int j = lane; j < k; j += 64) out[j] = 0;
  __builtin_amdgcn_wave_barrier();
  if (count <= kRoom) {
    for (int j = lane; j < count; j += 64) {
      const uint64_t key = room[w][j];
      int rank = 0;
#pragma unroll 8
      for (int i = 0; i < count; ++i) rank += room[w][i] > key;
      if (rank < k) out[rank] = key;
    }
  } else {
    uint64_t last = ~0ull;  // the one chosen last
    for (int j = 0; j < k; ++j) {
      uint64_t top = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int id = id_of(i);
        const uint64_t key = id >= 0 && id < vocab ? order_key(v[i], id) : 0;
        if (key < last && key > top) top = key;
      }
      last = wave_max_u64(top);
      if (lane == 0) out[j] = last;
      if (last == 0) break;
    }
  }
  __syncthreads();
  const int64_t o = (int64_t)row * runs + run;
  if (threadIdx.x == 0) {
    float mm = part[0].x, ss = 0.f;
#pragma unroll
    for (int i = 1; i < kRunWaves; ++i) mm = fmaxf(mm, part[i].x);
#pragma unroll
    for (int i = 0; i < kRunWaves; ++i)
      if (part[i].x > -INFINITY) ss += part[i].y * fast_exp2((part[i].x - mm) * kLog2e);
    sums[o] = make_float2(mm, ss);
  }
  // the waves' best joined: each is ranked among all (keys differ, but for the zeros behind the last)
  for (int j = threadIdx.x; j < kRunWaves * k; j += kRunWaves * 64) {
    const uint64_t key = best[j];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < kRunWaves * k; ++i) rank += best[i] > key || (best[i] == key && i < j);
    if (rank < k) keys[o * k + rank] = key;
  }
}

// A workgroup per group: the sums of its beams, then the k best of the runs' candidates, scored in float64.  Latency:
// 5.1 us for one group of four beams, 7.1 for sixteen groups of eight (1216 candidates each).
constexpr int kMergeWaves = 16, kSlots = 2;
__global__ __launch_bounds__(kMergeWaves * 64) void beam_merge_kernel(
    const float2* __restrict__ sums, const uint64_t* __restrict__ keys, const float* __restrict__ scores,
    const int32_t* __restrict__ finished, int beams, int vocab, int k, int runs, int eos, float* __restrict__ out_scores,
    int32_t* __restrict__ out_tokens, int32_t* __restrict__ out_parents, int32_t* __restrict__ out_finished) {
  __shared__ double base[kMaxBeams];  // scores[beam] - log sum exp, or NaN where all the beam's scores are -inf
  __shared__ int done[kMaxBeams];
  __shared__ Cand room[kMergeWaves][kRoom];
  __shared__ Cand best[kMergeWaves * kMaxK];
  const int g = blockIdx.x, lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = runs * k, all = beams * per;  // candidates (below 2^31: 64 beams, 2^18 runs, 64 each)
  // the first candidates are under way beside the sums
  uint64_t ahead[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i)
    ahead[i] = keys[(int64_t)g * all + min((w * kSlots + i) * 64 + lane, all - 1)];
  for (int b = w; b < beams; b += kMergeWaves) {
    const int row = g * beams + b;
    const double sc = (double)scores[row];
    const bool fin = finished && finished[row] != 0;
    double v = sc;
    if (!fin) {
      float m = -INFINITY;
      for (int r = lane; r < runs; r += 64) m = fmaxf(m, sums[(int64_t)row * runs + r].x);
      m = wave_max(m);
      double s = 0.0;
      for (int r = lane; r < runs; r += 64) {
        const float2 ms = sums[(int64_t)row * runs + r];
        if (ms.x > -INFINITY) s += (double)ms.y * exp((double)ms.x - (double)m);
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
      v = sc - ((double)m + log(s));
    }
    if (lane == 0) {
      base[b] = v == v && v > -INFINITY && v < INFINITY ? v : __builtin_nan("");
      done[b] = fin;
    }
  }
  __syncthreads();
  Cand* mine = best + w * k;
  for (int j = lane; j < k; j += 64) mine[j] = Cand{0, 0};
  for (int64_t i0 = 0; i0 < all; i0 += kMergeWaves * 64 * kSlots) {
    Cand c[kSlots + 1];
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int64_t at = i0 + (int64_t)(w * kSlots + i) * 64 + lane;
      c[i] = Cand{0, 0};
      if (at < all) {
        const int b = (int)at / per, n = (int)at - b * per;
        if (done[b]) {
          if (n == 0) c[i] = Cand{order_bits(base[b] == base[b] ? base[b] : -(double)INFINITY), cand_at(b, 0, 0)};
        } else if (base[b] != base[b]) {  // (at -inf the logits count as equal: the first tokens)
          if (n < k && n < vocab) c[i] = Cand{order_bits(-(double)INFINITY), cand_at(b, 0, n)};
        } else {
          const uint64_t key = i0 == 0 ? ahead[i] : keys[(int64_t)g * all + at];
          const uint32_t logit = (uint32_t)(key >> 32);
          if (key != 0) c[i] = Cand{order_bits((double)order_value(logit) + base[b]), cand_at(b, logit, n)};
        }
      }
    }
    c[kSlots] = lane < k ? mine[lane] : Cand{0, 0};  // the best so far
    wave_best<kSlots + 1>(c, k, room[w], mine);
  }
  __syncthreads();
  // the waves' best ranked among all, sixteen lanes to each
  for (int j = threadIdx.x / 16; j < kMergeWaves * k; j += kMergeWaves * 4) {
    const Cand u = best[j];
    const int b = (int)(u.at >> 56), n = (int)(u.at & 0xffffff);
    int t = done[b] ? eos : n;  // (a beam at -inf: its first tokens)
    if (u.hi != 0 && !done[b] && base[b] == base[b]) t = (int)(0xffffffffu - (uint32_t)keys[(int64_t)g * all + b * per + n]);
    int rank = 0;
    if (u.hi != 0)
#pragma unroll 4
      for (int i = threadIdx.x & 15; i < kMergeWaves * k; i += 16) rank += before(best[i], u);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) rank += __shfl_xor(rank, off, 16);
    if (u.hi == 0 || rank >= k || (threadIdx.x & 15) != 0) continue;
    const int o = g * k + rank;
    out_scores[o] = (float)order_value(u.hi);
    out_tokens[o] = t;
    out_parents[o] = b;
    if (out_finished) out_finished[o] = (done[b] || t == eos) ? 1 : 0;
  }
}

}  // namespace

extern "C" {

int kh_beam_select(const void* logits, const int64_t* strides, const float* scores, const int32_t* finished, int64_t groups,
                   int64_t beams, int64_t vocab, int k, int64_t eos, float* out_scores, int32_t* out_tokens,
                   int32_t* out_parents, int32_t* out_finished, int dtype) {
  KH_REQUIRE_INIT();
  KH_REQUIRE(dtype == KH_BF16 || dtype == KH_F32, "kh_beam_select: unsupported dtype %d", dtype);
  KH_REQUIRE(groups >= 0 && groups <= 65535 && beams >= 1 && beams <= kMaxBeams && groups * beams <= 65535,
             "kh_beam_select: %lld groups of %lld beams (1 to %d beams, at most 65535 rows)", (long long)groups, (long long)beams, kMaxBeams);
  KH_REQUIRE(vocab >= 1 && vocab < INT32_MAX - 2 * kRun, "kh_beam_select: bad vocabulary size %lld", (long long)vocab);
  KH_REQUIRE(k >= 1 && k <= kMaxK, "kh_beam_select: k %d outside 1..%d", k, kMaxK);
  KH_REQUIRE((finished != nullptr) == (out_finished != nullptr), "kh_beam_select: finished flags go in and come out together");
  // a group whose beams have all finished has that many continuations
  KH_REQUIRE(k <= (finished ? beams : beams * vocab), "kh_beam_select: %d continuations of %lld beams%s", k, (long long)beams,
             finished ? " that may have finished" : "");
  KH_REQUIRE(!finished || (eos >= 0 && eos < vocab), "kh_beam_select: end token %lld outside the vocabulary", (long long)eos);
  if (groups == 0) return KH_OK;
  KH_REQUIRE(logits && strides && scores && out_scores && out_tokens && out_parents, "kh_beam_select: null pointer");
  const int64_t rows = groups * beams;
  const int64_t size = dtype == KH_BF16 ? 2 : 4;
  KH_REQUIRE(!overlap({ints(out_scores, groups * k), ints(out_tokens, groups * k), ints(out_parents, groups * k),
                       ints(out_finished, groups * k)},
                      {ints(scores, rows), ints(finished, rows),
                       Span(logits, size * vocab, groups, size * strides[0], beams, size * strides[1])}),
             "kh_beam_select: the results must not share memory with the inputs or each other");
  const int shift = (dtype == KH_BF16 ? 8 : 4) - 1;  // a row may start this far inside a 16-byte block
  const int runs = (int)((vocab + shift + kRun - 1) / kRun);
  const size_t sum_bytes = ((size_t)rows * runs * sizeof(float2) + 255) / 256 * 256;
  uint8_t* scratch = (uint8_t*)scratch_alloc(sum_bytes + (size_t)rows * runs * k * 8);
  if (scratch == nullptr) return KH_ERR_OOM;
  float2* sums = (float2*)scratch;
  uint64_t* keys = (uint64_t*)(scratch + sum_bytes);
  const dim3 grid((unsigned)runs, (unsigned)rows);
  if (dtype == KH_BF16)
    beam_runs_kernel<uint16_t><<<grid, kRunWaves * 64, 0, stream()>>>((const uint16_t*)logits, strides[0], strides[1], (int)beams,
                                                          (int)vocab, finished, k, runs, sums, keys);
  else
    beam_runs_kernel<float><<<grid, kRunWaves * 64, 0, stream()>>>((const float*)logits, strides[0], strides[1], (int)beams, (int)vocab,
                                                       finished, k, runs, sums, keys);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) {
    beam_merge_kernel<<<(unsigned)groups, kMergeWaves * 64, 0, stream()>>>(sums, keys, scores, finished, (int)beams, (int)vocab, k, runs,
                                                              (int)eos, out_scores, out_tokens, out_parents, out_finished);
    e = hipGetLastError();
  }
  scratch_free(scratch);
  if (e != hipSuccess) {
    set_error("kh_beam_select: launch failed: %s", hipGetErrorString(e));
    return KH_ERR_HIP;
  }
  KH_DEBUG_SYNC();
  return KH_OK;
}

}  // extern "C"
