// The selection of a beam search step (kh_beam_select): the k best continuations of every group of beams
// over beams x vocabulary.
//
//   score(beam, token) = logits[beam, token] - log sum exp(logits[beam, :]) + scores[beam]
// A finished beam has one continuation: itself, with the end token.  NaN, as a logit or a score, counts
// as -inf.  Order: the larger score, then the lower beam, then the lower token.  Inside a beam the logits
// decide, so only the k largest of each beam are scored, in float64.
#include "common.h"

using namespace kh;

namespace {

constexpr int kMaxK = 64;
constexpr int kMaxBeams = 64;

// Order-preserving bits of a logit (-0 as +0), 1 at least: 0 stands for no candidate.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ uint64_t order_key(float x, int id) {
  return ((uint64_t)order_bits(x) << 32) | (uint64_t)(0xffffffffu - (uint32_t)id);
}
__device__ __forceinline__ float no_nan(float x) { return x != x ? -INFINITY : x; }

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor(v, o, 64);
    v = u > v ? u : v;
  }
  return v;
}

// A wave per run of 1024 logits of a row: their maximum, their sum of exponentials relative to it, and the
// keys of the k largest in order (0 behind the last).
constexpr int kRun = 1024, kPer = kRun / 64;
template <typename T>
__global__ __launch_bounds__(64) void beam_runs_kernel(const T* __restrict__ logits, int64_t sg, int64_t sb, int beams,
                                                       int vocab, const int32_t* __restrict__ finished, int k, int runs,
                                                       float2* __restrict__ sums, uint64_t* __restrict__ keys) {
  const int row = blockIdx.y, run = blockIdx.x, lane = threadIdx.x;
  if (finished && finished[row] != 0) return;
  const T* x = logits + (row / beams) * sg + (row % beams) * sb;
  uint64_t key[kPer];
  float v[kPer], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int id = run * kRun + i * 64 + lane;
    v[i] = id < vocab ? no_nan(Elem<T>::load(x, id)) : -INFINITY;
    key[i] = id < vocab ? order_key(v[i], id) : 0;
    m = fmaxf(m, v[i]);
  }
  m = wave_max(m);
  float s = 0.f;
  if (m > -INFINITY)
#pragma unroll
    for (int i = 0; i < kPer; ++i) s += __expf(v[i] - m);
  s = wave_sum(s);
  if (lane == 0) sums[(int64_t)row * runs + run] = make_float2(m, s);
  for (int j = 0; j < k; ++j) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = key[i] > best ? key[i] : best;
    best = wave_max_u64(best);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (key[i] == best) key[i] = 0;
    if (lane == 0) keys[((int64_t)row * runs + run) * k + j] = best;
  }
}

// A candidate of the last selection: its score and its place beam * vocab + token.
struct Best {
  double score;
  int64_t at;  // -1: none
};
__device__ __forceinline__ bool better(const Best& a, const Best& b) {
  if (a.at < 0 || b.at < 0) return b.at < 0 && a.at >= 0;
  return a.score > b.score || (a.score == b.score && a.at < b.at);
}

// A workgroup per group: the sums of its beams, then k rounds of the best candidate left.
__global__ __launch_bounds__(256) void beam_merge_kernel(const float2* __restrict__ sums, const uint64_t* __restrict__ keys,
                                                         const float* __restrict__ scores,
                                                         const int32_t* __restrict__ finished, int beams, int vocab, int k,
                                                         int runs, int eos, float* __restrict__ out_scores,
                                                         int32_t* __restrict__ out_tokens, int32_t* __restrict__ out_parents,
                                                         int32_t* __restrict__ out_finished) {
  __shared__ double base[kMaxBeams];  // scores[beam] - log sum exp, or NaN where all the beam's scores are -inf
  __shared__ double best_score[4];
  __shared__ int64_t best_at[4];
  const int g = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int b = w; b < beams; b += 4) {
    const int row = g * beams + b;
    const double sc = (double)scores[row];
    if (finished && finished[row] != 0) {
      if (lane == 0) base[b] = sc;
      continue;
    }
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
    if (lane == 0) {
      const double v = sc - ((double)m + log(s));
      base[b] = v == v && v > -INFINITY && v < INFINITY ? v : __builtin_nan("");
    }
  }
  __syncthreads();
  const int per = runs * k;
  Best last{INFINITY, -1};  // the one chosen last: the next one is the best behind it
  for (int j = 0; j < k; ++j) {
    Best mine{-INFINITY, -1};
    for (int64_t i = threadIdx.x; i < (int64_t)beams * per; i += 256) {
      const int b = (int)(i / per), c = (int)(i - (int64_t)b * per);
      const bool done = finished && finished[g * beams + b] != 0;
      Best x{-INFINITY, -1};
      if (done) {
        if (c == 0) x = Best{base[b] == base[b] ? base[b] : -INFINITY, (int64_t)b * vocab + eos};
      } else if (base[b] != base[b]) {
        if (c < k && c < vocab) x = Best{-INFINITY, (int64_t)b * vocab + c};
      } else {
        const uint64_t key = keys[(int64_t)(g * beams + b) * per + c];
        if (key != 0)
          x = Best{(double)order_value((uint32_t)(key >> 32)) + base[b],
                   (int64_t)b * vocab + (int64_t)(0xffffffffu - (uint32_t)key)};
      }
      if (x.at >= 0 && (last.at < 0 || better(last, x)) && better(x, mine)) mine = x;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const Best u{__shfl_xor(mine.score, o, 64), __shfl_xor(mine.at, o, 64)};
      if (better(u, mine)) mine = u;
    }
    __syncthreads();
    if (lane == 0) {
      best_score[w] = mine.score;
      best_at[w] = mine.at;
    }
    __syncthreads();
    last = Best{best_score[0], best_at[0]};
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      const Best u{best_score[i], best_at[i]};
      if (better(u, last)) last = u;
    }
    if (threadIdx.x == 0) {
      const int b = last.at < 0 ? 0 : (int)(last.at / vocab), t = last.at < 0 ? 0 : (int)(last.at - (int64_t)b * vocab);
      const int o = g * k + j;
      out_scores[o] = (float)last.score;
      out_tokens[o] = t;
      out_parents[o] = b;
      if (out_finished) out_finished[o] = (finished[g * beams + b] != 0 || t == eos) ? 1 : 0;
    }
    if (last.at < 0) break;
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
  KH_REQUIRE(vocab >= 1 && vocab < INT32_MAX - kRun, "kh_beam_select: bad vocabulary size %lld", (long long)vocab);
  KH_REQUIRE(k >= 1 && k <= kMaxK, "kh_beam_select: k %d outside 1..%d", k, kMaxK);
  KH_REQUIRE((finished != nullptr) == (out_finished != nullptr), "kh_beam_select: finished flags go in and come out together");
  // a group whose beams have all finished has that many continuations
  KH_REQUIRE(k <= (finished ? beams : beams * vocab), "kh_beam_select: %d continuations of %lld beams%s", k, (long long)beams,
             finished ? " that may have finished" : "");
  KH_REQUIRE(!finished || (eos >= 0 && eos < vocab), "kh_beam_select: end token %lld outside the vocabulary", (long long)eos);
  if (groups == 0) return KH_OK;
  KH_REQUIRE(logits && strides && scores && out_scores && out_tokens && out_parents, "kh_beam_select: null pointer");
  const int64_t rows = groups * beams;
  const int runs = (int)((vocab + kRun - 1) / kRun);
  const size_t sum_bytes = ((size_t)rows * runs * sizeof(float2) + 255) / 256 * 256;
  uint8_t* scratch = (uint8_t*)scratch_alloc(sum_bytes + (size_t)rows * runs * k * 8);
  if (scratch == nullptr) return KH_ERR_OOM;
  float2* sums = (float2*)scratch;
  uint64_t* keys = (uint64_t*)(scratch + sum_bytes);
  const dim3 grid((unsigned)runs, (unsigned)rows);
  if (dtype == KH_BF16)
    beam_runs_kernel<uint16_t><<<grid, 64, 0, stream()>>>((const uint16_t*)logits, strides[0], strides[1], (int)beams,
                                                          (int)vocab, finished, k, runs, sums, keys);
  else
    beam_runs_kernel<float><<<grid, 64, 0, stream()>>>((const float*)logits, strides[0], strides[1], (int)beams, (int)vocab,
                                                       finished, k, runs, sums, keys);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) {
    beam_merge_kernel<<<(unsigned)groups, 256, 0, stream()>>>(sums, keys, scores, finished, (int)beams, (int)vocab, k, runs,
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
