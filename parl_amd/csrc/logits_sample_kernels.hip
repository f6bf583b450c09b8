// logits_sample_kernels.hip — drawing actions from rows of logits: temperature, top-k, top-p, min-p, given uniforms.
//
// The actors' draw (examples/IMPALA/atari_agent.py:38-40: np.random.choice over softmax(logits)) for action sets of any
// size and with the usual filters.  Per row x of A logits with maximum m and temperature T:
//   w_i = e^{(x_i - m) / T} <= 1, weights below 2^-42 are 0
//   order the actions by (x descending, index ascending); keep the longest prefix with  position < top_k,
//   mass before < top_p * (mass of the first top_k),  w_i >= min_p   (the first always stays)
//   action = the first index i with  sum_{j <= i, kept} w_j > u * sum_{kept} w
// Every sum is an INTEGER: w is rounded once to a multiple of 2^-s (s = 44 for A = 2^18, more for fewer actions), so a sum
// is the same in any order and in any split over threads, and a border is met by the same action in every form of
// this kernel.  (Sums in float32 would move a draw in about one row of a hundred over 131,072 actions.)
#include "common.hpp"
#include "logits_common.hpp"

namespace parlhip {

constexpr int kSampleThreads = 256;
constexpr int64_t kSampleMaxActions = (int64_t)1 << 20;
constexpr double kWeightFloor = 0x1p-42;

struct SampleArgs {
  const double* uniforms;
  const float* temperature;   // per row, or NULL: the scalar
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_s, top_p_s, min_p_s;
  int32_t top_k_s;
  int64_t* actions;
  float* log_probs;
  int* err;
};

// the order of values as unsigned integers; -0 is 0
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// the weight of a logit: 2^-shift units; and as a double
__device__ __forceinline__ double weight(float x, float m, double inv_t) {
  const double w = exp(((double)x - (double)m) * inv_t);
  return w < kWeightFloor ? 0.0 : w;
}
__device__ __forceinline__ uint64_t weight_units(double w, double scale) { return (uint64_t)rint(w * scale); }

template <typename X>
__device__ __forceinline__ X block_sum(X v, X* lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  X t = 0;
  for (int w = 0; w < kSampleThreads / 64; ++w) t += lds[w];
  return t;
}

// One workgroup per row.  The borders of top-k and top-p are found by bisecting the 32 bits of the ordered value.
template <typename T>
__global__ __launch_bounds__(kSampleThreads) void logits_sample_kernel(const T* __restrict__ logits, int64_t stride,
                                                                       int64_t B, int A, int shift, SampleArgs q) {
  __shared__ uint64_t lds64[kSampleThreads / 64];
  __shared__ int lds32[kSampleThreads / 64];
  __shared__ float ldsf[kSampleThreads / 64];
  __shared__ int found;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * stride;
  const int tid = threadIdx.x;
  float t = q.temperature ? q.temperature[row] : q.temperature_s;
  int k = q.top_k ? q.top_k[row] : q.top_k_s;
  const float top_p = fmaxf(q.top_p ? q.top_p[row] : q.top_p_s, 0.f);
  const float min_p = fminf(q.min_p ? q.min_p[row] : q.min_p_s, 1.f);
  const bool greedy = !(t > 0.f);
  t = fminf(t, 3.0e38f);
  if (greedy) { t = 1.f; k = 1; }

  float m = -INFINITY;
  int bad = 0;
  for (int i = tid; i < A; i += kSampleThreads) {
    const float v = to_f32(x[i]);
    bad |= !(v < INFINITY);
    m = fmaxf(m, v);
  }
  m = wave_max_f32(m);
  bad = block_sum(bad, lds32);
  if ((tid & 63) == 0) ldsf[tid >> 6] = m;
  __syncthreads();
  for (int w = 0; w < kSampleThreads / 64; ++w) m = fmaxf(m, ldsf[w]);
  if (bad || m == -INFINITY) {   // no distribution, or nothing to choose from
    if (tid == 0) {
      q.actions[row] = -1;
      q.log_probs[row] = bad ? __builtin_nanf("") : 0.f;
      if (bad) *q.err = 1;
    }
    return;
  }
  const double inv_t = 1.0 / (double)t, scale = __builtin_ldexp(1.0, shift);
  auto units = [&](float v) { return weight_units(weight(v, m, inv_t), scale); };
  auto mass_from = [&](uint32_t key) {   // of the values with this key or a larger one
    uint64_t s = 0;
    for (int i = tid; i < A; i += kSampleThreads) {
      const float v = to_f32(x[i]);
      if (value_key(v) >= key) s += units(v);
    }
    return block_sum(s, lds64);
  };
  auto count_from = [&](uint32_t key) {
    int s = 0;
    for (int i = tid; i < A; i += kSampleThreads) s += value_key(to_f32(x[i])) >= key;
    return block_sum(s, lds32);
  };
  const uint32_t lowest = value_key(-INFINITY) + 1;   // of a legal action
  const uint64_t total = mass_from(lowest);
  const int legal = count_from(lowest);
  // the last value kept, and how many of its ties
  uint32_t cut = lowest;
  int ties = legal;
  uint64_t mass_k = total;
  if (k > 0 && k < legal) {
    uint32_t lo = lowest, hi = value_key(m);   // the largest key with at least k values from it on
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if (count_from(mid) >= k) lo = mid; else hi = mid - 1;
    }
    cut = lo;
    ties = k - count_from(cut + 1);
    mass_k = mass_from(cut + 1) + (uint64_t)ties * units(key_value(cut));
  }
  if (top_p < 1.0f) {
    uint64_t need = (uint64_t)ceil((double)top_p * (double)mass_k);
    if (need < 1) need = 1;
    uint32_t lo = lowest, hi = value_key(m);
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if (mass_from(mid) >= need) lo = mid; else hi = mid - 1;
    }
    if (lo >= cut) {
      const uint64_t above = mass_from(lo + 1), one = units(key_value(lo));
      const uint64_t n = (need - above + one - 1) / one;
      ties = lo > cut || n < (uint64_t)ties ? (int)n : ties;
      cut = lo;
    }
  }
  auto kept = [&](uint32_t key, double w, int before) { return (key > cut || (key == cut && before < ties)) && w >= (double)min_p; };
  // two passes in index order: the kept mass, then the draw
  uint64_t drawn = 0;
  uint64_t mass = 0;
  for (int pass = 0; pass < 2; ++pass) {
    uint64_t run = 0;
    int run_ties = 0;
    for (int base = 0; base < A; base += kSampleThreads) {
      const int i = base + tid;
      const float v = i < A ? to_f32(x[i]) : -INFINITY;
      const uint32_t key = value_key(v);
      // ties before this action, in index order
      const int tie = key == cut;
      int incl = tie;
      for (int off = 1; off < 64; off <<= 1) { const int o = __shfl_up(incl, off, 64); if ((tid & 63) >= off) incl += o; }
      __syncthreads();
      if ((tid & 63) == 63) lds32[tid >> 6] = incl;
      __syncthreads();
      int before = run_ties + incl - tie, all = 0;
      for (int w = 0; w < kSampleThreads / 64; ++w) { if (w < (tid >> 6)) before += lds32[w]; all += lds32[w]; }
      const double w = weight(v, m, inv_t);
      uint64_t u = key >= lowest && kept(key, w, before) ? weight_units(w, scale) : 0;
      uint64_t c = u;
      for (int off = 1; off < 64; off <<= 1) { const uint64_t o = __shfl_up(c, off, 64); if ((tid & 63) >= off) c += o; }
      __syncthreads();
      if ((tid & 63) == 63) lds64[tid >> 6] = c;
      if (tid == 0) found = 0x7fffffff;
      __syncthreads();
      uint64_t sum = 0;
      c += run;
      for (int w2 = 0; w2 < kSampleThreads / 64; ++w2) { if (w2 < (tid >> 6)) c += lds64[w2]; sum += lds64[w2]; }
      if (pass == 1 && c > drawn && c - u <= drawn && u > 0) found = i;   // one thread at most
      __syncthreads();
      if (pass == 1 && found != 0x7fffffff) {
        if (tid == 0) {
          const float v2 = to_f32(x[found]);
          q.actions[row] = found;
          q.log_probs[row] = greedy ? 0.f : (float)(((double)v2 - (double)m) * inv_t - log((double)total / scale));
        }
        return;
      }
      run += sum;
      run_ties += all;
    }
    if (pass == 0) {
      mass = run;
      // u * mass, rounded down, in whole units: u is a multiple of 2^-53
      double u = q.uniforms[row];
      u = u > 0.0 ? fmin(u, 1.0 - 0x1p-53) : 0.0;
      const uint64_t f = (uint64_t)(u * 0x1p53);
      drawn = (__umul64hi(f, mass) << 11) | ((f * mass) >> 53);
    }
  }
}

static inline int sample_shift(int64_t A) {
  int bits = 0;
  while (((int64_t)1 << bits) < A) ++bits;
  return 62 - bits < 51 ? 62 - bits : 51;
}

}  // namespace parlhip

using namespace parlhip;

PARLHIP_EXPORT size_t parlhip_logits_sample_workspace_bytes(int64_t B, int64_t A) { return 0; }

PARLHIP_EXPORT int parlhip_logits_sample(const void* logits, int dtype, int64_t row_stride, const double* uniforms,
                                         const float* temperature, const int32_t* top_k, const float* top_p,
                                         const float* min_p, float temperature_all, int32_t top_k_all, float top_p_all,
                                         float min_p_all, int64_t* actions, float* log_probs, int64_t B, int64_t A,
                                         void* workspace, size_t workspace_bytes, parlhip_stream_t stream) {
  if (B < 0 || A < 1 || row_stride < A) return PARLHIP_EINVAL;
  if (dtype != PARLHIP_F32 && dtype != PARLHIP_BF16 && dtype != PARLHIP_F16) return PARLHIP_ENOSUP;
  if (A > kSampleMaxActions || B > 0xffffffffLL / 1024) return PARLHIP_ENOSUP;
  if (!temperature && !(temperature_all >= 0.f && temperature_all < INFINITY)) return PARLHIP_EINVAL;
  if (!top_p && !(top_p_all >= 0.f)) return PARLHIP_EINVAL;
  if (!min_p && !(min_p_all >= 0.f && min_p_all <= 1.f)) return PARLHIP_EINVAL;
  if (B == 0) return PARLHIP_OK;
  if (!logits || !uniforms || !actions || !log_probs) return PARLHIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == PARLHIP_F32 ? 3 : 1)) return PARLHIP_EINVAL;
  SampleArgs q{uniforms, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all,
               actions, log_probs, device_error_flag()};
  if (!q.err) return PARLHIP_ELAUNCH;
  hipStream_t s = (hipStream_t)stream;
  const int shift = sample_shift(A);
  if (dtype == PARLHIP_F32)
    logits_sample_kernel<<<(int)B, kSampleThreads, 0, s>>>((const float*)logits, row_stride, B, (int)A, shift, q);
  else if (dtype == PARLHIP_BF16)
    logits_sample_kernel<<<(int)B, kSampleThreads, 0, s>>>((const bf16_t*)logits, row_stride, B, (int)A, shift, q);
  else
    logits_sample_kernel<<<(int)B, kSampleThreads, 0, s>>>((const f16_t*)logits, row_stride, B, (int)A, shift, q);
  return check_launch();
}
