// logits_logprob_kernels.hip — log-probability and entropy of taken actions, and their gradient, for action sets of any size.
//
// What the learners form with Categorical(logits).log_prob(actions) and .entropy() (parl/algorithms/torch/ppo.py:104-121,
// torch/a2c.py:56-70), with the temperature that the actions were drawn with.  Per row x of A logits, z = x / T:
//   lse = log sum_i exp z_i,  log p_i = z_i - lse,  log_prob = log p_a,  H = -sum_i p_i log p_i = lse - sum_i p_i z_i
//   d / d x_i = 1/T ( g_l ([i = a] - p_i) - g_h p_i (log p_i + H) )
// Forward: one pass over the row with the running maximum m, s = sum e^{z-m} and t = sum e^{z-m} (z - m), all in float32 and
// rescaled when m grows; H = log s - t / s.  The backward pass gets (m, s) and H, so it reads the row once and writes its
// gradient once; the probabilities are never stored.  Both passes are bound by HBM: one exp and some ten float
// operations per two or four bytes.  Rows of more than 512 actions whose action is -1 are not read (of fewer, all are: they
// lie side by side).  4,096 x 131,072 bf16, a tenth of the rows ignored: 579 us for both passes; under the tracer, which
// adds to them, forward 0.97 GB in 225 us (4.3 TB/s), backward 2.0 GB in 365 us (5.6 TB/s); a large copy moves 4.9 TB/s
// here.  At 51,200 x 6 each is a launch of 4 us, and the rest of a call's 31 to 54 us are the autograd engine's.
#include "common.hpp"
#include "logits_common.hpp"

namespace parlhip {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegBig = -1e4f;   // 2^kNegBig is 0 and stays 0 times any moment

// (maximum, sum, first moment) of some logits, in units of log 2 around the maximum: e = 2^{(x - m) c}, c = log2(e) / T
struct Stat {
  float m, s, t;
};

__device__ __forceinline__ Stat stat_empty() { return Stat{-INFINITY, 0.f, 0.f}; }

// moves the reference from a.m up to m (m >= a.m)
__device__ __forceinline__ void stat_raise(Stat& a, float m, float c) {
  if (a.m < m) {   // false for an equal or NaN maximum
    const float d = a.s > 0.f ? (a.m - m) * c : 0.f;   // nothing summed yet: nothing to move
    const float f = a.s > 0.f ? __builtin_amdgcn_exp2f(d) : 0.f;
    const float dd = fmaxf(d, kNegBig);                 // a.m - m may be beyond the float range
    if (a.s == a.s) {
      a.t = f * __builtin_fmaf(a.s, dd, a.t);
      a.s = a.s * f;
    }
    a.m = m;
  }
}

__device__ __forceinline__ void stat_join(Stat& a, const Stat& b, float c) {
  Stat o = b;
  const float m = fmaxf(a.m, o.m);
  stat_raise(a, m, c);
  stat_raise(o, m, c);
  a.s += o.s;
  a.t += o.t;
}

// adds n logits.  -inf is no choice: e = 0 and its term of t is 0.  NaN (and +inf - inf) makes s NaN and with it the row.
template <int n>
__device__ __forceinline__ void stat_add(Stat& a, const float (&x)[n], float c) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i < n; ++i) m = fmaxf(m, x[i]);
  stat_raise(a, fmaxf(a.m, m), c);
  const float base = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const float d = (x[i] - base) * c;
    const float e = __builtin_amdgcn_exp2f(d);
    a.s += e;
    a.t = __builtin_fmaf(e, fmaxf(d, kNegBig), a.t);
  }
}

template <int LANES>
__device__ __forceinline__ void stat_join_lanes(Stat& a, float c) {
#pragma unroll
  for (int off = LANES / 2; off > 0; off >>= 1) {
    Stat o;
    o.m = __shfl_xor(a.m, off, 64);
    o.s = __shfl_xor(a.s, off, 64);
    o.t = __shfl_xor(a.t, off, 64);
    stat_join(a, o, c);
  }
}

// nothing was added but -inf: a NaN alone leaves no maximum either, but makes the sum NaN
__device__ __forceinline__ bool nothing_legal(float m, float s) { return m == -INFINITY && s == 0.f; }

// the action of a row: -1 (no decision); an index outside [-1, A) is clamped and raises the data-error flag
__device__ __forceinline__ int64_t row_action(const int64_t* __restrict__ actions, int64_t row, int64_t A, int* err) {
  int64_t a = actions[row];
  if (a < -1 || a >= A) {
    if (err) *err = 1;
    a = a < 0 ? 0 : A - 1;
  }
  return a;
}

template <typename T>
__device__ __forceinline__ void row_finish(const Stat& st, const T* __restrict__ x, int64_t a, int64_t row, float inv_t,
                                           float* __restrict__ log_probs, float* __restrict__ entropies,
                                           float2* __restrict__ stats) {
  float lp = 0.f, h = 0.f;
  if (a >= 0 && !nothing_legal(st.m, st.s)) {
    const float log2s = __builtin_amdgcn_logf(st.s);
    lp = (to_f32(x[a]) - st.m) * inv_t - kLn2 * log2s;   // not in units of log 2: the lowest float stays finite
    h = kLn2 * (log2s - st.t / st.s);
  }
  log_probs[row] = lp;
  entropies[row] = h;
  if (stats) stats[row] = make_float2(st.m, st.s);
}

// Rows of at most 8 * LANES logits: LANES lanes of a wave share a row, every lane holds 8 of its logits in registers.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void logprob_small_kernel(const T* __restrict__ logits, int64_t stride,
                                                            const int64_t* __restrict__ actions,
                                                            float* __restrict__ log_probs, float* __restrict__ entropies,
                                                            float2* __restrict__ stats, int64_t N, int A, float c, float inv_t, int* err) {
  const int sub = threadIdx.x % LANES;
  const int64_t rows = 256 / LANES;
  for (int64_t row0 = (int64_t)blockIdx.x * rows; row0 < N; row0 += (int64_t)gridDim.x * rows) {
    const int64_t row = row0 + threadIdx.x / LANES;
    const bool live = row < N;
    const T* x = logits + (live ? row : 0) * stride;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = sub + i * LANES;
      v[i] = live && k < A ? to_f32(x[k]) : -INFINITY;
    }
    Stat st = stat_empty();
    stat_add(st, v, c);
    stat_join_lanes<LANES>(st, c);
    if (live && sub == 0) row_finish(st, x, row_action(actions, row, A, err), row, inv_t, log_probs, entropies, stats);
  }
}

// The part [begin, end) of a row, by NT threads; every thread ends with the whole part's sums.
template <typename T, int NT>
__device__ __forceinline__ Stat part_stat(const T* __restrict__ x, int64_t begin, int64_t end, float c, Stat* lds) {
  constexpr int V = Vec16<T>::n;
  Stat st = stat_empty();
  int64_t i = begin + (int64_t)threadIdx.x * V;
  for (; i + (int64_t)(3 * NT) * V + V <= end; i += (int64_t)4 * NT * V) {   // four loads in flight
    Vec16<T> v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u].load(x + i + (int64_t)u * NT * V);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float f[V];
      v[u].unpack(f);
      stat_add(st, f, c);
    }
  }
  for (; i < end; i += (int64_t)NT * V) {
    float f[V];
    if (i + V <= end) {
      Vec16<T> v;
      v.load(x + i);
      v.unpack(f);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = i + j < end ? to_f32(x[i + j]) : -INFINITY;
    }
    stat_add(st, f, c);
  }
  stat_join_lanes<64>(st, c);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = st;
    __syncthreads();
    st = lds[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) stat_join(st, lds[w], c);
    __syncthreads();
  }
  return st;
}

// One workgroup per (row, part): with one part it writes the row's results, else the part's sums for the join.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void logprob_row_kernel(const T* __restrict__ logits, int64_t stride,
                                                         const int64_t* __restrict__ actions,
                                                         float* __restrict__ log_probs, float* __restrict__ entropies,
                                                         float2* __restrict__ stats, Stat* __restrict__ parts, int64_t N,
                                                         int64_t A, int n_parts, int64_t part, float c, float inv_t, int* err) {
  __shared__ Stat lds[NT / 64];
  const int64_t row = (int64_t)blockIdx.x / n_parts;
  const int p = (int)(blockIdx.x % n_parts);
  const T* x = logits + row * stride;
  const int64_t begin = p * part;
  const int64_t end = begin + part < A ? begin + part : A;
  const int64_t a = row_action(actions, row, A, err);
  const Stat st = a >= 0 ? part_stat<T, NT>(x, begin, end, c, lds) : stat_empty();   // no decision: nothing to read
  if (threadIdx.x != 0) return;
  if (n_parts == 1)
    row_finish(st, x, a, row, inv_t, log_probs, entropies, stats);
  else
    parts[blockIdx.x] = st;
}

// a wave per row joins its parts
template <typename T>
__global__ __launch_bounds__(64) void logprob_join_kernel(const T* __restrict__ logits, int64_t stride,
                                                          const int64_t* __restrict__ actions,
                                                          float* __restrict__ log_probs, float* __restrict__ entropies,
                                                          float2* __restrict__ stats, const Stat* __restrict__ parts,
                                                          int64_t A, int n_parts, float c, float inv_t, int* err) {
  const int64_t row = blockIdx.x;
  Stat st = stat_empty();
  for (int p = threadIdx.x; p < n_parts; p += 64) stat_join(st, parts[row * n_parts + p], c);
  stat_join_lanes<64>(st, c);
  if (threadIdx.x == 0)
    row_finish(st, logits + row * stride, row_action(actions, row, A, err), row, inv_t, log_probs, entropies, stats);
}

// The row's scalars of the gradient: with l = log2 p_i = (x_i - m) c - log2 s,
//   dx_i = [i = a] g_l / T - p_i (k0 + k1 l),  k0 = (g_l + g_h H) / T,  k1 = g_h ln 2 / T
struct GradRow {
  float m, log2s, inv_s, k0, k1, one_hot;
  int64_t a;
  bool live;
};

__device__ __forceinline__ GradRow grad_row(const int64_t* __restrict__ actions, const float2* __restrict__ stats,
                                            const float* __restrict__ entropies, const float* __restrict__ g_logp,
                                            const float* __restrict__ g_ent, int64_t row, int64_t A, float inv_t) {
  GradRow r;
  const float2 st = stats[row];
  r.a = row_action(actions, row, A, nullptr);   // the forward pass raised the flag
  r.live = r.a >= 0 && !nothing_legal(st.x, st.y);
  const float gl = g_logp ? g_logp[row] : 0.f, gh = g_ent ? g_ent[row] : 0.f;
  r.m = st.x;
  r.log2s = __builtin_amdgcn_logf(st.y);
  r.inv_s = 1.0f / st.y;
  r.k0 = __builtin_fmaf(gh, entropies[row], gl) * inv_t;
  r.k1 = gh * inv_t * kLn2;
  r.one_hot = gl * inv_t;
  return r;
}

__device__ __forceinline__ float grad_at(const GradRow& r, float x, int64_t i, float c) {
  const float d = (x - r.m) * c;
  const float p = __builtin_amdgcn_exp2f(d) * r.inv_s;
  const float l = fmaxf(d, kNegBig) - r.log2s;              // p = 0 where x is -inf: 0 times a finite number
  const float g = -p * __builtin_fmaf(r.k1, l, r.k0);
  return i == r.a ? g + r.one_hot : g;
}

template <typename T, int LANES>
__global__ __launch_bounds__(256) void logprob_small_grad_kernel(
    const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ actions, const float2* __restrict__ stats,
    const float* __restrict__ entropies, const float* __restrict__ g_logp, const float* __restrict__ g_ent,
    T* __restrict__ grad, int64_t N, int A, float c, float inv_t) {
  const int sub = threadIdx.x % LANES;
  const int64_t rows = 256 / LANES;
  for (int64_t row0 = (int64_t)blockIdx.x * rows; row0 < N; row0 += (int64_t)gridDim.x * rows) {
    const int64_t row = row0 + threadIdx.x / LANES;
    if (row >= N) continue;
    const GradRow r = grad_row(actions, stats, entropies, g_logp, g_ent, row, A, inv_t);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = sub + i * LANES;
      if (k < A) from_f32(r.live ? grad_at(r, to_f32(logits[row * stride + k]), k, c) : 0.f, grad[row * A + k]);
    }
  }
}

// One workgroup per (row, part of the row), with two loads of each thread in flight.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void logprob_row_grad_kernel(
    const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ actions, const float2* __restrict__ stats,
    const float* __restrict__ entropies, const float* __restrict__ g_logp, const float* __restrict__ g_ent,
    T* __restrict__ grad, int64_t A, int n_parts, int64_t part, float c, float inv_t) {
  constexpr int V = Vec16<T>::n;
  const int64_t row = (int64_t)blockIdx.x / n_parts;
  const int64_t begin = (int64_t)(blockIdx.x % n_parts) * part;
  const int64_t end = begin + part < A ? begin + part : A;
  const T* x = logits + row * stride;
  T* o = grad + row * A;
  const GradRow r = grad_row(actions, stats, entropies, g_logp, g_ent, row, A, inv_t);
  int64_t i = begin + (int64_t)threadIdx.x * V;
  if (!r.live) {   // no decision: nothing to read
    const Vec16<T> zero{u32x4{0, 0, 0, 0}};
    for (; i + V <= end; i += (int64_t)NT * V) zero.store(o + i);
    for (; i < end; ++i) from_f32(0.f, o[i]);   // at most one thread has a rest of less than V
    return;
  }
  const auto put = [&](const Vec16<T>& v, int64_t at) {
    float f[V];
    v.unpack(f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = grad_at(r, f[j], at + j, c);
    Vec16<T> w;
    w.pack(f);
    w.store(o + at);
  };
  for (; i + (int64_t)NT * V + V <= end; i += (int64_t)2 * NT * V) {
    Vec16<T> v[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) v[u].load(x + i + (int64_t)u * NT * V);
#pragma unroll
    for (int u = 0; u < 2; ++u) put(v[u], i + (int64_t)u * NT * V);
  }
  for (; i + V <= end; i += (int64_t)NT * V) {
    Vec16<T> v;
    v.load(x + i);
    put(v, i);
  }
  for (; i < end; ++i) from_f32(grad_at(r, to_f32(x[i]), i, c), o[i]);
}

// How the rows are cut: few long rows are split over several workgroups so that about 1,024 of them (four per CU) run.
struct LogprobPlan {
  int n_parts;
  int64_t part;
};

static LogprobPlan logprob_plan(int64_t N, int64_t A) {
  constexpr int64_t kMinPart = 4096;   // elements a workgroup takes at least
  int64_t want = N >= 1024 ? 1 : (1024 + N - 1) / N;
  const int64_t most = (A + kMinPart - 1) / kMinPart;
  if (want > most) want = most;
  if (want < 1) want = 1;
  int64_t part = (A + want - 1) / want;
  part = (part + 15) / 16 * 16;
  const int64_t n = (A + part - 1) / part;
  return LogprobPlan{(int)(n < 1 ? 1 : n), part};
}

constexpr int64_t kMaxSmall = 512;      // 64 lanes x 8 logits
constexpr int64_t kMaxWaveRow = 4096;   // one wave per row up to here
// Above, by the length of a part: the more threads the longer the stretch of a row that is read at a time, and the fewer rows side by side: 4,096 rows
// of 131,072 bf16 take 613 / 594 / 579 us with 256 / 512 / 1,024 threads (both passes), 2,048 of 32,003 take 92 / 90 / 105.
constexpr int64_t kRow512 = 16384, kRow1024 = 65536;

static int row_threads(int64_t A, int64_t part) {
  return A <= kMaxWaveRow ? 64 : part < kRow512 ? 256 : part < kRow1024 ? 512 : 1024;
}

template <typename T>
static int logprob_forward(const T* logits, int64_t stride, const int64_t* actions, float* log_probs, float* entropies,
                           float2* stats, Stat* parts, int64_t N, int64_t A, float c, float inv_t, hipStream_t s) {
  int* err = device_error_flag();
  if (!err) return PARLHIP_ELAUNCH;
  if (A <= kMaxSmall) {
    const int lanes = A <= 32 ? 4 : A <= 128 ? 16 : 64;
    const int64_t want = (N * lanes + 255) / 256;
    const int grid = (int)(want < (1 << 20) ? want : (1 << 20));
    if (lanes == 4)
      logprob_small_kernel<T, 4><<<grid, 256, 0, s>>>(logits, stride, actions, log_probs, entropies, stats, N, (int)A, c, inv_t, err);
    else if (lanes == 16)
      logprob_small_kernel<T, 16><<<grid, 256, 0, s>>>(logits, stride, actions, log_probs, entropies, stats, N, (int)A, c, inv_t, err);
    else
      logprob_small_kernel<T, 64><<<grid, 256, 0, s>>>(logits, stride, actions, log_probs, entropies, stats, N, (int)A, c, inv_t, err);
    return check_launch();
  }
  const LogprobPlan p = logprob_plan(N, A);
  const int grid = (int)(N * p.n_parts);
  const int threads = row_threads(A, p.part);
  if (threads == 64)
    logprob_row_kernel<T, 64><<<grid, 64, 0, s>>>(logits, stride, actions, log_probs, entropies, stats, parts, N, A,
                                                  p.n_parts, p.part, c, inv_t, err);
  else if (threads == 256)
    logprob_row_kernel<T, 256><<<grid, 256, 0, s>>>(logits, stride, actions, log_probs, entropies, stats, parts,
        N, A, p.n_parts, p.part, c, inv_t, err);
  else if (threads == 512)
    logprob_row_kernel<T, 512><<<grid, 512, 0, s>>>(logits, stride, actions, log_probs, entropies, stats, parts,
        N, A, p.n_parts, p.part, c, inv_t, err);
  else
    logprob_row_kernel<T, 1024><<<grid, 1024, 0, s>>>(logits, stride, actions, log_probs, entropies, stats,
        parts, N, A, p.n_parts, p.part, c, inv_t, err);
  int rc = check_launch();
  if (rc || p.n_parts == 1) return rc;
  logprob_join_kernel<T><<<(int)N, 64, 0, s>>>(logits, stride, actions, log_probs, entropies, stats, parts, A, p.n_parts, c, inv_t, err);
  return check_launch();
}

template <typename T>
static int logprob_backward(const T* logits, int64_t stride, const int64_t* actions, const float2* stats,
                            const float* entropies, const float* g_logp, const float* g_ent, T* grad, int64_t N,
                            int64_t A, float c, float inv_t, hipStream_t s) {
  if (A <= kMaxSmall) {
    const int lanes = A <= 32 ? 4 : A <= 128 ? 16 : 64;
    const int64_t want = (N * lanes + 255) / 256;
    const int grid = (int)(want < (1 << 20) ? want : (1 << 20));
    if (lanes == 4)
      logprob_small_grad_kernel<T, 4><<<grid, 256, 0, s>>>(logits, stride, actions, stats, entropies, g_logp, g_ent, grad, N, (int)A, c, inv_t);
    else if (lanes == 16)
      logprob_small_grad_kernel<T, 16><<<grid, 256, 0, s>>>(logits, stride, actions, stats, entropies, g_logp, g_ent, grad, N, (int)A, c, inv_t);
    else
      logprob_small_grad_kernel<T, 64><<<grid, 256, 0, s>>>(logits, stride, actions, stats, entropies, g_logp, g_ent, grad, N, (int)A, c, inv_t);
    return check_launch();
  }
  const LogprobPlan p = logprob_plan(N, A);
  const int grid = (int)(N * p.n_parts);
  const int threads = row_threads(A, p.part);
  if (threads == 64)
    logprob_row_grad_kernel<T, 64><<<grid, 64, 0, s>>>(logits, stride, actions, stats, entropies, g_logp, g_ent, grad, A,
                                                       p.n_parts, p.part, c, inv_t);
  else if (threads == 256)
    logprob_row_grad_kernel<T, 256><<<grid, 256, 0, s>>>(logits, stride, actions, stats, entropies, g_logp,
        g_ent, grad, A, p.n_parts, p.part, c, inv_t);
  else if (threads == 512)
    logprob_row_grad_kernel<T, 512><<<grid, 512, 0, s>>>(logits, stride, actions, stats, entropies, g_logp,
        g_ent, grad, A, p.n_parts, p.part, c, inv_t);
  else
    logprob_row_grad_kernel<T, 1024><<<grid, 1024, 0, s>>>(logits, stride, actions, stats, entropies, g_logp,
        g_ent, grad, A, p.n_parts, p.part, c, inv_t);
  return check_launch();
}

static int logprob_check(const void* logits, int dtype, int64_t stride, const int64_t* actions, int64_t N, int64_t A,
                         float temperature) {
  if (N < 0 || A < 1 || stride < A) return PARLHIP_EINVAL;
  if (!(temperature > 0.f) || !(temperature < INFINITY) || !(kLog2e / temperature < INFINITY)) return PARLHIP_EINVAL;
  if (dtype != PARLHIP_F32 && dtype != PARLHIP_BF16 && dtype != PARLHIP_F16) return PARLHIP_ENOSUP;
  if (A > ((int64_t)1 << 31) || N > ((int64_t)1 << 40) / A) return PARLHIP_ENOSUP;
  if (N == 0) return PARLHIP_OK;
  if (A > kMaxSmall) {
    const LogprobPlan p = logprob_plan(N, A);
    if (N * p.n_parts > 0xffffffffLL / row_threads(A, p.part)) return PARLHIP_ENOSUP;   // one launch's threads
  }
  if (!logits || !actions) return PARLHIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == PARLHIP_F32 ? 3 : 1)) return PARLHIP_EINVAL;
  return PARLHIP_OK;
}

}  // namespace parlhip

using namespace parlhip;

PARLHIP_EXPORT size_t parlhip_logits_log_prob_workspace_bytes(int64_t N, int64_t A) {
  if (N <= 0 || A <= kMaxSmall) return 0;
  const LogprobPlan p = logprob_plan(N, A);
  return p.n_parts == 1 ? 0 : (size_t)N * p.n_parts * sizeof(Stat);
}

PARLHIP_EXPORT int parlhip_logits_log_prob(const void* logits, int dtype, int64_t row_stride, const int64_t* actions,
                                           float* log_probs, float* entropies, float* stats, int64_t N, int64_t A,
                                           float temperature, void* workspace, size_t workspace_bytes,
                                           parlhip_stream_t stream) {
  if (int rc = logprob_check(logits, dtype, row_stride, actions, N, A, temperature)) return rc;
  if (N == 0) return PARLHIP_OK;
  if (!log_probs || !entropies || (reinterpret_cast<uintptr_t>(stats) & 7)) return PARLHIP_EINVAL;
  const size_t need = parlhip_logits_log_prob_workspace_bytes(N, A);
  if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3))) return PARLHIP_EINVAL;
  if (workspace_bytes < need) return PARLHIP_ENOMEM;
  const float c = kLog2e / temperature, inv_t = 1.0f / temperature;
  hipStream_t s = (hipStream_t)stream;
  float2* st = (float2*)stats;
  Stat* parts = (Stat*)workspace;
  if (dtype == PARLHIP_F32)
    return logprob_forward((const float*)logits, row_stride, actions, log_probs, entropies, st, parts, N, A, c, inv_t, s);
  if (dtype == PARLHIP_BF16)
    return logprob_forward((const bf16_t*)logits, row_stride, actions, log_probs, entropies, st, parts, N, A, c, inv_t, s);
  return logprob_forward((const f16_t*)logits, row_stride, actions, log_probs, entropies, st, parts, N, A, c, inv_t, s);
}

PARLHIP_EXPORT int parlhip_logits_log_prob_backward(const void* logits, int dtype, int64_t row_stride,
                                                    const int64_t* actions, const float* stats, const float* entropies,
                                                    const float* grad_log_probs, const float* grad_entropies,
                                                    void* grad_logits, int64_t N, int64_t A, float temperature,
                                                    parlhip_stream_t stream) {
  if (int rc = logprob_check(logits, dtype, row_stride, actions, N, A, temperature)) return rc;
  if (N == 0) return PARLHIP_OK;
  if (!stats || !entropies || !grad_logits || (reinterpret_cast<uintptr_t>(stats) & 7)) return PARLHIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(grad_logits) & (dtype == PARLHIP_F32 ? 3 : 1)) return PARLHIP_EINVAL;
  const float c = kLog2e / temperature, inv_t = 1.0f / temperature;
  hipStream_t s = (hipStream_t)stream;
  const float2* st = (const float2*)stats;
  if (dtype == PARLHIP_F32)
    return logprob_backward((const float*)logits, row_stride, actions, st, entropies, grad_log_probs, grad_entropies,
                            (float*)grad_logits, N, A, c, inv_t, s);
  if (dtype == PARLHIP_BF16)
    return logprob_backward((const bf16_t*)logits, row_stride, actions, st, entropies, grad_log_probs, grad_entropies,
                            (bf16_t*)grad_logits, N, A, c, inv_t, s);
  return logprob_backward((const f16_t*)logits, row_stride, actions, st, entropies, grad_log_probs, grad_entropies,
                          (f16_t*)grad_logits, N, A, c, inv_t, s);
}
