// grad_norm_kernels.hip — the global norm of many gradient tensors, and clipping by it.
//
// The framework's update clips by the global norm (parl/algorithms/torch/a2c.py:76-78, torch/ppo.py:150-152:
// clip_grad_norm_(parameters, max_norm)).  ops.ClipAdam fuses that with Adam for at most 16 float32 tensors; this is the
// pair for any number of tensors of float32 / bfloat16 / float16 and any optimizer behind it:
//   norm = sqrt(sum over all tensors and elements of g^2),  c = min(1, max_norm / (norm + 1e-6)),  g <- c g
// Squares are formed and summed in float64 (a float32 square leaves the range at 1.8e19 and at 1e-23; the conversion and
// the multiply-add hide behind the loads), one partial per workgroup, all partials added in one fixed order: the same
// gradients give the same bits in every call.  The tensors' addresses travel as kernel arguments, so nothing is copied to
// the device and a captured call carries its own table.
#include "common.hpp"
#include "logits_common.hpp"
#include <algorithm>
#include <new>

namespace parlhip {

constexpr int kNormTensors = 96;          // tensors per launch: the table has to fit the 4 KB of kernel arguments
constexpr int kNormChunk = 16384;         // elements a workgroup takes at a time
constexpr int kNormMaxBlocks = 2048;      // per launch: 8 workgroups of 256 threads per CU
constexpr int kNormDirect = 1024;         // up to here every workgroup of the scaling launch adds the partials itself

struct NormTable {
  const void* g[kNormTensors];
  void* o[kNormTensors];
  int64_t numel[kNormTensors];
  int32_t first[kNormTensors + 1];        // prefix sums of ceil(numel / kNormChunk)
  uint8_t gt[kNormTensors];
  uint8_t ot[kNormTensors];
  int32_t n;
};
static_assert(sizeof(NormTable) + 64 <= 4096, "the table is a kernel argument");

// the tensor that chunk c belongs to (the same for the whole workgroup)
__device__ __forceinline__ int norm_tensor_of(const NormTable& t, int c) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double norm_block_sum(double x, double* red) {   // a fixed tree over 256 threads
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename T>
__device__ __forceinline__ double chunk_sqsum(const T* __restrict__ g, int64_t n) {
  constexpr int V = Vec16<T>::n;
  double s = 0.0;
  for (int64_t i = (int64_t)threadIdx.x * V; i < n; i += 256 * V) {
    if (i + V <= n) {
      Vec16<T> v;
      v.load(g + i);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double x = (double)v.get(j);
        s = __builtin_fma(x, x, s);
      }
    } else {
      for (int64_t j = i; j < n; ++j) {
        const double x = (double)to_f32(g[j]);
        s = __builtin_fma(x, x, s);
      }
    }
  }
  return s;
}

__global__ __launch_bounds__(256) void grad_norm_partial_kernel(NormTable t, double* __restrict__ partial) {
  __shared__ double red[4];
  double s = 0.0;
  for (int c = blockIdx.x; c < t.first[t.n]; c += gridDim.x) {
    const int k = norm_tensor_of(t, c);
    const int64_t base = (int64_t)(c - t.first[k]) * kNormChunk;
    const int64_t left = t.numel[k] - base;
    const int64_t n = left < kNormChunk ? left : kNormChunk;
    if (t.gt[k] == PARLHIP_F32) s += chunk_sqsum((const float*)t.g[k] + base, n);
    else if (t.gt[k] == PARLHIP_BF16) s += chunk_sqsum((const bf16_t*)t.g[k] + base, n);
    else s += chunk_sqsum((const f16_t*)t.g[k] + base, n);
  }
  s = norm_block_sum(s, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double norm_total(const double* __restrict__ partial, int n, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) s += partial[i];
  return norm_block_sum(s, red);
}

// one workgroup: the sum of all partials -> partial[0], the norm -> norm_out
__global__ __launch_bounds__(256) void grad_norm_total_kernel(double* __restrict__ partial, int n,
                                                              float* __restrict__ norm_out) {
  __shared__ double red[4];
  const double total = norm_total(partial, n, red);   // every read is done before the barrier in here
  if (threadIdx.x == 0) {
    partial[0] = total;
    if (norm_out) *norm_out = (float)sqrt(total);
  }
}

template <typename T, typename U>
__device__ __forceinline__ void chunk_scale(const T* g, U* o, int64_t n, float c) {
  constexpr int V = Vec16<T>::n;
  for (int64_t i = (int64_t)threadIdx.x * V; i < n; i += 256 * V) {
    if (i + V <= n) {
      Vec16<T> v;
      v.load(g + i);
      float f[V];
      v.unpack(f);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] *= c;
      if constexpr (sizeof(U) == sizeof(T)) {
        Vec16<U> w;
        w.pack(f);
        w.store(o + i);
      } else if constexpr (sizeof(U) == 4) {   // 8 values widened: two stores
        Vec16<float> w;
        const float a[4] = {f[0], f[1], f[2], f[3]}, b[4] = {f[4], f[5], f[6], f[7]};
        w.pack(a);
        w.store(o + i);
        w.pack(b);
        w.store(o + i + 4);
      } else {                                  // 4 values narrowed
#pragma unroll
        for (int j = 0; j < V; ++j) from_f32(f[j], o[i + j]);
      }
    } else {
      for (int64_t j = i; j < n; ++j) from_f32(to_f32(g[j]) * c, o[j]);
    }
  }
}

template <typename T>
__device__ __forceinline__ void chunk_scale_to(const T* g, void* o, int ot, int64_t base, int64_t n, float c) {
  if (ot == PARLHIP_F32) chunk_scale(g, (float*)o + base, n, c);
  else if (ot == PARLHIP_BF16) chunk_scale(g, (bf16_t*)o + base, n, c);
  else chunk_scale(g, (f16_t*)o + base, n, c);
}

// g and o may be the same memory (in place): a thread reads its own elements and then writes them, and no other does
__global__ __launch_bounds__(256) void grad_norm_scale_kernel(NormTable t, const double* __restrict__ partial,
                                                              int n_partial, double max_norm,
                                                              float* __restrict__ norm_out) {
  __shared__ double red[4];
  const double norm = sqrt(norm_total(partial, n_partial, red));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  double cd = max_norm / (norm + 1e-6);
  cd = cd < 1.0 ? cd : (cd != cd ? cd : 1.0);   // a NaN norm stays: every gradient turns NaN at once, as torch's do
  const float c = (float)cd;
  for (int i = blockIdx.x; i < t.first[t.n]; i += gridDim.x) {
    const int k = norm_tensor_of(t, i);
    if (t.g[k] == t.o[k] && c == 1.0f) continue;   // in place and under the bound: g * 1 is g
    const int64_t base = (int64_t)(i - t.first[k]) * kNormChunk;
    const int64_t left = t.numel[k] - base;
    const int64_t n = left < kNormChunk ? left : kNormChunk;
    if (t.gt[k] == PARLHIP_F32) chunk_scale_to((const float*)t.g[k] + base, t.o[k], t.ot[k], base, n, c);
    else if (t.gt[k] == PARLHIP_BF16) chunk_scale_to((const bf16_t*)t.g[k] + base, t.o[k], t.ot[k], base, n, c);
    else chunk_scale_to((const f16_t*)t.g[k] + base, t.o[k], t.ot[k], base, n, c);
  }
}

static inline int64_t norm_chunks(int64_t numel) { return (numel + kNormChunk - 1) / kNormChunk; }

// launches over at most kNormTensors non-empty tensors each; blocks(i) of one launch
struct NormPlan {
  int64_t launches = 0, partials = 0;
};

// Walks the tensors in launches: f(table, chunks) for each.  Returns a PARLHIP code.
template <typename F>
static int norm_walk(int n_tensors, const void* const* grads, void* const* outs, const int64_t* numel,
                     const int32_t* gt, const int32_t* ot, F&& f) {
  NormTable t;
  t.n = 0;
  int64_t chunks = 0;
  auto flush = [&]() -> int {
    if (t.n == 0) return PARLHIP_OK;
    t.first[t.n] = (int32_t)chunks;
    const int rc = f(t, (int)chunks);
    t.n = 0;
    chunks = 0;
    return rc;
  };
  for (int i = 0; i < n_tensors; ++i) {
    if (numel[i] == 0) continue;
    const int64_t c = norm_chunks(numel[i]);
    if (t.n == kNormTensors || chunks + c > 0x7fffffffLL)
      if (int rc = flush()) return rc;
    t.g[t.n] = grads ? grads[i] : nullptr;
    t.o[t.n] = outs ? outs[i] : const_cast<void*>(t.g[t.n]);
    t.numel[t.n] = numel[i];
    t.first[t.n] = (int32_t)chunks;
    t.gt[t.n] = gt ? (uint8_t)gt[i] : 0;
    t.ot[t.n] = ot ? (uint8_t)ot[i] : t.gt[t.n];
    ++t.n;
    chunks += c;
  }
  return flush();
}

static inline int norm_grid(int chunks) { return chunks < kNormMaxBlocks ? chunks : kNormMaxBlocks; }

static inline int type_size(int t) { return t == PARLHIP_F32 ? 4 : 2; }
static inline bool type_ok(int t) { return t == PARLHIP_F32 || t == PARLHIP_BF16 || t == PARLHIP_F16; }

// partials of all launches; < 0: an argument is wrong
static int64_t norm_partials(int n_tensors, const int64_t* numel) {
  if (n_tensors < 0 || (n_tensors > 0 && !numel)) return -1;
  for (int i = 0; i < n_tensors; ++i)
    if (numel[i] < 0 || numel[i] > ((int64_t)1 << 44)) return -1;
  int64_t p = 0;
  norm_walk(n_tensors, nullptr, nullptr, numel, nullptr, nullptr, [&](const NormTable&, int chunks) {
    p += norm_grid(chunks);
    return PARLHIP_OK;
  });
  return p;
}

static int norm_check(int n_tensors, const void* const* grads, const int64_t* numel, const int32_t* types) {
  if (n_tensors < 0) return PARLHIP_EINVAL;
  if (n_tensors > 0 && (!grads || !numel || !types)) return PARLHIP_EINVAL;
  for (int i = 0; i < n_tensors; ++i) {
    if (!type_ok(types[i])) return PARLHIP_ENOSUP;
    if (numel[i] < 0 || numel[i] > ((int64_t)1 << 44) || (numel[i] > 0 && !grads[i])) return PARLHIP_EINVAL;
    if (numel[i] > 0 && (reinterpret_cast<uintptr_t>(grads[i]) & (type_size(types[i]) - 1))) return PARLHIP_EINVAL;
  }
  return PARLHIP_OK;
}

// What is written may overlap nothing else that the call reads or writes, but a gradient its own output: two workgroups
// would race on the same memory.  Sorts the written and the read ranges by address.
static int norm_overlap(int n_tensors, const void* const* grads, void* const* outs, const int64_t* numel,
                        const int32_t* gt, const int32_t* ot) {
  struct Range { uintptr_t at, end; int32_t tensor; bool written; };
  Range* r = new (std::nothrow) Range[2 * (size_t)n_tensors];
  if (!r) return PARLHIP_ENOMEM;
  size_t n = 0;
  for (int i = 0; i < n_tensors; ++i) {
    if (numel[i] == 0) continue;
    const uintptr_t g = (uintptr_t)grads[i], o = (uintptr_t)outs[i];
    r[n++] = {o, o + (uintptr_t)numel[i] * type_size(ot[i]), i, true};
    if (g != o) r[n++] = {g, g + (uintptr_t)numel[i] * type_size(gt[i]), i, false};
  }
  std::sort(r, r + n, [](const Range& a, const Range& b) { return a.at < b.at; });
  int rc = PARLHIP_OK;
  uintptr_t end_any = 0, end_written = 0;   // how far what came before reaches
  for (size_t i = 0; i < n && rc == PARLHIP_OK; ++i) {
    if (r[i].at < end_written || (r[i].written && r[i].at < end_any)) rc = PARLHIP_EINVAL;
    if (r[i].end > end_any) end_any = r[i].end;
    if (r[i].written && r[i].end > end_written) end_written = r[i].end;
  }
  delete[] r;
  return rc;
}

static int norm_run(int n_tensors, const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* gt,
                    const int32_t* ot, bool clip, double max_norm, void* workspace, size_t workspace_bytes,
                    float* norm_out, hipStream_t s) {
  const int64_t p = norm_partials(n_tensors, numel);
  if (p < 0 || p > 0x7fffffffLL) return PARLHIP_EINVAL;
  if (!norm_out) return PARLHIP_EINVAL;
  double* partial = (double*)workspace;
  if (!partial || (reinterpret_cast<uintptr_t>(partial) & 7)) return PARLHIP_EINVAL;
  if (workspace_bytes < (size_t)(p > 0 ? p : 1) * sizeof(double)) return PARLHIP_ENOMEM;
  int64_t at = 0;
  int rc = norm_walk(n_tensors, grads, outs, numel, gt, ot, [&](const NormTable& t, int chunks) {
    const int grid = norm_grid(chunks);
    grad_norm_partial_kernel<<<grid, 256, 0, s>>>(t, partial + at);
    at += grid;
    return check_launch();
  });
  if (rc) return rc;
  // Up to kNormDirect partials every workgroup of the scaling launch adds them itself (8 KB out of the L2); above, one
  // workgroup adds them first, one launch more.
  int n_partial = (int)p;
  const bool direct = clip && p > 0 && p <= kNormDirect;
  if (!direct) {
    grad_norm_total_kernel<<<1, 256, 0, s>>>(partial, n_partial, norm_out);
    if ((rc = check_launch())) return rc;
    n_partial = 1;
  }
  if (!clip) return PARLHIP_OK;
  return norm_walk(n_tensors, grads, outs, numel, gt, ot, [&](const NormTable& t, int chunks) {
    grad_norm_scale_kernel<<<norm_grid(chunks), 256, 0, s>>>(t, partial, n_partial, max_norm,
                                                             direct ? norm_out : nullptr);
    return check_launch();
  });
}

}  // namespace parlhip

using namespace parlhip;

PARLHIP_EXPORT size_t parlhip_grad_norm_workspace_bytes(int n_tensors, const int64_t* numel) {
  const int64_t p = norm_partials(n_tensors, numel);
  return p < 0 ? 0 : (size_t)(p > 0 ? p : 1) * sizeof(double);
}

PARLHIP_EXPORT int parlhip_grad_norm(int n_tensors, const void* const* grads, const int64_t* numel,
                                     const int32_t* types, void* workspace, size_t workspace_bytes, float* norm_out,
                                     parlhip_stream_t stream) {
  if (int rc = norm_check(n_tensors, grads, numel, types)) return rc;
  return norm_run(n_tensors, grads, nullptr, numel, types, nullptr, false, 0.0, workspace, workspace_bytes, norm_out,
                  (hipStream_t)stream);
}

PARLHIP_EXPORT int parlhip_clip_grad_norm(int n_tensors, const void* const* grads, void* const* outs,
                                          const int64_t* numel, const int32_t* types, const int32_t* out_types,
                                          double max_norm, void* workspace, size_t workspace_bytes, float* norm_out,
                                          parlhip_stream_t stream) {
  if (int rc = norm_check(n_tensors, grads, numel, types)) return rc;
  if (!(max_norm >= 0.0)) return PARLHIP_EINVAL;
  if (!outs != !out_types) return PARLHIP_EINVAL;
  if (outs)
    if (int rc = norm_check(n_tensors, (const void* const*)outs, numel, out_types)) return rc;
  for (int i = 0; outs && i < n_tensors; ++i)
    if (numel[i] > 0 && grads[i] == outs[i] && types[i] != out_types[i]) return PARLHIP_EINVAL;
  if (n_tensors > 0)
    if (int rc = norm_overlap(n_tensors, grads, outs ? outs : (void* const*)grads, numel, types,
                              outs ? out_types : types))
      return rc;
  return norm_run(n_tensors, grads, outs, numel, types, out_types, true, max_norm, workspace, workspace_bytes, norm_out,
                  (hipStream_t)stream);
}
