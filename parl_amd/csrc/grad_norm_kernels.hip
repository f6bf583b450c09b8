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
// Measured: 1.1 G bf16 values in 435 tensors into bf16, read twice and written once (6.6 GB), 1,284 us = 5.1 TB/s (a large copy:
// 4.9); 120 M into float32 (240 MB read twice, 480 written) 232 us: two launches of 81 together for the norm, which alone,
// call after call, takes 54, and two of 150 that move 4.8 TB/s; the 42x42 model's ten float32 gradients 9.3 us, two
// launches of 4.  In place and under the bound the scaling launches still walk over their chunks: 1.1 G values 584 us, the
// norm alone 428.  Four workgroups per CU were 3 % slower than two over 2 GB, one 30 %.
#include "common.hpp"
#include "logits_common.hpp"
#include <algorithm>
#include <new>

namespace parlhip {

constexpr int kNormMaxBlocks = 512;       // per launch: 2 workgroups of 256 threads per CU
constexpr int kNormDirect = 4096;         // up to here every workgroup of the scaling launch adds the partials itself

// The tensors of one launch, as its argument: at most 4 KB.  An address and its type share a word (addresses have 48 bits);
// a tensor's size is its number of chunks less what its last one lacks.
template <int N>
struct NormTable {
  uint64_t g[N];
  uint32_t first[N + 1];                  // prefix sums of the chunks
  uint16_t lack[N];
  uint16_t n, chunk;                      // tensors; elements that a workgroup takes at a time
};
constexpr int kNormRead = 256, kNormWrite = 168;   // tensors per launch: 14 bytes each, 22 with an output
constexpr int kNormFew = 16;                        // a shorter table where that is enough: a launch copies its arguments
template <int N>
struct NormOut {
  uint64_t o[N];
};
static_assert(sizeof(NormTable<kNormRead>) + 32 <= 4096 && sizeof(NormTable<kNormWrite>) + sizeof(NormOut<kNormWrite>) + 48 <= 4096,
              "the tables are kernel arguments");
constexpr int kTypeShift = 56;
constexpr uint64_t kAddress = ((uint64_t)1 << kTypeShift) - 1;

__device__ __forceinline__ double norm_block_sum(double x, double* red) {   // a fixed tree over 256 threads
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// f(tensor, first element, elements) for every `stride`th chunk of a launch from c on, the same for the whole workgroup.  The
// workgroups take neighbouring chunks side by side: a stretch of chunks for each was a tenth slower over 2 GB.
template <int N, typename F>
__device__ __forceinline__ void norm_chunks_of(const NormTable<N>& t, int64_t c, int64_t stride, F&& f) {
  const int64_t chunks = t.first[t.n];
  int k = 0;
  for (; c < chunks; c += stride) {
    int hi = t.n - 1;
    while (k < hi) {                      // the last tensor that begins at c or before
      const int mid = (k + hi + 1) >> 1;
      if (t.first[mid] <= c) k = mid; else hi = mid - 1;
    }
    f(k, (c - t.first[k]) * t.chunk, c + 1 == t.first[k + 1] ? t.chunk - t.lack[k] : t.chunk);
  }
}

template <typename T>
__device__ __forceinline__ double chunk_sqsum(const T* __restrict__ g, int n) {
  constexpr int V = Vec16<T>::n;
  double s = 0.0;
  int i = (int)threadIdx.x * V;
  for (; i + 3 * 256 * V + V <= n; i += 4 * 256 * V) {   // four loads in flight
    Vec16<T> v[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) v[a].load(g + i + a * 256 * V);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double x = (double)v[a].get(j);
        s = __builtin_fma(x, x, s);
      }
  }
  for (; i < n; i += 256 * V) {
    if (i + V <= n) {
      Vec16<T> v;
      v.load(g + i);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double x = (double)v.get(j);
        s = __builtin_fma(x, x, s);
      }
    } else {
      for (int j = i; j < n; ++j) {
        const double x = (double)to_f32(g[j]);
        s = __builtin_fma(x, x, s);
      }
    }
  }
  return s;
}

template <int N>
__global__ __launch_bounds__(256) void grad_norm_partial_kernel(NormTable<N> t, double* __restrict__ partial) {
  __shared__ double red[4];
  double s = 0.0;
  norm_chunks_of(t, blockIdx.x, gridDim.x,
                 [&](int k, int64_t base, int n) {
                   const void* g = (const void*)(t.g[k] & kAddress);
                   const int type = (int)(t.g[k] >> kTypeShift);
                   if (type == PARLHIP_F32) s += chunk_sqsum((const float*)g + base, n);
                   else if (type == PARLHIP_BF16) s += chunk_sqsum((const bf16_t*)g + base, n);
                   else s += chunk_sqsum((const f16_t*)g + base, n);
                 });
  s = norm_block_sum(s, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double norm_total(const double* __restrict__ partial, int n, double* red) {
  double s = 0.0;
  int i = threadIdx.x;
  for (; i + 3 * 256 < n; i += 4 * 256) {
    const double a = partial[i], b = partial[i + 256], c = partial[i + 512], d = partial[i + 768];
    s += (a + b) + (c + d);
  }
  for (; i < n; i += 256) s += partial[i];
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
__device__ __forceinline__ void scale_vec(const Vec16<T>& v, U* o, float c) {
  constexpr int V = Vec16<T>::n;
  float f[V];
  v.unpack(f);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] *= c;
  if constexpr (sizeof(U) == sizeof(T)) {
    Vec16<U> w;
    w.pack(f);
    w.store(o);
  } else if constexpr (sizeof(U) == 4) {    // 8 values widened: two stores
    Vec16<float> w;
    const float a[4] = {f[0], f[1], f[2], f[3]}, b[4] = {f[4], f[5], f[6], f[7]};
    w.pack(a);
    w.store(o);
    w.pack(b);
    w.store(o + 4);
  } else {                                  // 4 values narrowed
#pragma unroll
    for (int j = 0; j < V; ++j) from_f32(f[j], o[j]);
  }
}

template <typename T, typename U>
__device__ __forceinline__ void chunk_scale(const T* g, U* o, int n, float c) {
  constexpr int V = Vec16<T>::n;
  int i = (int)threadIdx.x * V;
  for (; i + 3 * 256 * V + V <= n; i += 4 * 256 * V) {
    Vec16<T> v[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) v[a].load(g + i + a * 256 * V);
#pragma unroll
    for (int a = 0; a < 4; ++a) scale_vec(v[a], o + i + a * 256 * V, c);
  }
  for (; i < n; i += 256 * V) {
    if (i + V <= n) {
      Vec16<T> v;
      v.load(g + i);
      scale_vec(v, o + i, c);
    } else {
      for (int j = i; j < n; ++j) from_f32(to_f32(g[j]) * c, o[j]);
    }
  }
}

template <typename T>
__device__ __forceinline__ void chunk_scale_to(const T* g, void* o, int ot, int64_t base, int n, float c) {
  if (ot == PARLHIP_F32) chunk_scale(g, (float*)o + base, n, c);
  else if (ot == PARLHIP_BF16) chunk_scale(g, (bf16_t*)o + base, n, c);
  else chunk_scale(g, (f16_t*)o + base, n, c);
}

// g and o may be the same memory (in place): a thread reads its own elements and then writes them, and no other does.
template <int N>
__global__ __launch_bounds__(256) void grad_norm_scale_kernel(NormTable<N> t, NormOut<N> out, const double* __restrict__ partial, int n_partial,
                                                              double max_norm, float* __restrict__ norm_out) {
  __shared__ double red[4];
  const double norm = sqrt(norm_total(partial, n_partial, red));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  double cd = max_norm / (norm + 1e-6);
  cd = cd < 1.0 ? cd : (cd != cd ? cd : 1.0);   // a NaN norm stays: every gradient turns NaN at once, as torch's do
  const float c = (float)cd;
  norm_chunks_of(t, blockIdx.x, gridDim.x,
                 [&](int k, int64_t base, int n) {
                   if (t.g[k] == out.o[k] && c == 1.0f) return;   // in place and under the bound: g * 1 is g
                   const void* g = (const void*)(t.g[k] & kAddress);
                   const int type = (int)(t.g[k] >> kTypeShift), to = (int)(out.o[k] >> kTypeShift);
                   void* o = (void*)(out.o[k] & kAddress);
                   if (type == PARLHIP_F32) chunk_scale_to((const float*)g + base, o, to, base, n, c);
                   else if (type == PARLHIP_BF16) chunk_scale_to((const bf16_t*)g + base, o, to, base, n, c);
                   else chunk_scale_to((const f16_t*)g + base, o, to, base, n, c);
                 });
}

// Elements that a workgroup takes at a time: four loads for each of its threads; a quarter where the card would be short
// of workgroups.
static int norm_chunk(int n_tensors, const int64_t* numel) {
  int64_t total = 0;
  for (int i = 0; i < n_tensors; ++i) total += numel[i];
  return total < (int64_t)8192 * kNormMaxBlocks ? 2048 : 8192;
}

static inline int norm_grid(int64_t chunks) { return (int)(chunks < kNormMaxBlocks ? chunks : kNormMaxBlocks); }

// Walks the tensors in launches of at most N non-empty ones: f(table, outputs, chunks) for each.  Returns a PARLHIP code.
template <int N, typename F>
static int norm_walk(int n_tensors, const void* const* grads, void* const* outs, const int64_t* numel,
                     const int32_t* gt, const int32_t* ot, F&& f) {
  NormTable<N> t;
  uint64_t o[N] = {};
  t.n = 0;
  t.chunk = (uint16_t)norm_chunk(n_tensors, numel);
  int64_t chunks = 0;
  auto flush = [&]() -> int {
    if (t.n == 0) return PARLHIP_OK;
    t.first[t.n] = (uint32_t)chunks;
    const int rc = f(t, o, chunks);
    t.n = 0;
    chunks = 0;
    return rc;
  };
  for (int i = 0; i < n_tensors; ++i) {
    if (numel[i] == 0) continue;
    const int64_t c = (numel[i] + t.chunk - 1) / t.chunk;
    if (t.n == N || chunks + c > 0x7fffffffLL)
      if (int rc = flush()) return rc;
    t.g[t.n] = ((uint64_t)(uintptr_t)(grads ? grads[i] : nullptr) & kAddress) | ((uint64_t)(gt ? gt[i] : 0) << kTypeShift);
    o[t.n] = outs ? ((uint64_t)(uintptr_t)outs[i] & kAddress) | ((uint64_t)(ot ? ot[i] : 0) << kTypeShift) : t.g[t.n];
    t.lack[t.n] = (uint16_t)(c * t.chunk - numel[i]);
    t.first[t.n] = (uint32_t)chunks;
    ++t.n;
    chunks += c;
  }
  return flush();
}

static inline int type_size(int t) { return t == PARLHIP_F32 ? 4 : 2; }
constexpr int64_t kNormMaxNumel = (int64_t)1 << 40;   // 2^29 chunks
static inline bool type_ok(int t) { return t == PARLHIP_F32 || t == PARLHIP_BF16 || t == PARLHIP_F16; }

// partials of all launches; < 0: an argument is wrong
static int64_t norm_partials(int n_tensors, const int64_t* numel) {
  if (n_tensors < 0 || (n_tensors > 0 && !numel)) return -1;
  for (int i = 0; i < n_tensors; ++i)
    if (numel[i] < 0 || numel[i] > kNormMaxNumel) return -1;
  int64_t p = 0;
  norm_walk<kNormRead>(n_tensors, nullptr, nullptr, numel, nullptr, nullptr,
                       [&](const NormTable<kNormRead>&, const uint64_t*, int64_t chunks) {
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
    if (numel[i] < 0 || numel[i] > kNormMaxNumel || (numel[i] > 0 && !grads[i])) return PARLHIP_EINVAL;
    if (numel[i] > 0 && (reinterpret_cast<uintptr_t>(grads[i]) & ((type_size(types[i]) - 1) | ~kAddress))) return PARLHIP_EINVAL;
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

// The partials and the norm overlap neither each other nor a tensor of the call.
static bool norm_scratch_apart(int n_tensors, const void* const* grads, void* const* outs, const int64_t* numel,
                               const int32_t* gt, const int32_t* ot, const void* workspace, size_t bytes, const float* norm_out) {
  const auto meets = [](const void* a, size_t an, const void* b, size_t bn) {
    return (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
  };
  const auto hit = [&](const void* p, size_t n) { return meets(p, n, workspace, bytes) || meets(p, n, norm_out, sizeof(float)); };
  if (meets(workspace, bytes, norm_out, sizeof(float))) return false;
  for (int i = 0; i < n_tensors; ++i) {
    if (numel[i] == 0) continue;
    if (hit(grads[i], (size_t)numel[i] * type_size(gt[i])) || (outs && hit(outs[i], (size_t)numel[i] * type_size(ot[i])))) return false;
  }
  return true;
}

template <int READ, int WRITE>
static int norm_launch(int n_tensors, const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* gt,
                       const int32_t* ot, bool clip, double max_norm, double* partial, int n_partial, float* norm_out,
                       hipStream_t s) {
  int64_t at = 0;
  int rc = norm_walk<READ>(n_tensors, grads, nullptr, numel, gt, nullptr,
                           [&](const NormTable<READ>& t, const uint64_t*, int64_t chunks) {
                             const int grid = norm_grid(chunks);
                             grad_norm_partial_kernel<READ><<<grid, 256, 0, s>>>(t, partial + at);
                             at += grid;
                             return check_launch();
                           });
  if (rc) return rc;
  // Up to kNormDirect partials every workgroup of the scaling launch adds them itself (32 KB out of the L2); above, one
  // workgroup adds them first, one launch more.
  const bool direct = clip && n_partial > 0 && n_partial <= kNormDirect;
  if (!direct) {
    grad_norm_total_kernel<<<1, 256, 0, s>>>(partial, n_partial, norm_out);
    if ((rc = check_launch())) return rc;
    n_partial = 1;
  }
  if (!clip) return PARLHIP_OK;
  return norm_walk<WRITE>(n_tensors, grads, outs, numel, gt, ot,
                          [&](const NormTable<WRITE>& t, const uint64_t* o, int64_t chunks) {
                            NormOut<WRITE> out;
                            std::copy(o, o + WRITE, out.o);
                            grad_norm_scale_kernel<WRITE><<<norm_grid(chunks), 256, 0, s>>>(
                                t, out, partial, n_partial, max_norm, direct ? norm_out : nullptr);
                            return check_launch();
                          });
}

static int norm_run(int n_tensors, const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* gt,
                    const int32_t* ot, bool clip, double max_norm, void* workspace, size_t workspace_bytes,
                    float* norm_out, hipStream_t s) {
  const int64_t p = norm_partials(n_tensors, numel);
  if (p < 0 || p > 0x7fffffffLL) return PARLHIP_EINVAL;
  if (!norm_out) return PARLHIP_EINVAL;
  double* partial = (double*)workspace;
  if (!partial || (reinterpret_cast<uintptr_t>(partial) & 7)) return PARLHIP_EINVAL;
  const size_t bytes = (size_t)(p > 0 ? p : 1) * sizeof(double);
  if (workspace_bytes < bytes) return PARLHIP_ENOMEM;
  if (!norm_scratch_apart(n_tensors, grads, outs, numel, gt, ot, workspace, bytes, norm_out)) return PARLHIP_EINVAL;
  if (n_tensors <= kNormFew)
    return norm_launch<kNormFew, kNormFew>(n_tensors, grads, outs, numel, gt, ot, clip, max_norm, partial, (int)p, norm_out, s);
  return norm_launch<kNormRead, kNormWrite>(n_tensors, grads, outs, numel, gt, ot, clip, max_norm, partial, (int)p, norm_out, s);
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
