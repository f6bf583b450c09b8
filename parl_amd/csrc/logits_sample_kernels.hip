// logits_sample_kernels.hip — drawing actions from rows of logits: temperature, top-k, top-p, min-p, given uniforms.
//
// The actors' draw (examples/IMPALA/atari_agent.py:38-40: np.random.choice over softmax(logits)) for action sets of any
// size and with the usual filters.  Per row x of A logits with maximum m and temperature T:
//   w_i = e^{(x_i - m) / T} <= 1, weights below 2^-42 are 0
//   order the actions by (x descending, index ascending); keep the longest prefix with  position < top_k,
//   mass before < top_p * (mass of the first top_k),  w_i >= min_p   (the first always stays)
//   action = the first index i with  sum_{j <= i, kept} w_j > u * sum_{kept} w
//
// Every sum is an INTEGER: w is formed in float64 and rounded once to a multiple of 2^-s (s = 44 for A = 2^18, more for
// fewer actions), so a sum is the same in any order and in any split over threads, atomics included, and the forms of this
// kernel below draw the same action from the same row.  (Sums in float32 would move the draw of about one row in a
// hundred over 131,072 actions: the border between two actions has to be right to far less than their weights.)
//
// No sort.  What top-k and top-p keep is "larger than a cut value, and the first few that equal it".  The cut is found by a
// histogram of counts and masses over 256 classes of -log2 w, a scan of the classes, and the same again inside the class
// that holds the border (on a list of its values in LDS, or on the row where a flat row puts more into one class than
// the list takes) until a class is a single value.  Then one pass sums what is kept, segment by segment in index order, and
// the segment that the draw falls into is scanned.  Three forms by size: lanes of a wave (A <= 64), a workgroup per row,
// and three launches over parts of the row where the rows are few and long.
#include "common.hpp"
#include "logits_common.hpp"

namespace parlhip {

constexpr int64_t kSampleMaxActions = (int64_t)1 << 20;
constexpr double kFloorLog2 = -42.0;     // weights under 2^-42 are 0
constexpr int kBins = 256;
constexpr int kList = 4096;

struct SampleArgs {
  const double* uniforms;
  const float* temperature;   // per row, or NULL: the scalar behind it
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_s, top_p_s, min_p_s;
  int32_t top_k_s;
  int64_t* actions;
  float* log_probs;
  int* err;
  int shift;                  // weights are multiples of 2^-shift
};

// one row's settings, with what lies outside a range moved to its end (a NaN to the narrower one)
struct Row {
  double c;        // log2(e) / T
  double ymin;     // log2 of the smallest weight that min_p keeps
  float top_p;
  int k;           // 0: off
  bool greedy;
};

__device__ __forceinline__ Row row_settings(const SampleArgs& q, int64_t row) {
  Row r;
  float t = q.temperature ? q.temperature[row] : q.temperature_s;
  r.k = q.top_k ? q.top_k[row] : q.top_k_s;
  r.top_p = fmaxf(q.top_p ? q.top_p[row] : q.top_p_s, 0.f);
  const float min_p = fminf(q.min_p ? q.min_p[row] : q.min_p_s, 1.f);
  r.greedy = !(t > 0.f);
  t = fminf(t, 3.0e38f);
  if (r.greedy) { t = 1.f; r.k = 1; }
  if (r.k < 0) r.k = 0;
  if (r.top_p == 0.f) r.k = 1;            // only the first action
  if (r.k == 1) r.top_p = 1.f;
  r.c = 1.4426950408889634 / (double)t;
  r.ymin = min_p > 0.f ? fmax(kFloorLog2, log2((double)min_p)) : kFloorLog2;
  return r;
}

// whether the cut needs the histogram
__device__ __forceinline__ bool needs_histogram(const Row& r) { return r.k > 1 || r.top_p < 1.f; }

// the order of values as unsigned integers; -0 is 0
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// log2 of a weight; 0 at the maximum
__device__ __forceinline__ double log2_weight(float x, float m, double c) { return ((double)x - (double)m) * c; }

// 2^y in units of 2^-shift, rounded to nearest; y in [-42, 0], shift <= 51.  2^r = 1 + r q(r) on |r| <= 1/2 with q the
// interpolation of (2^r - 1) / r at nine Chebyshev nodes: relative error 4e-14, and 2^0 is 1.  Adding 2^52 to a number below
// it leaves its nearest integer in the low bits.
__device__ __forceinline__ uint64_t weight_units(double y, int shift) {
  const double n = rint(y), r = y - n;
  double p = 0x1.b63880a30e9ffp-24;
  p = __builtin_fma(p, r, 0x1.63d136366db24p-20);
  p = __builtin_fma(p, r, 0x1.ffcb9515a8016p-17);
  p = __builtin_fma(p, r, 0x1.4308ac85aa947p-13);
  p = __builtin_fma(p, r, 0x1.5d87fe86fe88ep-10);
  p = __builtin_fma(p, r, 0x1.3b2ab7181b755p-7);
  p = __builtin_fma(p, r, 0x1.c6b08d7047e52p-5);
  p = __builtin_fma(p, r, 0x1.ebfbdff823cedp-3);
  p = __builtin_fma(p, r, 0x1.62e42fefa39efp-1);
  p = __builtin_fma(p, r, 1.0);
  const double v = __builtin_amdgcn_ldexp(p, (int)n + shift) + 0x1p52;
  return (uint64_t)__double_as_longlong(v) & 0xfffffffffffffULL;
}

// the class of a weight: 0 for the largest, 255 for those just above 2^-42
__device__ __forceinline__ int weight_bin(double y) {
  const int b = (int)(y * (-(double)kBins / 42.0));
  return b < kBins - 1 ? b : kBins - 1;
}

// u * mass rounded down to whole units; u is a multiple of 2^-53, so this is exact: the draw is the first action whose
// running mass exceeds it, and there always is one
__device__ __forceinline__ uint64_t draw_target(double u, uint64_t mass) {
  u = u > 0.0 ? fmin(u, 1.0 - 0x1p-53) : 0.0;
  const uint64_t f = (uint64_t)(u * 0x1p53);
  return (__umul64hi(f, mass) << 11) | ((f * mass) >> 53);
}

// the least mass that reaches the share top_p of mass_k
__device__ __forceinline__ uint64_t top_p_mass(float top_p, uint64_t mass_k) {
  const uint64_t need = (uint64_t)ceil((double)top_p * (double)mass_k);
  return need < 1 ? 1 : need;
}

__device__ __forceinline__ float log_prob_of(float x, float m, const Row& r, uint64_t total, int shift) {
  if (r.greedy) return 0.f;
  const double d = log2_weight(x, m, r.c) * 0.6931471805599453;
  return (float)(d - log(__builtin_amdgcn_ldexp((double)total, -shift)));
}

// ------------------------------------------------------------------------------------------------------------------
// A <= 64: LP lanes share a row, a lane holds one action.  The position and the mass before an action are summed over
// the row's lanes directly.
template <typename T, int LP>
__global__ __launch_bounds__(256) void sample_small_kernel(const T* __restrict__ logits, int64_t stride, int64_t B, int A,
                                                           SampleArgs q) {
  const int sub = threadIdx.x % LP;
  const int64_t row = (int64_t)blockIdx.x * (256 / LP) + threadIdx.x / LP;
  const bool live = row < B;
  const float x = live && sub < A ? to_f32(logits[row * stride + sub]) : -INFINITY;
  int bad = !(x < INFINITY);
  float m = x;
#pragma unroll
  for (int off = LP / 2; off > 0; off >>= 1) {
    m = fmaxf(m, __shfl_xor(m, off, 64));
    bad |= __shfl_xor(bad, off, 64);
  }
  const Row r = row_settings(q, live ? row : 0);
  const bool usable = !bad && m > -INFINITY;
  const double y = usable && x > -INFINITY ? log2_weight(x, m, r.c) : -1e300;
  const uint64_t u = y >= kFloorLog2 ? weight_units(y, q.shift) : 0;
  uint64_t total = u;
#pragma unroll
  for (int off = LP / 2; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
  bool keep = u > 0;
  if (__any(r.k > 0 || r.top_p < 1.f)) {
    int position = 0;
    uint64_t before = 0;
    for (int j = 0; j < LP; ++j) {
      const float xj = __shfl(x, j, LP);
      const uint64_t uj = __shfl(u, j, LP);
      if (uj > 0 && (xj > x || (xj == x && j < sub))) {
        ++position;
        before += uj;
      }
    }
    keep = keep && (r.k == 0 || position < r.k);
    uint64_t mass_k = keep ? u : 0;
#pragma unroll
    for (int off = LP / 2; off > 0; off >>= 1) mass_k += __shfl_xor(mass_k, off, 64);
    keep = keep && (r.top_p >= 1.f || before < top_p_mass(r.top_p, mass_k));
  }
  keep = keep && y >= r.ymin;
  uint64_t run = keep ? u : 0;
#pragma unroll
  for (int off = 1; off < LP; off <<= 1) {
    const uint64_t o = __shfl_up(run, off, LP);
    if (sub >= off) run += o;
  }
  const uint64_t mass = __shfl(run, LP - 1, LP);
  if (!live) return;
  if (!usable) {
    if (sub == 0) {
      q.actions[row] = -1;
      q.log_probs[row] = bad ? __builtin_nanf("") : 0.f;
      if (bad) *q.err = 1;
    }
    return;
  }
  const uint64_t target = draw_target(q.uniforms[row], mass);
  if (keep && run > target && run - u <= target) {
    q.actions[row] = sub;
    q.log_probs[row] = log_prob_of(x, m, r, total, q.shift);
  }
}

// ------------------------------------------------------------------------------------------------------------------
// A workgroup per row (or per part of a row).

template <typename T, int NT>
struct RowWork {
  static constexpr int kWaves = NT / 64;
  uint64_t mass[kBins];
  uint32_t count[kBins];
  uint32_t list[kList];
  uint64_t seg_mass[kWaves];
  uint32_t seg_ties[kWaves];
  uint64_t red64[kWaves];
  uint32_t red32[kWaves];
  uint32_t lo, hi, n;                    // of the class under refinement
  int bin;                               // what the scan found
  uint64_t above_mass;
  uint32_t above_count;
  int found;
};

// f(value, index) for the elements [begin, end) of a row, spread over NT threads, four loads in flight; no order
template <typename T, int NT, typename F>
__device__ __forceinline__ void for_each(const T* __restrict__ x, int64_t begin, int64_t end, int tid, F&& f) {
  constexpr int V = Vec16<T>::n;
  int64_t i = begin + (int64_t)tid * V;
  for (; i + (int64_t)(3 * NT) * V + V <= end; i += (int64_t)4 * NT * V) {
    Vec16<T> v[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) v[a].load(x + i + (int64_t)a * NT * V);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int j = 0; j < V; ++j) f(v[a].get(j));
  }
  for (; i < end; i += (int64_t)NT * V) {
    if (i + V <= end) {
      Vec16<T> v;
      v.load(x + i);
#pragma unroll
      for (int j = 0; j < V; ++j) f(v.get(j));
    } else {
      for (int64_t j = i; j < end; ++j) f(to_f32(x[j]));
    }
  }
}

template <typename X, int NT>
__device__ __forceinline__ X group_sum(X v, X* lds) {   // every thread gets the sum
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (NT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v += lds[w];
  }
  return v;
}

// the maximum of [begin, end); bad: a NaN or +inf among them
template <typename T, int NT>
__device__ __forceinline__ float part_max(const T* __restrict__ x, int64_t begin, int64_t end, bool& bad, uint32_t* lds) {
  float m = -INFINITY;
  uint32_t b = 0;
  for_each<T, NT>(x, begin, end, threadIdx.x, [&](float v) {
    b |= !(v < INFINITY);
    m = fmaxf(m, v);
  });
  m = wave_max_f32(m);
  b = __any(b) ? 1 : 0;
  if constexpr (NT > 64) {
    const int w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[w] = value_key(m) | 0;
    __syncthreads();
    uint32_t k = lds[0];
#pragma unroll
    for (int o = 1; o < NT / 64; ++o) k = lds[o] > k ? lds[o] : k;
    m = key_value(k);
    b = group_sum<uint32_t, NT>((threadIdx.x & 63) == 0 ? b : 0, lds);
  }
  bad = b != 0;
  return m;
}

// counts and masses of the classes of [begin, end) -> w.count, w.mass (cleared here); returns this thread's mass
template <typename T, int NT>
__device__ __forceinline__ uint64_t part_histogram(const T* __restrict__ x, int64_t begin, int64_t end, float m, const Row& r,
                                                   int shift, RowWork<T, NT>& w) {
  for (int i = threadIdx.x; i < kBins; i += NT) { w.mass[i] = 0; w.count[i] = 0; }
  __syncthreads();
  uint64_t total = 0;
  for_each<T, NT>(x, begin, end, threadIdx.x, [&](float v) {
    const double y = log2_weight(v, m, r.c);
    if (y >= kFloorLog2) {
      const uint64_t u = weight_units(y, shift);
      total += u;
      const int b = weight_bin(y);
      atomicAdd(&w.count[b], 1u);
      atomicAdd((unsigned long long*)&w.mass[b], (unsigned long long)u);
    }
  });
  __syncthreads();
  return total;
}

// Finds the class that reaches `need` (a count, or a mass) counted from class 0 -> w.bin and what lies above it.  The first
// wave scans, four classes a lane.  bin = -1: the classes together do not reach it.
template <typename T, int NT>
__device__ __forceinline__ void scan_classes(RowWork<T, NT>& w, bool by_mass, uint64_t need) {
  __syncthreads();
  if (threadIdx.x < 64) {
    const int l = threadIdx.x;
    uint32_t c[4];
    uint64_t s[4];
    uint32_t cs = 0;
    uint64_t ss = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = w.count[4 * l + j];
      s[j] = w.mass[4 * l + j];
      cs += c[j];
      ss += s[j];
    }
    uint32_t ci = cs;
    uint64_t si = ss;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t co = __shfl_up(ci, off, 64);
      const uint64_t so = __shfl_up(si, off, 64);
      if (l >= off) { ci += co; si += so; }
    }
    if (l == 0) w.bin = -1;
    uint32_t ca = ci - cs;   // above this lane's classes
    uint64_t sa = si - ss;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool here = by_mass ? (sa < need && sa + s[j] >= need) : ((uint64_t)ca < need && (uint64_t)ca + c[j] >= need);
      if (here) {
        w.bin = 4 * l + j;
        w.above_count = ca;
        w.above_mass = sa;
      }
      ca += c[j];
      sa += s[j];
    }
  }
  __syncthreads();
}

struct Cut {
  float value;          // kept: larger than this, and the first `ties` that equal it
  uint32_t ties;
  uint64_t above;       // mass of the larger ones
};

// The value at which the count (or mass) counted from the top reaches `need`, inside class `bin` of the histogram.
template <typename T, int NT>
__device__ __forceinline__ Cut refine(const T* __restrict__ x, int64_t A, float m, const Row& r, int shift,
                                      RowWork<T, NT>& w, int bin, uint64_t above_mass, uint64_t above_count, bool by_mass,
                                      uint64_t need) {
  __syncthreads();
  if (threadIdx.x == 0) { w.n = 0; w.lo = 0xffffffffu; w.hi = 0; }
  __syncthreads();
  uint32_t lo = 0xffffffffu, hi = 0;
  for_each<T, NT>(x, 0, A, threadIdx.x, [&](float v) {
    const double y = log2_weight(v, m, r.c);
    if (y >= kFloorLog2 && weight_bin(y) == bin) {
      const uint32_t k = value_key(v);
      lo = k < lo ? k : lo;
      hi = k > hi ? k : hi;
      const uint32_t at = atomicAdd(&w.n, 1u);
      if (at < kList) w.list[at] = k;
    }
  });
  if (hi != 0) {
    atomicMin(&w.lo, lo);
    atomicMax(&w.hi, hi);
  }
  __syncthreads();
  lo = w.lo;
  hi = w.hi;
  const uint32_t n = w.n;
  const bool listed = n <= kList;
  while (lo < hi) {   // at least 8 bits less each time
    int sh = 24 - __clz(hi - lo);
    if (sh < 0) sh = 0;
    for (int i = threadIdx.x; i < kBins; i += NT) { w.mass[i] = 0; w.count[i] = 0; }
    __syncthreads();
    auto add = [&](uint32_t k) {
      if (k >= lo && k <= hi) {
        const int b = (int)((hi - k) >> sh);
        atomicAdd(&w.count[b], 1u);
        atomicAdd((unsigned long long*)&w.mass[b], (unsigned long long)weight_units(log2_weight(key_value(k), m, r.c), shift));
      }
    };
    if (listed)
      for (uint32_t i = threadIdx.x; i < n; i += NT) add(w.list[i]);
    else
      for_each<T, NT>(x, 0, A, threadIdx.x, [&](float v) { add(value_key(v)); });
    scan_classes(w, by_mass, need - (by_mass ? above_mass : above_count));
    const int b = w.bin < 0 ? 0 : w.bin;   // it is there: the class as a whole reaches `need`
    above_mass += w.above_mass;
    above_count += w.above_count;
    const uint32_t top = hi - ((uint32_t)b << sh);
    const uint32_t width = (1u << sh) - 1;
    hi = top;
    lo = top - lo > width ? top - width : lo;
    if (sh == 0) lo = hi;
    __syncthreads();
  }
  Cut cut;
  cut.value = key_value(hi);
  cut.above = above_mass;
  const uint64_t one = weight_units(log2_weight(cut.value, m, r.c), shift);
  cut.ties = by_mass ? (uint32_t)((need - above_mass + one - 1) / one) : (uint32_t)(need - above_count);
  return cut;
}

// the cut of top-k and top-p, from the row's histogram in w (which it uses up)
template <typename T, int NT>
__device__ __forceinline__ Cut find_cut(const T* __restrict__ x, int64_t A, float m, const Row& r, int shift, uint64_t total,
                                        RowWork<T, NT>& w) {
  Cut cut{-INFINITY, 0xffffffffu, 0};
  uint64_t mass_k = total;
  int bin_k = -1, bin_p = -1;
  uint64_t am_k = 0, am_p = 0, ac_k = 0, ac_p = 0;
  if (r.k > 1) {
    scan_classes(w, false, (uint64_t)r.k);
    bin_k = w.bin;
    am_k = w.above_mass;
    ac_k = w.above_count;
  }
  uint64_t need = 0;
  if (bin_k >= 0) {   // the histogram is needed again for top-p: scan for it before it is used up
    if (r.top_p < 1.f) {
      // mass_k lies between the masses above and through class bin_k; the class of the top-p border is known
      // only when mass_k is.  Keep the classes in registers of the first wave's lanes.
      uint64_t keep_m[4];
      uint32_t keep_c[4];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 4 * (threadIdx.x & 63) + j;
        keep_m[j] = w.mass[i];
        keep_c[j] = w.count[i];
      }
      cut = refine(x, A, m, r, shift, w, bin_k, am_k, ac_k, false, (uint64_t)r.k);
      mass_k = cut.above + (uint64_t)cut.ties * weight_units(log2_weight(cut.value, m, r.c), shift);
      __syncthreads();
      if (threadIdx.x < 64) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w.mass[4 * threadIdx.x + j] = keep_m[j];
          w.count[4 * threadIdx.x + j] = keep_c[j];
        }
      }
    } else {
      return refine(x, A, m, r, shift, w, bin_k, am_k, ac_k, false, (uint64_t)r.k);
    }
  }
  if (r.top_p < 1.f) {
    need = top_p_mass(r.top_p, mass_k);
    scan_classes(w, true, need);
    bin_p = w.bin;
    am_p = w.above_mass;
    ac_p = w.above_count;
    const Cut p = refine(x, A, m, r, shift, w, bin_p < 0 ? 0 : bin_p, am_p, ac_p, true, need);
    if (p.value > cut.value || (p.value == cut.value && p.ties < cut.ties)) cut = p;
  }
  return cut;
}

// What is kept of [begin, end), by the lanes of one wave: mass of the values above the cut, number of values at the cut,
// and (all) the mass of everything.
template <typename T>
__device__ __forceinline__ void kept_mass(const T* __restrict__ x, int64_t begin, int64_t end, float m, const Row& r,
                                          int shift, const Cut& cut, bool want_all, uint64_t& mass, uint32_t& ties,
                                          uint64_t& all) {
  uint64_t s = 0, a = 0;
  uint32_t t = 0;
  for_each<T, 64>(x, begin, end, threadIdx.x & 63, [&](float v) {
    const bool above = v > cut.value;
    t += v == cut.value;
    if (above || want_all) {
      const double y = log2_weight(v, m, r.c);
      if (y >= kFloorLog2) {
        const uint64_t u = weight_units(y, shift);
        a += u;
        if (above && y >= r.ymin) s += u;
      }
    }
  });
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    s += __shfl_xor(s, off, 64);
    a += __shfl_xor(a, off, 64);
    t += __shfl_xor(t, off, 64);
  }
  mass = s;
  ties = t;
  all = a;
}

// the segments of a row that are summed one by one: `n` of `len` elements
__device__ __forceinline__ int64_t segment_length(int64_t A, int n) {
  const int64_t len = (A + n - 1) / n;
  return (len + 511) / 512 * 512;
}

// The draw: seg_mass / seg_ties hold n segments' sums.  Thread-uniform result: the segment, and the target and the ties left
// at its beginning.  Then the segment is scanned in index order.
template <typename T, int NT>
__device__ __forceinline__ void pick(const T* __restrict__ x, int64_t A, float m, const Row& r, const SampleArgs& q,
                                     int64_t row, const Cut& cut, uint64_t total, const uint64_t* seg_mass,
                                     const uint32_t* seg_ties, int n, int64_t len, RowWork<T, NT>& w) {
  constexpr int V = Vec16<T>::n;
  const double y_cut = log2_weight(cut.value, m, r.c);
  // the values at the cut are kept if min_p keeps them
  const uint64_t one = cut.value > -INFINITY && y_cut >= r.ymin ? weight_units(y_cut, q.shift) : 0;
  uint64_t mass = 0;
  uint32_t left = one ? cut.ties : 0;
  for (int s = 0; s < n; ++s) {
    const uint32_t t = seg_ties[s] < left ? seg_ties[s] : left;
    mass += seg_mass[s] + (uint64_t)t * one;
    left -= t;
  }
  uint64_t target = draw_target(q.uniforms[row], mass);
  left = one ? cut.ties : 0;
  int s = 0;
  for (; s < n - 1; ++s) {
    const uint32_t t = seg_ties[s] < left ? seg_ties[s] : left;
    const uint64_t here = seg_mass[s] + (uint64_t)t * one;
    if (here > target) break;
    target -= here;
    left -= t;
  }
  const int64_t begin = s * len, end = begin + len < A ? begin + len : A;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t base = begin; base < end; base += (int64_t)NT * V) {
    const int64_t i0 = base + (int64_t)threadIdx.x * V;
    float v[V];
    uint64_t u[V];
    uint32_t tie = 0;
    bool full = i0 + V <= end;
    if (full) {
      Vec16<T> raw;
      raw.load(x + i0);
      raw.unpack(v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = i0 + j < end ? to_f32(x[i0 + j]) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) tie += one && v[j] == cut.value;
    uint32_t ti = tie;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t o = __shfl_up(ti, off, 64);
      if (lane >= off) ti += o;
    }
    uint32_t tie_before = ti - tie, tie_all = 0;
    if constexpr (NT > 64) {
      __syncthreads();
      if (lane == 63) w.red32[wave] = ti;
      __syncthreads();
#pragma unroll
      for (int o = 0; o < NT / 64; ++o) {
        if (o < wave) tie_before += w.red32[o];
        tie_all += w.red32[o];
      }
    } else {
      tie_all = __shfl(ti, 63, 64);
    }
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      u[j] = 0;
      if (v[j] > cut.value) {
        const double y = log2_weight(v[j], m, r.c);
        if (y >= r.ymin) u[j] = weight_units(y, q.shift);
      } else if (one && v[j] == cut.value) {
        if (tie_before < left) u[j] = one;
        ++tie_before;
      }
      sum += u[j];
    }
    uint64_t si = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint64_t o = __shfl_up(si, off, 64);
      if (lane >= off) si += o;
    }
    uint64_t before = si - sum, here = 0;
    if constexpr (NT > 64) {
      __syncthreads();
      if (lane == 63) w.red64[wave] = si;
      __syncthreads();
#pragma unroll
      for (int o = 0; o < NT / 64; ++o) {
        if (o < wave) before += w.red64[o];
        here += w.red64[o];
      }
    } else {
      here = __shfl(si, 63, 64);
    }
    if (here > target) {   // it is in this tile, and one thread has it
      if (before <= target && before + sum > target) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (before <= target && before + u[j] > target) {
            q.actions[row] = i0 + j;
            q.log_probs[row] = log_prob_of(v[j], m, r, total, q.shift);
          }
          before += u[j];
        }
      }
      return;
    }
    target -= here;
    left -= tie_all < left ? tie_all : left;
  }
}

// -1 for a row that has no distribution or nothing to choose from; true if it was one
__device__ __forceinline__ bool no_draw(const SampleArgs& q, int64_t row, float m, bool bad) {
  if (!bad && m > -INFINITY) return false;
  if (threadIdx.x == 0) {
    q.actions[row] = -1;
    q.log_probs[row] = bad ? __builtin_nanf("") : 0.f;
    if (bad) *q.err = 1;
  }
  return true;
}

// A workgroup per row: the maximum, the cut where a filter asks for one, the kept mass of each wave's segment, the draw.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_row_kernel(const T* __restrict__ logits, int64_t stride, int64_t A, SampleArgs q) {
  __shared__ RowWork<T, NT> w;
  constexpr int kWaves = NT / 64;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * stride;
  const Row r = row_settings(q, row);
  bool bad;
  const float m = part_max<T, NT>(x, 0, A, bad, w.red32);
  if (no_draw(q, row, m, bad)) return;
  Cut cut{-INFINITY, 0, 0};
  uint64_t total = 0;
  const bool hist = needs_histogram(r);
  if (hist) {
    total = group_sum<uint64_t, NT>(part_histogram(x, 0, A, m, r, q.shift, w), w.red64);
    cut = find_cut(x, A, m, r, q.shift, total, w);
  } else if (r.k == 1) {
    cut = Cut{m, 1, 0};
  }
  const int64_t len = segment_length(A, kWaves);
  const int wave = threadIdx.x >> 6;
  const int64_t begin = wave * len < A ? wave * len : A, end = begin + len < A ? begin + len : A;
  uint64_t mass, all;
  uint32_t ties;
  kept_mass(x, begin, end, m, r, q.shift, cut, !hist && !r.greedy, mass, ties, all);
  if ((threadIdx.x & 63) == 0) {
    w.seg_mass[wave] = mass;
    w.seg_ties[wave] = ties;
  }
  if (!hist) total = group_sum<uint64_t, NT>((threadIdx.x & 63) == 0 ? all : 0, w.red64);
  __syncthreads();
  pick(x, A, m, r, q, row, cut, total, w.seg_mass, w.seg_ties, kWaves, len, w);
}

static inline int sample_shift(int64_t A) {
  int bits = 0;
  while (((int64_t)1 << bits) < A) ++bits;
  return 62 - bits < 51 ? 62 - bits : 51;
}

template <typename T>
static int sample_run(const T* logits, int64_t stride, int64_t B, int64_t A, const SampleArgs& q, hipStream_t s) {
  if (A <= 64) {
    const int lanes = A <= 8 ? 8 : A <= 16 ? 16 : A <= 32 ? 32 : 64;
    const int grid = (int)((B * lanes + 255) / 256);
    if (lanes == 8) sample_small_kernel<T, 8><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
    else if (lanes == 16) sample_small_kernel<T, 16><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
    else if (lanes == 32) sample_small_kernel<T, 32><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
    else sample_small_kernel<T, 64><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
  } else if (A <= 2048) {
    sample_row_kernel<T, 64><<<(int)B, 64, 0, s>>>(logits, stride, A, q);
  } else if (A <= 16384) {
    sample_row_kernel<T, 256><<<(int)B, 256, 0, s>>>(logits, stride, A, q);
  } else {
    sample_row_kernel<T, 1024><<<(int)B, 1024, 0, s>>>(logits, stride, A, q);
  }
  return check_launch();
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
  if (A > kSampleMaxActions || B > 0xffffffffLL / 1024) return PARLHIP_ENOSUP;   // one launch's threads
  if (!temperature && !(temperature_all >= 0.f && temperature_all < INFINITY)) return PARLHIP_EINVAL;
  if (!top_p && !(top_p_all >= 0.f)) return PARLHIP_EINVAL;
  if (!min_p && !(min_p_all >= 0.f && min_p_all <= 1.f)) return PARLHIP_EINVAL;
  if (B == 0) return PARLHIP_OK;
  if (!logits || !uniforms || !actions || !log_probs) return PARLHIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == PARLHIP_F32 ? 3 : 1)) return PARLHIP_EINVAL;
  SampleArgs q{uniforms, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all,
               actions, log_probs, device_error_flag(), sample_shift(A)};
  if (!q.err) return PARLHIP_ELAUNCH;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PARLHIP_F32) return sample_run((const float*)logits, row_stride, B, A, q, s);
  if (dtype == PARLHIP_BF16) return sample_run((const bf16_t*)logits, row_stride, B, A, q, s);
  return sample_run((const f16_t*)logits, row_stride, B, A, q, s);
}
