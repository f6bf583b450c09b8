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
// hundred over 131,072 actions: the border between two actions has to be right to far less than their weights.)  So every
// form reads the row for its maximum before it forms a weight.  Sums of stretches relative to their own maxima would need
// no such pass, but count what is under 2^-42 of the row's largest, and round every weight at another place.
//
// No sort.  Rows of at most 64 actions (512 where nothing has to be ranked) lie in the registers of a wave.  Longer rows:
//   no filter   one pass for the maximum of every 4 KB, one in which every wave sums the weights of 4 KB at a time; the piece
//               that the draw falls into is found among the sums and scanned.
//   filters     what they keep is "larger than a cut value, and the first few that equal it".  One pass for the maximum,
//               one that adds masses (and counts, for top-k) into 256 classes of -log2 w, for each segment of the
//               row; the class that holds the border is found by a scan and taken apart on a list of its
//               values in LDS, by the same histogram over ever fewer bits (or on the row itself, where a flat row puts
//               more values into one class than the list takes).  The classes above the border and the list give the
//               kept mass of every segment, and the segment that the draw falls into is scanned.
// Rows of up to 4,096 actions do that in one wave each.  Above, every pass over the rows is a launch of its own over segments of
// all rows, which fills the card whether the rows are many or few and long, and a workgroup per row finishes.
//
// Measured (a large copy on this card moves 4.9 TB/s): 1,024 x 131,072 bf16 without filters 140 to 144 us, 55 us of which one
// read of the 268 MB would take; under the tracer 40 for the maxima (HBM and cache), 102 for the masses (the vector unit, which
// issues in 91 % of its slots, 25 instructions a value), 8 for the finish.  Sums relative to the pieces' own maxima, in one
// pass, took 110 and were another distribution (above).  1,024 x 100,003 with top-p 0.95: 31 us for the maxima, 84 for the
// classes (24 instructions a value), 93 for the finish (a pass over the row by each workgroup, and the chain of scans behind
// it), 205 to 212 for the call.  One row of 131,072 with top-k and top-p: 26 us, three launches of 4, 7 and 14, the last a
// chain of scans.  Values that lie close together meet in few classes: 1,024 x 131,072 with top-p 0.9 takes 217 us at a
// spread of 2.5 and 625 at 0.3.
#include "common.hpp"
#include "logits_common.hpp"
#include <algorithm>

namespace parlhip {

constexpr int64_t kSampleMaxActions = (int64_t)1 << 20;
constexpr double kFloorLog2 = -42.0;     // weights under 2^-42 are 0
constexpr float kFloor = 0x1p-42f;
constexpr int kBins = 256;
constexpr double kPerHalving = 6.0;
constexpr int kLastBin = 252;            // 42 halvings
constexpr int kMaxParts = 64;            // segments of a row

// Running sums over the lanes of a wave, by the data-parallel moves of the vector unit (a shuffle goes through LDS and takes
// several times as long): within rows of 16 lanes, then the rows' last lanes into the rows behind them.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_move(uint32_t x) {   // 0 where there is no source
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t lane_move(uint64_t x) {
  return (uint64_t)lane_move<CTRL, ROWS>((uint32_t)x) | (uint64_t)lane_move<CTRL, ROWS>((uint32_t)(x >> 32)) << 32;
}
template <typename X>
__device__ __forceinline__ X wave_scan(X x) {
  x += lane_move<0x111, 0xf>(x);   // from 1, 2, 4, 8 lanes below, inside a row
  x += lane_move<0x112, 0xf>(x);
  x += lane_move<0x114, 0xf>(x);
  x += lane_move<0x118, 0xf>(x);
  x += lane_move<0x142, 0xa>(x);   // lane 15 of the row below, into rows 1 and 3
  x += lane_move<0x143, 0xc>(x);   // lane 31, into rows 2 and 3
  return x;
}
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }
__device__ __forceinline__ uint64_t last_lane(uint64_t x) {
  return (uint64_t)last_lane((uint32_t)x) | (uint64_t)last_lane((uint32_t)(x >> 32)) << 32;
}
template <typename X>
__device__ __forceinline__ X wave_total(X x) { return last_lane(wave_scan(x)); }

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
  r.ymin = min_p > kFloor ? fmax(kFloorLog2, log2((double)min_p)) : kFloorLog2;
  return r;
}

// whether anything but the maximum and the whole mass is asked for
__device__ __forceinline__ bool filtered(const Row& r) { return !r.greedy && (r.k > 0 || r.top_p < 1.f || r.ymin > kFloorLog2); }

// whether nothing but the maximum and the whole mass is
__device__ __forceinline__ bool weighed(const Row& r) { return !r.greedy && !filtered(r); }

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

// 2^y in units of 2^-shift, rounded to nearest, 0 where y < -42, plus kUnitsBase; y <= 0, shift <= 51.  2^r = 1 + r q(r) on
// |r| <= 1/2 with q the interpolation of (2^r - 1) / r at seven Chebyshev nodes: relative error 1.1e-10, and 2^0 is 1.
// (The error is a function of r alone, so most of it cancels between a running sum and the whole: over 131,072 actions a
// border moves by some 1e-13 of the mass.)  Adding 2^52 to a number below it leaves its nearest integer in the low bits.  No
// branch: the weights of a load are formed side by side, 15 instructions of the vector unit each (13 where the caller knows
// that y >= -42: CHECK false); float64 runs at float32's rate here.
// a b + c with c in scalar registers: left to itself the compiler copies the constant into the result's registers first, one
// instruction more for every step
__device__ __forceinline__ double fma_const(double a, double b, double c) {
  double d;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
  return d;
}
constexpr uint64_t kUnitsBase = 0x4330000000000000ULL;
template <bool CHECK = true>
__device__ __forceinline__ uint64_t weight_bits(double y, int shift) {
  if constexpr (CHECK) y = fmax(y, -1000.0);   // -inf: no NaN below
  // adding 1.5 * 2^52 rounds to an integer, which then is the low word: n + shift + 1023, the exponent of the weight
  const double magic = 0x1.8p52 + (shift + 1023), t = y + magic, r = y - (t - magic);
  double p = 0x1.00a581594758ep-16;
  p = fma_const(p, r, 0x1.443fffc90db59p-13);
  p = fma_const(p, r, 0x1.5d879ead06a82p-10);
  p = fma_const(p, r, 0x1.3b2a1b7152befp-7);
  p = fma_const(p, r, 0x1.c6b08d883dca1p-5);
  p = fma_const(p, r, 0x1.ebfbe045f4d3cp-3);
  p = fma_const(p, r, 0x1.62e42fefa39efp-1);
  p = __builtin_fma(p, r, 1.0);
  const double scale = __hiloint2double(!CHECK || y >= kFloorLog2 ? __double2loint(t) << 20 : 0, 0);   // 2^(n + shift)
  return (uint64_t)__double_as_longlong(__builtin_fma(p, scale, 0x1p52));
}
__device__ __forceinline__ uint64_t weight_units(double y, int shift) { return weight_bits(y, shift) - kUnitsBase; }

// the class of a weight: six for each halving, 0 for the largest, 252 for 2^-42
__device__ __forceinline__ int weight_bin(double y) { return (int)(y * -kPerHalving); }

// u * mass rounded down to whole units, exactly (u itself is taken to a multiple of 2^-53): the draw is the first action whose
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
// the row's lanes directly.  1,024 rows of 18 take 4 us (one launch), 65,536 of them 20 us, with top-p 39.
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
  if (__any(r.k == 1)) {   // the first of the largest
    const uint64_t largest = __ballot(x == m) >> (threadIdx.x % 64 / LP * LP);
    if (r.k == 1) keep = keep && x == m && !(largest & (((uint64_t)1 << sub) - 1));
  }
  if (__any(r.k > 1 || r.top_p < 1.f)) {
    int position = 0;
    uint64_t before = 0;
    for (int j = 0; j < A; ++j) {
      float xj;
      uint64_t uj;
      if constexpr (LP == 64) {   // one row: through scalar registers
        xj = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), j));
        uj = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, j) |
             (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), j) << 32;
      } else {
        xj = __shfl(x, j, LP);
        uj = __shfl(u, j, LP);
      }
      const bool above = xj > x || (xj == x && j < sub);   // one without weight adds none, and is above none that has
      position += above;
      before += above ? uj : 0;
    }
    keep = keep && (r.k <= 1 || position < r.k);
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

// 64 < A <= 64 E, and neither top-k beyond 1 nor top-p: a wave per row, a lane holds E neighbouring actions.  (A filter that
// ranks needs the classes below.)  65,536 rows of 100 take 36 us, where the wave kernel below takes 143.
template <typename T, int E>
__global__ __launch_bounds__(256) void sample_lanes_kernel(const T* __restrict__ logits, int64_t stride, int64_t B, int A,
                                                           SampleArgs q) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= B) return;   // whole wave
  const T* x = logits + row * stride;
  float v[E];
  float m = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = lane * E + e;
    v[e] = i < A ? to_f32(x[i]) : -INFINITY;
    bad |= !(v[e] < INFINITY);
    m = fmaxf(m, v[e]);
  }
  bad = __any(bad);
  m = wave_max_f32(m);
  if (bad || m == -INFINITY) {
    if (lane == 0) {
      q.actions[row] = -1;
      q.log_probs[row] = bad ? __builtin_nanf("") : 0.f;
      if (bad) *q.err = 1;
    }
    return;
  }
  const Row r = row_settings(q, row);
  uint64_t u[E], kept = 0, all = 0;
  bool had = false;   // the largest value, in an action before
  const uint64_t largest = __ballot(([&] {
    bool any = false;
#pragma unroll
    for (int e = 0; e < E; ++e) any |= v[e] == m;
    return any;
  })());
  had = r.k == 1 && (largest & (((uint64_t)1 << lane) - 1)) != 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const double y = log2_weight(v[e], m, r.c);
    u[e] = weight_units(y, q.shift);
    all += u[e];
    bool keep = y >= r.ymin;
    if (r.k == 1) {
      keep = v[e] == m && !had;
      had |= keep;
    }
    if (!keep) u[e] = 0;
    kept += u[e];
  }
  const uint64_t total = wave_total(all), run = wave_scan(kept);
  const uint64_t target = draw_target(q.uniforms[row], last_lane(run));
  uint64_t before = run - kept;
  if (before <= target && run > target) {   // one lane
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (before <= target && before + u[e] > target) {
        q.actions[row] = lane * E + e;
        q.log_probs[row] = log_prob_of(v[e], m, r, total, q.shift);
      }
      before += u[e];
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Longer rows: a workgroup of NT threads for a row or a part of one.

// f(v, i) for the vectors of [begin, end) of a row, by the threads tid < NT, four loads in flight: v are the V elements from
// i on; what lies behind the end is -inf, which has no weight.  begin is a multiple of V.  All threads make all rounds.
template <typename T, int NT, typename F>
__device__ __forceinline__ void for_each_vec(const T* __restrict__ x, int begin, int end, int tid, F&& f) {
  constexpr int V = Vec16<T>::n;
  int base = begin;
  for (; base + 4 * NT * V <= end; base += 4 * NT * V) {
    Vec16<T> v[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) v[a].load(x + base + (a * NT + tid) * V);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      float g[V];
      v[a].unpack(g);
      f(g, base + (a * NT + tid) * V);
    }
  }
  for (; base < end; base += NT * V) {
    const int i = base + tid * V;
    float g[V];
    if (i + V <= end) {
      Vec16<T> v;
      v.load(x + i);
      v.unpack(g);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = i + j < end ? to_f32(x[i + j]) : -INFINITY;
    }
    f(g, i);
  }
}

// the pieces of a row whose maxima and masses are kept: what a wave loads at a time
template <typename T>
__host__ __device__ constexpr int piece_length() { return 64 * 4 * 16 / (int)sizeof(T); }

struct Pieces {          // of one row
  uint64_t* mass;
  float* max;            // NaN: a NaN or +inf was among them
};

template <int NT>
struct RowWork {
  static constexpr int kWaves = NT / 64;
  static constexpr int kList = NT == 1024 || NT == 64 ? 512 : 1024;   // of each wave
  uint64_t mass[kBins];                  // of the row, or of the class that is being taken apart
  uint32_t count[kBins];
  uint32_t list[kWaves][kList];          // the values (keys; 0: none) of a class and the segments that they are in
  uint8_t list_seg[kWaves][kList];
  uint32_t list_n[kWaves];
  uint64_t seg_mass[kMaxParts];
  uint32_t seg_ties[kMaxParts];
  uint64_t red64[kWaves];
  uint32_t red32[kWaves];
  uint32_t lo, hi;                       // of the listed class
  bool listed;                           // whether the lists took all of it
  int bin;                               // what the scan found
  uint64_t above_mass;
  uint32_t above_count;
  int found;
  uint64_t found_target;
};

// a row, its settings, and the segments that its sums are kept by
template <typename T>
struct RowView {
  const T* x;
  int A;
  float m;
  Row r;
  int shift;
  int n_seg, seg_len;                    // segment s: [s * seg_len, ...); seg_len is a multiple of every vector
  const uint64_t* seg_hist;              // [n_seg][kBins]: masses of the classes
  const uint32_t* seg_count;             // and counts
  const uint32_t* seg_first;             // [n_seg][kBins], or NULL: where a class begins among the segment's values,
  const float* values;                   // [n_seg][seg_len], which then are in the order of their classes
};

template <typename X, int NT>
__device__ __forceinline__ X group_sum(X v, X* lds) {   // every thread gets the sum
  v = wave_total(v);
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

// the largest value over the group; NaN if any thread's is
template <int NT>
__device__ __forceinline__ float group_max(float m, uint32_t* lds) {
  const bool bad = __any(m != m);
  m = bad ? __builtin_nanf("") : wave_max_f32(m);
  if constexpr (NT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = bad ? 0xffffffffu : value_key(m);   // no number has that key
    __syncthreads();
    uint32_t k = lds[0];
#pragma unroll
    for (int o = 1; o < NT / 64; ++o) k = lds[o] > k ? lds[o] : k;
    m = k == 0xffffffffu ? __builtin_nanf("") : key_value(k);
  }
  return m;
}

__device__ __forceinline__ float maximum3(float a, float b, float c) {   // NaN if any is
  return __builtin_elementwise_maximum(a, __builtin_elementwise_maximum(b, c));
}

// piece p of a row by the lanes of a wave; -inf, which has no weight, behind the row's end
template <typename T>
__device__ __forceinline__ void load_piece(const T* __restrict__ x, int A, int p, Vec16<T> (&raw)[4]) {
  constexpr int V = Vec16<T>::n, kLen = piece_length<T>();
  const int base = p * kLen + (int)(threadIdx.x & 63) * V;
  if (p * kLen + kLen <= A) {
#pragma unroll
    for (int a = 0; a < 4; ++a) raw[a].load(x + base + a * 64 * V);
    return;
  }
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const int i0 = base + a * 64 * V;
    if (i0 + V <= A) {
      raw[a].load(x + i0);
    } else {
      float g[V];
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = i0 + j < A ? to_f32(x[i0 + j]) : -INFINITY;
      raw[a].pack(g);   // exact: they came from this type
    }
  }
}

// the maxima of the pieces [first, last) of a row, one after the other by each of the waves `wave` of `waves`
template <typename T>
__device__ __forceinline__ void max_pieces(const T* __restrict__ x, int A, int first, int last, int wave, int waves,
                                           float* __restrict__ max) {
  constexpr int V = Vec16<T>::n;
  for (int p = first + wave; p < last; p += waves) {
    Vec16<T> raw[4];
    load_piece(x, A, p, raw);
    float m = -INFINITY;   // a NaN stays
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int j = 0; j < V; j += 2) m = maximum3(m, raw[a].get(j), raw[a].get(j + 1));
    m = group_max<64>(m < INFINITY ? m : __builtin_nanf(""), nullptr);
    if ((threadIdx.x & 63) == 0) max[p] = m;
  }
}

// their masses, with the row's maximum m
template <typename T>
__device__ __forceinline__ void sum_pieces(const T* __restrict__ x, int A, float m, double c, int shift, int first, int last,
                                           int wave, int waves, const Pieces& out) {
  constexpr int V = Vec16<T>::n, kLen = piece_length<T>();
  for (int p = first + wave; p < last; p += waves) {
    const int loads = A - p * kLen >= kLen ? 4 : (A - p * kLen + 64 * V - 1) / (64 * V);   // of the wave
    uint64_t mass = 0;
    if (log2_weight(out.max[p], m, c) >= kFloorLog2) {   // else nothing in it has a weight
      Vec16<T> raw[4];
      load_piece(x, A, p, raw);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        if (a >= loads) break;
#pragma unroll
        for (int j = 0; j < V; ++j) mass += weight_bits(log2_weight(raw[a].get(j), m, c), shift);
      }
      mass -= (uint64_t)(loads * V) * kUnitsBase;
      mass = wave_total(mass);
    }
    if ((threadIdx.x & 63) == 0) out.mass[p] = mass;
  }
}

// the row's maximum, from those of its pieces
template <typename T, int NT>
__device__ __forceinline__ float row_max(const Pieces& p, int A, uint32_t* lds) {
  const int n = (A + piece_length<T>() - 1) / piece_length<T>();
  float m = -INFINITY;
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += NT) {
    const float o = p.max[i];
    bad |= o != o;
    m = fmaxf(m, o);
  }
  return group_max<NT>(bad ? __builtin_nanf("") : m, lds);
}

// masses (and counts) of the classes of [begin, end), added into `mass` and `count` by NT threads
template <typename T, int NT>
__device__ __forceinline__ void add_classes(const T* __restrict__ x, int begin, int end, float m, const Row& r, int shift,
                                            uint64_t* mass, uint32_t* count, bool counts) {
  constexpr int V = Vec16<T>::n;
  for_each_vec<T, NT>(x, begin, end, threadIdx.x, [&](const float (&v)[V], int) {
    double y[V];
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] = log2_weight(v[j], m, r.c);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (y[j] >= kFloorLog2) {   // the additions need the branch; with the weight inside it the registers allow twice the waves
        const int b = weight_bin(y[j]);
        atomicAdd((unsigned long long*)&mass[b], (unsigned long long)(weight_bits<false>(y[j], shift) - kUnitsBase));
        if (counts) atomicAdd(&count[b], 1u);
      }
    }
  });
}

// the row's classes: the sum of its segments' -> w.mass, w.count; every thread gets the whole mass
template <typename T, int NT>
__device__ __forceinline__ uint64_t sum_classes(const RowView<T>& v, RowWork<NT>& w) {
  constexpr int kGroups = NT > kBins ? NT / kBins : 1;   // of segments, side by side
  __syncthreads();
  if constexpr (kGroups > 1) {
    if (threadIdx.x < kBins) { w.mass[threadIdx.x] = 0; w.count[threadIdx.x] = 0; }
    __syncthreads();
  }
  uint64_t total = 0;
  for (int b = threadIdx.x % kBins; b < kBins; b += NT) {
    uint64_t s = 0;
    uint32_t c = 0;
    int g = threadIdx.x / kBins;
    for (; g + 7 * kGroups < v.n_seg; g += 8 * kGroups) {   // eight loads in flight
      uint64_t t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = v.seg_hist[(g + j * kGroups) * kBins + b];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += t[j];
      if (v.r.k > 0) {
        uint32_t n[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) n[j] = v.seg_count[(g + j * kGroups) * kBins + b];
#pragma unroll
        for (int j = 0; j < 8; ++j) c += n[j];
      }
    }
    for (; g < v.n_seg; g += kGroups) {
      s += v.seg_hist[g * kBins + b];
      if (v.r.k > 0) c += v.seg_count[g * kBins + b];
    }
    if constexpr (kGroups > 1) {
      atomicAdd((unsigned long long*)&w.mass[b], (unsigned long long)s);
      atomicAdd(&w.count[b], c);
    } else {
      w.mass[b] = s;
      w.count[b] = c;
    }
    total += s;
  }
  return group_sum<uint64_t, NT>(total, w.red64);
}

// Finds the class that reaches `need` (a count, or a mass) counted from class 0 -> w.bin and what lies above it.  The first
// wave scans, four classes a lane.  bin = -1: the classes together do not reach it.
template <int NT>
__device__ __forceinline__ void scan_classes(RowWork<NT>& w, bool by_mass, uint64_t need) {
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
    uint32_t ca = wave_scan(cs) - cs;   // above this lane's classes
    uint64_t sa = wave_scan(ss) - ss;
    int bin = -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool here = by_mass ? (sa < need && sa + s[j] >= need) : ((uint64_t)ca < need && (uint64_t)ca + c[j] >= need);
      if (here) {
        bin = 4 * l + j;
        w.above_count = ca;
        w.above_mass = sa;
      }
      ca += c[j];
      sa += s[j];
    }
    const uint64_t who = __ballot(bin >= 0);   // one lane, or none
    bin = who ? __shfl(bin, __ffsll((unsigned long long)who) - 1, 64) : -1;
    if (l == 0) w.bin = bin;
  }
  __syncthreads();
}

struct Cut {
  float value;          // kept: larger than this, and the first `ties` that equal it
  uint32_t ties;
  uint64_t above;       // mass of the larger ones
};

// f(key, segment) for the listed class, if the lists took it
template <int NT, typename F>
__device__ __forceinline__ void for_listed(RowWork<NT>& w, F&& f) {
  const int wave = threadIdx.x >> 6;
  const uint32_t n = w.list_n[wave];
  for (uint32_t i = threadIdx.x & 63; i < n; i += 64) f(w.list[wave][i], (int)w.list_seg[wave][i]);
}

// f(value) for class `bin` of segment s, where the values lie by class; by the lanes of a wave
template <typename T, typename F>
__device__ __forceinline__ void for_stretch(const RowView<T>& v, int s, int bin, F&& f) {
  const uint32_t last = v.seg_first[s * kBins + bin + 1];
  for (uint32_t i = v.seg_first[s * kBins + bin] + (threadIdx.x & 63); i < last; i += 64) f(v.values[s * v.seg_len + i]);
}

// The values of class `bin` -> w.list (w.listed: all of them), their range -> w.lo, w.hi.
template <typename T, int NT>
__device__ __forceinline__ void gather_class(const RowView<T>& v, RowWork<NT>& w, int bin) {
  constexpr int V = Vec16<T>::n, kList = RowWork<NT>::kList;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (threadIdx.x == 0) { w.listed = true; w.lo = 0xffffffffu; w.hi = 0; }
  uint32_t n = 0;   // of this wave's list, the same in every lane
  if (v.values) {
    // the class lies in one stretch of each segment's values: lane s has the stretch of segment s
    const int bin0 = lane * kBins + bin;
    const uint32_t from = lane < v.n_seg ? v.seg_first[bin0] : 0, to = lane < v.n_seg ? v.seg_first[bin0 + 1] : 0;
    for (int s = wave; s < v.n_seg; s += NT / 64) {
      const uint32_t first = __shfl(from, s, 64), last = __shfl(to, s, 64);
      for (uint32_t i = first + lane; i < last; i += 64) {
        const uint32_t at = n + (i - first);
        if (at < kList) {
          w.list[wave][at] = __float_as_uint(v.values[s * v.seg_len + i]);
          w.list_seg[wave][at] = (uint8_t)s;
        }
      }
      n += last - first;
    }
  } else {
    // A little more than the class' range: one comparison for a load's values together where they are all below it, else two
    // for each.  A wave appends what it finds to a list of its own; whether it is of the class is seen afterwards, on
    // the list (float64 in this loop would run for every second load of a wave).
    const double step = 1.0 / kPerHalving / v.r.c, slack = 1e-6 * (fabs((double)v.m) + (bin + 1) * step) + 1e-37;
    const float top = (float)((double)v.m - bin * step + slack);
    const float bottom = bin == kLastBin ? -3.4028235e38f : (float)((double)v.m - (bin + 1) * step - slack);
    const uint32_t inv = (65536u + (v.seg_len >> 11) - 1) / (v.seg_len >> 11);   // segments are multiples of 2,048
    for_each_vec<T, NT>(v.x, 0, v.A, threadIdx.x, [&](const float (&g)[V], int i) {
      float most = g[0];
#pragma unroll
      for (int j = 1; j < V; ++j) most = fmaxf(most, g[j]);
      if (!__any(most >= bottom)) return;
      const uint32_t seg = ((uint32_t)(i >> 11) * inv) >> 16;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool hit = g[j] <= top && g[j] >= bottom;
        const uint64_t mask = __ballot(hit);
        if (mask) {
          const uint32_t at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
          if (hit && at < kList) {
            w.list[wave][at] = __float_as_uint(g[j]);
            w.list_seg[wave][at] = (uint8_t)seg;
          }
          n += (uint32_t)__popcll(mask);
        }
      }
    });
  }
  __syncthreads();
  if (lane == 0) {
    w.list_n[wave] = n < kList ? n : kList;
    if (n > kList) w.listed = false;
  }
  __syncthreads();
  uint32_t lo = 0xffffffffu, hi = 0;
  const auto of_class = [&](float x) {
    const double y = log2_weight(x, v.m, v.r.c);
    if (!(y >= kFloorLog2) || weight_bin(y) != bin) return 0u;
    const uint32_t k = value_key(x);
    lo = k < lo ? k : lo;
    hi = k > hi ? k : hi;
    return k;
  };
  if (w.listed)
    for (uint32_t i = lane; i < n; i += 64) w.list[wave][i] = of_class(__uint_as_float(w.list[wave][i]));
  else if (v.values)
    for (int s = wave; s < v.n_seg; s += NT / 64) for_stretch(v, s, bin, of_class);
  else
    for_each_vec<T, NT>(v.x, 0, v.A, threadIdx.x, [&](const float (&g)[V], int) {
#pragma unroll
      for (int j = 0; j < V; ++j) of_class(g[j]);
    });
  if (hi != 0) {
    atomicMin(&w.lo, lo);
    atomicMax(&w.hi, hi);
  }
  __syncthreads();
}

// The value at which the count (or mass) counted from the top reaches `need`, inside the listed class.
template <typename T, int NT>
__device__ __forceinline__ Cut refine(const RowView<T>& v, RowWork<NT>& w, int bin, uint64_t above_mass,
                                      uint64_t above_count, bool by_mass, uint64_t need) {
  constexpr int V = Vec16<T>::n;
  uint32_t lo = w.lo, hi = w.hi;
  const bool listed = w.listed;
  while (lo < hi) {   // at least 8 bits less each time
    int sh = 24 - __clz(hi - lo);
    if (sh < 0) sh = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += NT) { w.mass[i] = 0; w.count[i] = 0; }
    __syncthreads();
    auto add = [&](uint32_t k) {
      if (k >= lo && k <= hi) {
        const int b = (int)((hi - k) >> sh);
        atomicAdd(&w.count[b], 1u);
        atomicAdd((unsigned long long*)&w.mass[b],
                  (unsigned long long)weight_units(log2_weight(key_value(k), v.m, v.r.c), v.shift));
      }
    };
    if (listed)
      for_listed(w, [&](uint32_t k, int) { add(k); });
    else if (v.values)
      for (int s = threadIdx.x >> 6; s < v.n_seg; s += NT / 64) for_stretch(v, s, bin, [&](float x) { add(value_key(x)); });
    else
      for_each_vec<T, NT>(v.x, 0, v.A, threadIdx.x, [&](const float (&g)[V], int) {
#pragma unroll
        for (int j = 0; j < V; ++j) add(value_key(g[j]));
      });
    scan_classes(w, by_mass, need - (by_mass ? above_mass : above_count));
    const int b = w.bin < 0 ? 0 : w.bin;   // it is there: the class as a whole reaches `need`
    above_mass += w.above_mass;
    above_count += w.above_count;
    const uint32_t top = hi - ((uint32_t)b << sh), width = (1u << sh) - 1;
    hi = top;
    lo = top - lo > width ? top - width : lo;
  }
  Cut cut;
  cut.value = key_value(hi);
  cut.above = above_mass;
  const uint64_t one = weight_units(log2_weight(cut.value, v.m, v.r.c), v.shift);
  cut.ties = by_mass ? (uint32_t)((need - above_mass + one - 1) / one) : (uint32_t)(need - above_count);
  return cut;
}

// The cut of top-k and top-p, from the row's classes in w.mass, w.count.  `listed` is the class in w.list afterwards.
template <typename T, int NT>
__device__ __forceinline__ Cut find_cut(const RowView<T>& v, RowWork<NT>& w, uint64_t total, int& listed) {
  constexpr int kKeep = NT < kBins ? kBins / NT : 1;
  Cut cut{-INFINITY, 0, 0};
  uint64_t mass_k = total;
  listed = -1;
  if (v.r.k > 0) {
    scan_classes(w, false, (uint64_t)v.r.k);
    const int bin = w.bin;
    if (bin >= 0) {   // else fewer than k have any weight
      const uint64_t am = w.above_mass, ac = w.above_count;
      uint64_t keep[kKeep];   // the masses are needed again for top-p
#pragma unroll
      for (int j = 0; j < kKeep; ++j) keep[j] = w.mass[(threadIdx.x + j * NT) % kBins];
      gather_class(v, w, bin);
      listed = bin;
      cut = refine(v, w, bin, am, ac, false, (uint64_t)v.r.k);
      mass_k = cut.above + (uint64_t)cut.ties * weight_units(log2_weight(cut.value, v.m, v.r.c), v.shift);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kKeep; ++j) w.mass[(threadIdx.x + j * NT) % kBins] = keep[j];
    }
  }
  if (v.r.top_p < 1.f) {
    const uint64_t need = top_p_mass(v.r.top_p, mass_k);
    scan_classes(w, true, need);
    const int bin = w.bin < 0 ? 0 : w.bin;   // it is there: need <= total
    const uint64_t am = w.above_mass;
    if (bin != listed) gather_class(v, w, bin);
    listed = bin;
    const Cut p = refine(v, w, bin, am, 0, true, need);
    if (p.value > cut.value || (p.value == cut.value && p.ties < cut.ties)) cut = p;
  }
  return cut;
}

// The kept mass and the values at the cut of every segment -> w.seg_mass, w.seg_ties.
template <typename T, int NT>
__device__ __forceinline__ void sum_segments(const RowView<T>& v, RowWork<NT>& w, const Cut& cut, int listed) {
  constexpr int V = Vec16<T>::n, kWaves = NT / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double y_cut = cut.value > -INFINITY ? log2_weight(cut.value, v.m, v.r.c) : kFloorLog2;
  const int bin = weight_bin(fmax(y_cut, v.r.ymin));   // above it everything is kept, below it nothing
  if (bin != listed) gather_class(v, w, bin);
  __syncthreads();
  if (w.listed || v.values) {
    for (int s = wave; s < v.n_seg; s += kWaves) {
      uint64_t mass = 0;
      uint32_t ties = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (64 * j + lane < bin) mass += v.seg_hist[s * kBins + 64 * j + lane];
      if (!w.listed) {
        for_stretch(v, s, bin, [&](float x) {
          const double y = log2_weight(x, v.m, v.r.c);
          ties += x == cut.value;
          mass += x > cut.value && y >= v.r.ymin ? weight_units(y, v.shift) : 0;
        });
        ties = wave_total(ties);
      }
      mass = wave_total(mass);
      if (lane == 0) {
        w.seg_mass[s] = mass;
        w.seg_ties[s] = ties;
      }
    }
    __syncthreads();
    if (w.listed)
      for_listed(w, [&](uint32_t k, int s) {
        const float x = key_value(k);
        const double y = log2_weight(x, v.m, v.r.c);
        if (x == cut.value)   // x is NaN where there is none
          atomicAdd(&w.seg_ties[s], 1u);
        else if (x > cut.value && y >= v.r.ymin)
          atomicAdd((unsigned long long*)&w.seg_mass[s], (unsigned long long)weight_units(y, v.shift));
      });
  } else {   // a flat row: over the whole of it again
    for (int s = wave; s < v.n_seg; s += kWaves) {
      const int begin = s * v.seg_len < v.A ? s * v.seg_len : v.A, end = begin + v.seg_len < v.A ? begin + v.seg_len : v.A;
      uint64_t mass = 0;
      uint32_t ties = 0;
      for_each_vec<T, 64>(v.x, begin, end, lane, [&](const float (&g)[V], int) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double y = log2_weight(g[j], v.m, v.r.c);
          const uint64_t u = weight_units(y, v.shift);
          mass += g[j] > cut.value && y >= v.r.ymin ? u : 0;
          ties += g[j] == cut.value;
        }
      });
      mass = wave_total(mass);
      ties = wave_total(ties);
      if (lane == 0) {
        w.seg_mass[s] = mass;
        w.seg_ties[s] = ties;
      }
    }
  }
  __syncthreads();
}

// Scans [begin, end) in index order for the first action whose running kept mass exceeds target; of the values at the cut
// the first `left` are kept, each with `one` (0: none are).  It is there: the range's mass is the same sum.
template <typename T, int NT>
__device__ __forceinline__ void scan_draw(const RowView<T>& v, RowWork<NT>& w, const SampleArgs& q, int64_t row, int begin,
                                          int end, const Cut& cut, uint64_t one, uint32_t left, uint64_t target,
                                          uint64_t total) {
  constexpr int V = Vec16<T>::n;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int base = begin; base < end; base += NT * V) {
    const int i0 = base + (int)threadIdx.x * V;
    float g[V];
    uint64_t u[V];
    if (i0 + V <= end) {
      Vec16<T> raw;
      raw.load(v.x + i0);
      raw.unpack(g);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = i0 + j < end ? to_f32(v.x[i0 + j]) : -INFINITY;
    }
    uint32_t tie_before = 0, tie_all = 0;
    if (one) {   // the same for the whole group
      uint32_t tie = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) tie += g[j] == cut.value;
      const uint32_t run = wave_scan(tie);
      tie_before = run - tie;
      if constexpr (NT > 64) {
        __syncthreads();
        if (lane == 63) w.red32[wave] = run;
        __syncthreads();
#pragma unroll
        for (int o = 0; o < NT / 64; ++o) {
          if (o < wave) tie_before += w.red32[o];
          tie_all += w.red32[o];
        }
      } else {
        tie_all = last_lane(run);
      }
    }
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double y = log2_weight(g[j], v.m, v.r.c);
      u[j] = g[j] > cut.value && y >= v.r.ymin ? weight_units(y, v.shift) : 0;
      if (one && g[j] == cut.value) {
        if (tie_before < left) u[j] = one;
        ++tie_before;
      }
      sum += u[j];
    }
    const uint64_t run = wave_scan(sum);
    uint64_t before = run - sum, here = 0;
    if constexpr (NT > 64) {
      __syncthreads();
      if (lane == 63) w.red64[wave] = run;
      __syncthreads();
#pragma unroll
      for (int o = 0; o < NT / 64; ++o) {
        if (o < wave) before += w.red64[o];
        here += w.red64[o];
      }
    } else {
      here = last_lane(run);
    }
    if (here > target) {   // it is in this tile, and one thread has it
      if (before <= target && before + sum > target) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (before <= target && before + u[j] > target) {
            q.actions[row] = i0 + j;
            q.log_probs[row] = log_prob_of(g[j], v.m, v.r, total, v.shift);
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

// The draw of a filtered row, from its segments' classes.
template <typename T, int NT>
__device__ __forceinline__ void draw_filtered(const RowView<T>& v, RowWork<NT>& w, const SampleArgs& q, int64_t row) {
  const uint64_t total = sum_classes(v, w);
  int listed;
  const Cut cut = find_cut(v, w, total, listed);
  sum_segments(v, w, cut, listed);
  const double y_cut = cut.value > -INFINITY ? log2_weight(cut.value, v.m, v.r.c) : 0.0;
  // the values at the cut are kept if min_p keeps them
  const uint64_t one = cut.value > -INFINITY && y_cut >= v.r.ymin ? weight_units(y_cut, v.shift) : 0;
  // the first wave: a lane for each segment, its kept ties and its mass, their running sums, the draw's segment
  static_assert(kMaxParts == 64, "a lane for each segment");
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const uint32_t keep = one ? cut.ties : 0;
    const uint32_t ties = lane < v.n_seg ? w.seg_ties[lane] : 0;
    const uint32_t tie_before = wave_scan(ties) - ties;
    const uint32_t left = tie_before < keep ? keep - tie_before : 0;
    const uint64_t mass = (lane < v.n_seg ? w.seg_mass[lane] : 0) + (uint64_t)(ties < left ? ties : left) * one;
    const uint64_t run = wave_scan(mass);
    const uint64_t target = draw_target(q.uniforms[row], last_lane(run));
    if (run > target && run - mass <= target) {   // one lane
      w.found = lane;
      w.found_target = target - (run - mass);
      w.lo = left;
    }
  }
  __syncthreads();
  const int s = w.found;
  const uint32_t left = w.lo;
  const uint64_t target = w.found_target;
  const int begin = s * v.seg_len, end = begin + v.seg_len < v.A ? begin + v.seg_len : v.A;
  scan_draw(v, w, q, row, begin, end, cut, one, left, target, total);
}

// The draw of a row without filters, from the masses of its n <= NT pieces.
template <typename T, int NT>
__device__ __forceinline__ void draw_pieces(const RowView<T>& v, RowWork<NT>& w, const SampleArgs& q, int64_t row, const Pieces& p,
                                            int n) {
  constexpr int kLen = piece_length<T>();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = threadIdx.x;
  const uint64_t mass = i < n ? p.mass[i] : 0;
  const uint64_t run = wave_scan(mass);
  uint64_t before = run - mass, total = 0;
  if constexpr (NT > 64) {
    __syncthreads();
    if (lane == 63) w.red64[wave] = run;
    __syncthreads();
#pragma unroll
    for (int o = 0; o < NT / 64; ++o) {
      if (o < wave) before += w.red64[o];
      total += w.red64[o];
    }
  } else {
    total = last_lane(run);
  }
  const uint64_t target = draw_target(q.uniforms[row], total);
  if (before <= target && before + mass > target) {   // one thread
    w.found = i;
    w.found_target = target - before;
  }
  __syncthreads();
  const int begin = w.found * kLen, end = begin + kLen < v.A ? begin + kLen : v.A;
  const Cut all{-INFINITY, 0, 0};
  scan_draw(v, w, q, row, begin, end, all, 0, 0, w.found_target, total);
}

// the largest logit, the first among equals
template <typename T, int NT>
__device__ __forceinline__ void draw_greedy(const RowView<T>& v, RowWork<NT>& w, const SampleArgs& q, int64_t row) {
  constexpr int V = Vec16<T>::n;
  if (threadIdx.x == 0) w.found = 0x7fffffff;
  __syncthreads();
  int first = 0x7fffffff;
  for_each_vec<T, NT>(v.x, 0, v.A, threadIdx.x, [&](const float (&g)[V], int i) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (g[j] == v.m && i + j < first) first = i + j;
  });
  if (first != 0x7fffffff) atomicMin(&w.found, first);
  __syncthreads();
  if (threadIdx.x == 0) {
    q.actions[row] = w.found;
    q.log_probs[row] = 0.f;
  }
}

// -1 for a row that has no distribution or nothing to choose from; true if it was one
__device__ __forceinline__ bool no_draw(const SampleArgs& q, int64_t row, float m) {
  if (m > -INFINITY) return false;
  if (threadIdx.x == 0) {
    const bool bad = m != m;
    q.actions[row] = -1;
    q.log_probs[row] = bad ? m : 0.f;
    if (bad) *q.err = 1;
  }
  return true;
}

// the draw of a row whose maximum, pieces or classes are there
template <typename T, int NT>
__device__ __forceinline__ void draw_row(const RowView<T>& v, RowWork<NT>& w, const SampleArgs& q, int64_t row,
                                         const Pieces& p) {
  if (no_draw(q, row, v.m)) return;
  if (v.r.greedy) draw_greedy(v, w, q, row);
  else if (filtered(v.r)) draw_filtered(v, w, q, row);
  else draw_pieces(v, w, q, row, p, (v.A + piece_length<T>() - 1) / piece_length<T>());
}

// Rows of up to kWaveRow actions: one wave each.
constexpr int kWaveRow = 4096;

template <typename T>
__global__ __launch_bounds__(64) void sample_wave_kernel(const T* __restrict__ logits, int64_t stride, int A, SampleArgs q) {
  constexpr int kPieces = kWaveRow / piece_length<T>();
  __shared__ RowWork<64> w;
  __shared__ uint64_t hist[kBins], piece_mass[kPieces];
  __shared__ uint32_t count[kBins];
  __shared__ float piece_max[kPieces];
  const int64_t row = blockIdx.x;
  RowView<T> v;
  v.x = logits + row * stride;
  v.A = A;
  v.r = row_settings(q, row);
  v.shift = q.shift;
  v.n_seg = 1;
  v.seg_len = kWaveRow;
  v.seg_hist = hist;
  v.seg_count = count;
  v.seg_first = nullptr;
  v.values = nullptr;
  const Pieces p{piece_mass, piece_max};
  const int pieces = (A + piece_length<T>() - 1) / piece_length<T>();
  max_pieces(v.x, A, 0, pieces, 0, 1, p.max);
  __syncthreads();
  v.m = row_max<T, 64>(p, A, w.red32);
  if (v.m > -INFINITY && weighed(v.r)) {
    sum_pieces(v.x, A, v.m, v.r.c, v.shift, 0, pieces, 0, 1, p);
    __syncthreads();
  } else if (v.m > -INFINITY && filtered(v.r)) {
    for (int i = threadIdx.x; i < kBins; i += 64) { hist[i] = 0; count[i] = 0; }
    __syncthreads();
    add_classes<T, 64>(v.x, 0, A, v.m, v.r, v.shift, hist, count, v.r.k > 0);
    __syncthreads();
  }
  draw_row(v, w, q, row, p);
}

// Longer rows: how a batch is cut.  What a row leaves in the workspace: its pieces' masses and maxima and, where it has
// filters, its segments' classes.
constexpr int64_t kFewElements = (int64_t)8 << 20;
struct SamplePlan {
  int64_t bytes;
  int n_seg, seg_len, n_piece;
  int64_t group;                         // rows that go through the three launches together
  uint64_t* piece_mass;                  // [B][n_piece]
  uint64_t* seg_hist;                    // [group][n_seg][kBins]
  uint32_t* seg_count;                   // [group][n_seg][kBins]
  float* piece_max;                      // [B][n_piece]
  uint32_t* seg_first;                   // [B][n_seg][kBins], and
  float* values;                         // [B][n_seg][seg_len]: the values by class, where the rows are few; else NULL
};

constexpr int kPartThreads = 256;

// a workgroup for `per` pieces: their maxima
template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_maxima_kernel(const T* __restrict__ logits, int64_t stride, int A,
                                                                     SamplePlan plan, int64_t row0, int per) {
  const int n = (A + piece_length<T>() - 1) / piece_length<T>();
  const uint32_t groups = (n + per - 1) / per;
  const int64_t row = row0 + blockIdx.x / groups;
  const int first = (int)(blockIdx.x % groups) * per, last = first + per < n ? first + per : n;
  max_pieces(logits + row * stride, A, first, last, threadIdx.x >> 6, kPartThreads / 64, plan.piece_max + row * plan.n_piece);
}

// a workgroup for `per` pieces: their masses, where no row has a filter
template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_masses_kernel(const T* __restrict__ logits, int64_t stride, int A,
                                                                     SampleArgs q, SamplePlan plan, int64_t row0, int per) {
  __shared__ uint32_t red[kPartThreads / 64];
  const int n = (A + piece_length<T>() - 1) / piece_length<T>();
  const uint32_t groups = (n + per - 1) / per;
  const int64_t row = row0 + blockIdx.x / groups;
  const Row r = row_settings(q, row);
  const int first = (int)(blockIdx.x % groups) * per, last = first + per < n ? first + per : n;
  const Pieces p{plan.piece_mass + row * plan.n_piece, plan.piece_max + row * plan.n_piece};
  const float m = row_max<T, kPartThreads>(p, A, red);
  if (m > -INFINITY)
    sum_pieces(logits + row * stride, A, m, r.c, q.shift, first, last, threadIdx.x >> 6, kPartThreads / 64, p);
}

// A workgroup per segment: its classes, where the row has filters.  MIXED: the settings are each row's own, and where they
// are no filters the segment's pieces are summed.
template <typename T, bool MIXED>
__global__ __launch_bounds__(kPartThreads) void sample_classes_kernel(const T* __restrict__ logits, int64_t stride, int A,
                                                                      SampleArgs q, SamplePlan plan, int64_t row0) {
  __shared__ uint64_t hist[kBins];
  __shared__ uint32_t count[kBins], red[kPartThreads / 64];
  const int64_t row = row0 + blockIdx.x / plan.n_seg;
  const int seg = blockIdx.x % plan.n_seg;
  const Row r = row_settings(q, row);
  if (MIXED ? r.greedy : !filtered(r)) return;
  const Pieces p{plan.piece_mass + row * plan.n_piece, plan.piece_max + row * plan.n_piece};
  const float m = row_max<T, kPartThreads>(p, A, red);
  if (!(m > -INFINITY)) return;
  if constexpr (MIXED) {
    if (weighed(r)) {
      const int n = (A + piece_length<T>() - 1) / piece_length<T>(), of = plan.seg_len / piece_length<T>();   // exact
      const int first = seg * of, last = first + of < n ? first + of : n;
      sum_pieces(logits + row * stride, A, m, r.c, q.shift, first, last, threadIdx.x >> 6, kPartThreads / 64, p);
      return;
    }
  }
  static_assert(kPartThreads == kBins, "a thread for each class");
  const int b = threadIdx.x;
  hist[b] = 0;
  count[b] = 0;
  __syncthreads();
  const bool counts = r.k > 0 || plan.values;
  const int begin = seg * plan.seg_len, end = begin + plan.seg_len < A ? begin + plan.seg_len : A;
  const T* x = logits + row * stride;
  add_classes<T, kPartThreads>(x, begin, end, m, r, q.shift, hist, count, counts);
  __syncthreads();
  const int64_t part = (row - row0) * plan.n_seg + seg;
  const uint32_t n = count[b];
  plan.seg_hist[part * kBins + b] = hist[b];
  if (counts) plan.seg_count[part * kBins + b] = n;
  if (!plan.values) return;
  // A few rows leave no work for most of the card while a workgroup each looks for the values of a class in them: here they are
  // put in the order of their classes, by all the segments' workgroups.
  const int lane = b & 63, wave = b >> 6;
  uint32_t run = wave_scan(n);
  if (lane == 63) red[wave] = run;
  __syncthreads();   // every count has been read
  for (int w = 0; w < wave; ++w) run += red[w];
  plan.seg_first[part * kBins + b] = run - n;
  count[b] = run - n;
  __syncthreads();
  float* values = plan.values + part * plan.seg_len;
  for_each_vec<T, kPartThreads>(x, begin, end, b, [&](const float (&g)[Vec16<T>::n], int) {
#pragma unroll
    for (int j = 0; j < Vec16<T>::n; ++j) {
      const double y = log2_weight(g[j], m, r.c);
      if (y >= kFloorLog2) values[atomicAdd(&count[weight_bin(y)], 1u)] = g[j];
    }
  });
}

// a workgroup per row: the rest
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_finish_kernel(const T* __restrict__ logits, int64_t stride, int A, SampleArgs q,
                                                           SamplePlan plan, int64_t row0) {
  __shared__ RowWork<NT> w;
  const int64_t row = row0 + blockIdx.x;
  RowView<T> v;
  v.x = logits + row * stride;
  v.A = A;
  v.r = row_settings(q, row);
  v.shift = q.shift;
  v.n_seg = plan.n_seg;
  v.seg_len = plan.seg_len;
  v.seg_hist = plan.seg_hist + blockIdx.x * (int64_t)plan.n_seg * kBins;
  v.seg_count = plan.seg_count + blockIdx.x * (int64_t)plan.n_seg * kBins;
  v.seg_first = plan.values ? plan.seg_first + blockIdx.x * (int64_t)plan.n_seg * kBins : nullptr;
  v.values = plan.values ? plan.values + blockIdx.x * (int64_t)plan.n_seg * plan.seg_len : nullptr;
  const Pieces p{plan.piece_mass + row * plan.n_piece, plan.piece_max + row * plan.n_piece};
  v.m = row_max<T, NT>(p, A, w.red32);
  draw_row(v, w, q, row, p);
}

static inline int sample_shift(int64_t A) {
  int bits = 0;
  while (((int64_t)1 << bits) < A) ++bits;
  return 62 - bits < 51 ? 62 - bits : 51;
}

static SamplePlan sample_plan(int64_t B, int64_t A, void* workspace) {
  constexpr int64_t kPiece = piece_length<float>();   // the shorter ones
  SamplePlan p;
  p.group = ((int64_t)256 << 20) / A;                 // 100 MB of classes, 201 where a row is little more than a segment
  if (p.group < 1) p.group = 1;
  if (p.group > B) p.group = B;
  // segments of about 8,192 actions (the last pass scans one of them), of fewer where the rows are few
  int64_t n = (A + 8191) / 8192;
  const int64_t few = 2048 / p.group, most = (A + 4095) / 4096;
  if (n < few) n = few < most ? few : most;
  if (n > kMaxParts) n = kMaxParts;
  p.seg_len = (int)(((A + n - 1) / n + 2047) / 2048 * 2048);
  p.n_seg = (int)((A + p.seg_len - 1) / p.seg_len);
  p.n_piece = (int)((A + kPiece - 1) / kPiece);
  const bool by_class = B * A <= kFewElements;
  char* at = (char*)workspace;
  p.piece_mass = (uint64_t*)at;
  at += B * p.n_piece * 8;
  p.seg_hist = (uint64_t*)at;
  at += p.group * p.n_seg * kBins * 8;
  p.seg_count = (uint32_t*)at;
  at += p.group * p.n_seg * kBins * 4;
  p.seg_first = (uint32_t*)at;
  if (by_class) at += p.group * p.n_seg * kBins * 4;
  p.values = by_class ? (float*)at : nullptr;
  if (by_class) at += p.group * p.n_seg * p.seg_len * 4;
  p.piece_max = (float*)at;
  at += B * p.n_piece * 4;
  p.bytes = at - (char*)workspace;
  return p;
}

static size_t sample_workspace(int64_t B, int64_t A) {
  if (B <= 0 || A <= kWaveRow) return 0;
  return (size_t)sample_plan(B, A, nullptr).bytes;
}

template <typename T>
static int sample_run(const T* logits, int64_t stride, int64_t B, int64_t A, const SampleArgs& q, void* workspace,
                      hipStream_t s) {
  if (A <= 64) {
    const int lanes = A <= 8 ? 8 : A <= 16 ? 16 : A <= 32 ? 32 : 64;
    const int grid = (int)((B * lanes + 255) / 256);
    if (lanes == 8) sample_small_kernel<T, 8><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
    else if (lanes == 16) sample_small_kernel<T, 16><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
    else if (lanes == 32) sample_small_kernel<T, 32><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
    else sample_small_kernel<T, 64><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
    return check_launch();
  }
  const bool ranked = q.top_k || q.top_p || q.top_k_s > 1 || (q.top_p_s < 1.f && q.top_p_s > 0.f);
  if (A <= 512 && (!ranked || (!q.temperature && q.temperature_s == 0.f))) {
    const int grid = (int)((B + 3) / 4);
    if (A <= 128) sample_lanes_kernel<T, 2><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
    else if (A <= 256) sample_lanes_kernel<T, 4><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
    else sample_lanes_kernel<T, 8><<<grid, 256, 0, s>>>(logits, stride, B, (int)A, q);
    return check_launch();
  }
  if (A <= kWaveRow) {
    sample_wave_kernel<T><<<(int)B, 64, 0, s>>>(logits, stride, (int)A, q);
    return check_launch();
  }
  const SamplePlan p = sample_plan(B, A, workspace);
  const bool per_row = q.temperature || q.top_k || q.top_p || q.min_p;
  const bool greedy = !per_row && q.temperature_s == 0.f;
  const bool filters = per_row || (!greedy && (q.top_k_s > 0 || q.top_p_s < 1.f || q.min_p_s > kFloor));   // as filtered()
  const int pieces = (int)((A + piece_length<T>() - 1) / piece_length<T>());
  // a launch has fewer than 2^32 threads: a workgroup for every four of a row's pieces at most, 1,024 threads to finish it
  const int64_t row_threads = std::max<int64_t>(kPartThreads * ((pieces + 3) / 4), 1024);
  const int64_t group = std::min<int64_t>(filters ? p.group : B, 0xffffffffLL / row_threads);
  for (int64_t row0 = 0; row0 < B; row0 += group) {
    const int64_t rows = row0 + group < B ? group : B - row0;
    // a piece for each wave, or two where that makes more than enough workgroups: with one, two and four for the masses 1,024
    // rows of 131,072 take 149, 144 and 142 us, one row 11, 13 and 16
    const int per = rows * pieces >= 65536 ? 8 : 4;
    const int groups = (int)(rows * ((pieces + per - 1) / per));
    sample_maxima_kernel<T><<<groups, kPartThreads, 0, s>>>(logits, stride, (int)A, p, row0, per);
    if (int rc = check_launch()) return rc;
    if (per_row)
      sample_classes_kernel<T, true><<<(int)(rows * p.n_seg), kPartThreads, 0, s>>>(logits, stride, (int)A, q, p, row0);
    else if (filters)
      sample_classes_kernel<T, false><<<(int)(rows * p.n_seg), kPartThreads, 0, s>>>(logits, stride, (int)A, q, p, row0);
    else if (!greedy)
      sample_masses_kernel<T><<<groups, kPartThreads, 0, s>>>(logits, stride, (int)A, q, p, row0, per);
    if (int rc = check_launch()) return rc;
    // a thread for each piece of a row; else smaller workgroups, more rows side by side, where the rows are many
    if (pieces > 512)
      sample_finish_kernel<T, 1024><<<(int)rows, 1024, 0, s>>>(logits, stride, (int)A, q, p, row0);
    else if (rows < 512 || pieces > 256)
      sample_finish_kernel<T, 512><<<(int)rows, 512, 0, s>>>(logits, stride, (int)A, q, p, row0);
    else
      sample_finish_kernel<T, 256><<<(int)rows, 256, 0, s>>>(logits, stride, (int)A, q, p, row0);
    if (int rc = check_launch()) return rc;
  }
  return PARLHIP_OK;
}

}  // namespace parlhip

using namespace parlhip;

PARLHIP_EXPORT size_t parlhip_logits_sample_workspace_bytes(int64_t B, int64_t A) {
  return A < 1 || A > kSampleMaxActions ? 0 : sample_workspace(B, A);
}

PARLHIP_EXPORT int parlhip_logits_sample(const void* logits, int dtype, int64_t row_stride, const double* uniforms,
                                         const float* temperature, const int32_t* top_k, const float* top_p,
                                         const float* min_p, float temperature_all, int32_t top_k_all, float top_p_all,
                                         float min_p_all, int64_t* actions, float* log_probs, int64_t B, int64_t A,
                                         void* workspace, size_t workspace_bytes, parlhip_stream_t stream) {
  if (B < 0 || A < 1 || row_stride < A) return PARLHIP_EINVAL;
  if (dtype != PARLHIP_F32 && dtype != PARLHIP_BF16 && dtype != PARLHIP_F16) return PARLHIP_ENOSUP;
  // up to 4,096 actions one launch of fewer than 2^32 threads: 64 for a row, four rows to a workgroup
  if (A > kSampleMaxActions || B > (A <= kWaveRow ? ((int64_t)1 << 26) - 4 : ((int64_t)1 << 40) / A)) return PARLHIP_ENOSUP;
  if (!temperature && !(temperature_all >= 0.f && temperature_all < INFINITY)) return PARLHIP_EINVAL;
  if (!top_p && !(top_p_all >= 0.f)) return PARLHIP_EINVAL;
  if (!min_p && !(min_p_all >= 0.f && min_p_all <= 1.f)) return PARLHIP_EINVAL;
  if (B == 0) return PARLHIP_OK;
  if (!logits || !uniforms || !actions || !log_probs) return PARLHIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == PARLHIP_F32 ? 3 : 1)) return PARLHIP_EINVAL;
  const size_t need = sample_workspace(B, A);
  if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 7))) return PARLHIP_EINVAL;
  if (workspace_bytes < need) return PARLHIP_ENOMEM;
  SampleArgs q{uniforms, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all,
               actions, log_probs, device_error_flag(), sample_shift(A)};
  if (!q.err) return PARLHIP_ELAUNCH;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PARLHIP_F32) return sample_run((const float*)logits, row_stride, B, A, q, workspace, s);
  if (dtype == PARLHIP_BF16) return sample_run((const bf16_t*)logits, row_stride, B, A, q, workspace, s);
  return sample_run((const f16_t*)logits, row_stride, B, A, q, workspace, s);
}
