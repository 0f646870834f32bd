// Row operators over vocabulary logits [R, V]: the k largest entries of a row with its
// log-sum-exp, and sampling from a row's filtered softmax with a given uniform.
//
// Two launches. The scan reads every logit once, at HBM speed, over as many CTAs as there are slices:
// it leaves the largest key of each group of 32 neighbouring entries (3 % of the row's bytes) and per
// slice its maximum and, where it is needed, its softmax weight. Then one CTA per row
// finishes from those:
//   - The k largest entries: the k-th largest group maximum is at most the k-th largest entry, and
//     little below it unless the row is arranged against it, so the few groups at or above it are read
//     again (from L2) and the entries at or above it, k and a few more, are ordered in shared memory.
//   - A nucleus without top-k is looked for among the 1024 largest entries first; a wider one's border
//     is bracketed by a histogram and found exactly among the entries in the bracket.
//   - Without a filter the slices' weights say which slice holds the uniform's share.
// Where the gathered entries are too many for shared memory (rows of equal values, nuclei of many
// thousands), the CTA goes over the whole row again: a radix selection that is right for every row, and
// a walk in index order.
//
// Candidates are the entries that are neither -inf nor NaN. Entries are ordered by (descending
// value, ascending index); -0 counts as +0.
#pragma once

#include <cuda_bf16.h>

#include "sm100.cuh"

namespace orthrus {

constexpr int kRowThreads = 512;          // of the CTA that finishes a row
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kScanThreads = 256;
constexpr int kRowGroup = 32;             // entries behind one group maximum
constexpr int kRowBins = 2048;
constexpr int kRowMaxK = 1024;            // largest k of topk_rows
constexpr int kRowList = 2048;            // most entries gathered into shared memory
constexpr int kRowMaxV = 1 << 20;         // the group maxima of a longer row do not fit shared memory

// ------------------------------------------------------------------------------------------------
// Keys: unsigned integers that order as the values do; 0 marks an entry that is no candidate.
// ------------------------------------------------------------------------------------------------

template <typename T>
struct RowKey;

template <>
struct RowKey<float> {
  using type = uint32_t;
  static constexpr int BITS = 32;
  static constexpr int VEC = 4;  // elements per 16-byte load
  __device__ static __forceinline__ uint32_t of(float x) { return of_bits(__float_as_uint(x)); }
  __device__ static __forceinline__ uint32_t of_bits(uint32_t b) {
    if ((b << 1) == 0u) b = 0u;                                       // -0 as +0
    if ((b << 1) > 0xFF000000u || b == 0xFF800000u) return 0u;        // NaN, -inf
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  }
  __device__ static __forceinline__ float value(uint32_t k) {
    return k == 0u ? -INFINITY : __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
  }
};

template <>
struct RowKey<__nv_bfloat16> {
  using type = uint16_t;
  static constexpr int BITS = 16;
  static constexpr int VEC = 8;
  __device__ static __forceinline__ uint32_t of(float x) { return of_bits(__float_as_uint(x) >> 16); }  // x is a bf16
  __device__ static __forceinline__ uint32_t of_bits(uint32_t b) {
    if ((b & 0x7FFFu) == 0u) b = 0u;
    if ((b & 0x7FFFu) > 0x7F80u || b == 0xFF80u) return 0u;
    return (b & 0x8000u) ? (~b & 0xFFFFu) : (b | 0x8000u);
  }
  __device__ static __forceinline__ float value(uint32_t k) {
    return k == 0u ? -INFINITY : __uint_as_float(((k & 0x8000u) ? (k & 0x7FFFu) : (~k & 0xFFFFu)) << 16);
  }
};

// ------------------------------------------------------------------------------------------------
// A row in 16-byte blocks
// ------------------------------------------------------------------------------------------------

// Block b of a row of any alignment covers the entries b * VEC - off .. + VEC - 1, where off is the
// row's distance in entries from the 16-byte boundary before it; entries outside the row count as no
// candidates and are never read.
template <typename T>
struct RowView {
  using K = RowKey<T>;
  static constexpr int VEC = K::VEC;
  const T* p;
  int V, off, blocks;

  __device__ __forceinline__ RowView(const T* row, int n)
      : p(row), V(n), off(static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T))),
        blocks((n + off + VEC - 1) / VEC) {}
  __device__ __forceinline__ int first(int b) const { return b * VEC - off; }
  __device__ __forceinline__ bool whole(int b) const { return first(b) >= 0 && first(b) + VEC <= V; }
  __device__ __forceinline__ uint4 load(int b) const { return __ldg(reinterpret_cast<const uint4*>(p + first(b))); }
  // the keys of a block loaded as 16 bytes
  __device__ __forceinline__ static void keys_of(const uint4& q, uint32_t (&k)[VEC]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      k[e] = sizeof(T) == 4 ? K::of_bits(w[e]) : K::of_bits((e & 1) ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu);
  }
  // its values, with -inf for what is no candidate
  __device__ __forceinline__ static void values_of(const uint4& q, float (&x)[VEC]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const uint32_t b = sizeof(T) == 4 ? w[e] : (e & 1) ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16;
      x[e] = fmaxf(__uint_as_float(b), -INFINITY);  // NaN gives way
    }
  }
  __device__ __forceinline__ void values(int b, float (&x)[VEC]) const {
    if (b < blocks && whole(b)) {
      values_of(load(b), x);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = b < blocks ? K::value(key(first(b) + e)) : -INFINITY;
    }
  }
  __device__ __forceinline__ uint32_t key(int i) const {
    if (i < 0 || i >= V) return 0u;
    if constexpr (sizeof(T) == 4)
      return K::of_bits(__ldg(reinterpret_cast<const uint32_t*>(p) + i));
    else
      return K::of_bits(__ldg(reinterpret_cast<const uint16_t*>(p) + i));
  }
  __device__ __forceinline__ void edge(int b, uint32_t (&k)[VEC]) const {
#pragma unroll
    for (int e = 0; e < VEC; ++e) k[e] = b < blocks ? key(first(b) + e) : 0u;
  }
  __device__ __forceinline__ void keys(int b, uint32_t (&k)[VEC]) const {
    if (b < blocks && whole(b))
      keys_of(load(b), k);
    else
      edge(b, k);
  }
};

// ------------------------------------------------------------------------------------------------
// Block helpers
// ------------------------------------------------------------------------------------------------

struct RowScratch {
  uint64_t hist[kRowBins];   // radix selection and nucleus: counts (32-bit words) or weights; else a list
  uint64_t list[kRowList];   // gathered entries, (key << 32 | ~index)
  double exp_tab[64];        // 2^(-j/64)
  uint64_t warp[kRowWarps];
  uint32_t top[kRowWarps];
  uint64_t found[2];         // result of a block-wide search
  uint32_t groups[kRowList]; // numbers of the groups to read again
  uint32_t ngroups, listed;
};

__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Block-wide sum; every thread gets it. Leaves warp_u64 free for reuse.
__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, RowScratch& sh) {
  v = warp_sum_u64(v);
  if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) t += sh.warp[w];
  __syncthreads();
  return t;
}

// Exclusive prefix sum over the block's threads; `total` is the block's sum.
__device__ __forceinline__ uint64_t block_exclusive_u64(uint64_t v, RowScratch& sh, uint64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) sh.warp[warp] = inc;
  __syncthreads();
  uint64_t before = 0, t = 0;
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) {
    if (w == warp) before = t;
    t += sh.warp[w];
  }
  __syncthreads();
  total = t;
  return before + inc - v;
}

// ------------------------------------------------------------------------------------------------
// Softmax weights as 64-bit integers
// ------------------------------------------------------------------------------------------------

// w(x) = round(2^S exp((x - top) / T)). Integer weights make every sum exact, so running sums do not
// depend on how a row is split over threads, and comparisons with a uniform's share of the total
// fall the same way on every path. S = min(44, 62 - ceil(log2 V)) keeps a row's sum below
// 2^62; a weight is off by at most half a unit plus 2^-44 of itself.
//
// The exponential is the table method (P. T. P. Tang, "Table-driven implementation of the
// exponential function in IEEE floating-point arithmetic", ACM TOMS 15, 1989): y = 64 (max - x) log2(e) / T
// = n + f with |f| <= 1/2, exp = 2^-(n >> 6) * tab[n & 63] * e^(-f ln2 / 64), the last factor by
// its Taylor polynomial of degree 4 (error below (0.0055)^5 / 120 = 4e-14).
struct RowWeight {
  float top;         // the maximum the weights refer to
  int S;
  double scale, at;  // 64 log2(e) / T; top * scale
  const double* tab;

  __device__ __forceinline__ uint64_t operator()(float x) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    constexpr double kInt = 4503599627370496.0;    // 2^52
    constexpr double c = -0.6931471805599453 / 64.0;
    const double y = x == top ? 0.0 : fma(-static_cast<double>(x), scale, at);
    if (!(y < 64.0 * (S + 2))) return 0;  // rounds to 0; also an infinite maximum's other entries
    const double r = y + kRound;
    const int n = __double2loint(r);
    const double f = y - (r - kRound);
    const double p = fma(fma(fma(fma(f, c * c * c * c / 24.0, c * c * c / 6.0), f, c * c / 2.0), f, c), f, 1.0) * tab[n & 63];
    // times 2^(S - n / 64), by the exponent
    const double w = __hiloint2double(__double2hiint(p) + ((S - (n >> 6)) << 20), __double2loint(p)) + kInt;
    return static_cast<uint64_t>(__double_as_longlong(w)) & 0xFFFFFFFFFFFFFull;
  }
};

__host__ __device__ inline int row_weight_bits(int V) {
  int b = 0;
  while ((1ll << b) < V) ++b;
  return 62 - b < 44 ? 62 - b : 44;
}

__device__ __forceinline__ void row_exp_table(double* tab) {
  if (threadIdx.x < 64) tab[threadIdx.x] = exp2(-static_cast<double>(threadIdx.x) / 64.0);
}

__device__ __forceinline__ RowWeight row_weight(float top, float temperature, int S, const double* tab) {
  const double scale = 92.33248261893567 / static_cast<double>(temperature);  // 64 log2(e) / T
  return {top, S, scale, static_cast<double>(top) * scale, tab};
}

// floor(f * z) for f in [0, 1) and z < 2^62, exactly (f is an integer of 24 bits times a power of
// two). Negative or NaN f count as 0; f >= 1 gives z - 1 (z > 0).
__device__ __forceinline__ uint64_t floor_share(float f, uint64_t z) {
  if (!(f > 0.f)) return 0;
  if (f >= 1.f) return z - 1;
  const uint32_t b = __float_as_uint(f);
  const int e = static_cast<int>(b >> 23);
  const uint64_t m = e == 0 ? b : ((b & 0x7FFFFFu) | 0x800000u);
  const int shift = 150 - (e == 0 ? 1 : e);  // f = m * 2^-shift, shift >= 24
  const uint64_t lo = m * z, hi = __umul64hi(m, z);
  if (shift >= 128) return 0;
  if (shift >= 64) return hi >> (shift - 64);
  return (hi << (64 - shift)) | (lo >> shift);
}

// ------------------------------------------------------------------------------------------------
// The scan
// ------------------------------------------------------------------------------------------------

struct RowSlice {
  uint32_t top;    // largest key
  float sum;       // sum of exp((x - slice's largest) / T) (top-k)
  uint64_t mass;   // the same, 2^S fold (sampling)
};

// What the scan leaves of R rows: group maxima [R, groups] (groups a multiple of four, so that a row's
// are read as vectors) and slices [R, slices].
struct RowScan {
  uint32_t* group;
  RowSlice* slice;
  int groups, slices;
};

struct SampleKnobs {
  const float* temperature;  // [R], or null: one value for every row
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature1, top_p1, min_p1;
  int top_k1;
};

// How a row is sampled, from its knobs.
struct SampleRow {
  float temperature, top_p, min_p;
  int top_k;
  bool greedy;
  __device__ __forceinline__ SampleRow(const SampleKnobs& k, int64_t row)
      : temperature(k.temperature ? k.temperature[row] : k.temperature1),
        top_p(k.top_p ? k.top_p[row] : k.top_p1),
        min_p(k.min_p ? k.min_p[row] : k.min_p1),
        top_k(k.top_k ? k.top_k[row] : k.top_k1),
        greedy(temperature < 1e-5f) {}
  // whether the slices' weights are asked for: no filter, or a nucleus of the whole row
  __device__ __forceinline__ bool wants_mass() const { return !greedy && top_k < 1 && (top_p < 1.f || !(min_p > 0.f)); }
};

// One slice of BLOCKS * 256 16-byte blocks per CTA (slices of a row first), every load issued before the
// first is used. The slice's weight is the fp32 sum of exponentials, or, to SAMPLE, integer weights
// for the rows that want them.
template <typename T, int BLOCKS, bool SAMPLE>
__global__ void __launch_bounds__(kScanThreads)
    row_scan_kernel(const T* __restrict__ x, int64_t ldx, int V, float temperature, int S, SampleKnobs knobs,
                    RowScan out) {
  using View = RowView<T>;
  using K = RowKey<T>;
  constexpr int VEC = View::VEC;
  constexpr int LANES = kRowGroup / VEC;  // neighbouring lanes of a group
  __shared__ double tab[64];
  __shared__ float wtop[kScanThreads / 32], wsum[kScanThreads / 32];
  __shared__ uint64_t wmass[kScanThreads / 32];
  griddep_launch_dependents();
  const int64_t row = blockIdx.x / static_cast<unsigned>(out.slices);
  const int slice = static_cast<int>(blockIdx.x % static_cast<unsigned>(out.slices));
  const View v(x + row * ldx, V);
  const int b0 = slice * BLOCKS * kScanThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bool mass_wanted = true;
  if constexpr (SAMPLE) {
    const SampleRow knob(knobs, row);
    temperature = knob.temperature;
    mass_wanted = knob.wants_mass();
    if (mass_wanted) row_exp_table(tab);
  }
  float val[BLOCKS][VEC];
  if (v.whole(b0) && v.whole(b0 + BLOCKS * kScanThreads - 1)) {
    uint4 q[BLOCKS];
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) q[j] = v.load(b0 + j * kScanThreads + threadIdx.x);
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) View::values_of(q[j], val[j]);
  } else {  // the row's ends
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) v.values(b0 + j * kScanThreads + threadIdx.x, val[j]);
  }
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) {
    float m = val[j][0];
#pragma unroll
    for (int e = 1; e < VEC; ++e) m = fmaxf(m, val[j][e]);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    top = fmaxf(top, m);
    const int g = (b0 + j * kScanThreads + static_cast<int>(threadIdx.x)) / LANES;
    if (lane % LANES == 0 && g < out.groups) out.group[row * out.groups + g] = K::of(m);
  }
#pragma unroll
  for (int o = 16; o >= LANES; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) wtop[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kScanThreads / 32; ++w) top = fmaxf(top, wtop[w]);
  uint64_t mass = 0;
  float sum = 0.f;
  if constexpr (SAMPLE) {
    if (mass_wanted && top > -INFINITY) {
      const RowWeight weight = row_weight(top, temperature, S, tab);
#pragma unroll
      for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) mass += weight(val[j][e]);
      mass = warp_sum_u64(mass);
    }
    if (lane == 0) wmass[warp] = mass;
  } else {
    const float c = kLog2e / temperature;
    float part[4] = {0.f, 0.f, 0.f, 0.f};
    if (top > -INFINITY && top < INFINITY) {
#pragma unroll
      for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) part[e & 3] += ex2_approx((val[j][e] - top) * c);
    }
    sum = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) wsum[warp] = sum;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    RowSlice r{K::of(top), 0.f, 0ull};
    for (int w = 0; w < kScanThreads / 32; ++w) {
      if constexpr (SAMPLE) r.mass += wmass[w];
      else r.sum += wsum[w];
    }
    out.slice[row * out.slices + slice] = r;
  }
}

// ------------------------------------------------------------------------------------------------
// The few largest entries
// ------------------------------------------------------------------------------------------------

// The row's group maxima into shared memory and its largest key (0: no candidates), for every thread.
__device__ __forceinline__ uint32_t row_open(const RowScan& scan, int64_t row, uint32_t* maxima, RowScratch& sh) {
  const uint4* g = reinterpret_cast<const uint4*>(scan.group + row * scan.groups);
  uint4* m = reinterpret_cast<uint4*>(maxima);
  uint32_t top = 0;
  for (int i = threadIdx.x; i < scan.slices; i += kRowThreads) top = max(top, scan.slice[row * scan.slices + i].top);
#pragma unroll 4
  for (int i = threadIdx.x; i < scan.groups / 4; i += kRowThreads) m[i] = g[i];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) sh.top[threadIdx.x >> 5] = top;
  if (threadIdx.x == 0) sh.ngroups = sh.listed = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) top = max(top, sh.top[w]);
  return top;
}

// A key with at least k entries of the row at or above it, and not many more: between the k-th largest
// group maximum and a little below it; 1 if fewer than k groups hold a candidate. Histograms of the
// maxima over the range of keys that can hold the bound, 1024 bins at a time.
__device__ __forceinline__ uint32_t row_bound(const uint32_t* maxima, int groups, int k, uint32_t top_key,
                                              RowScratch& sh) {
  constexpr int BINS = 2 * kRowThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t* counts = reinterpret_cast<uint32_t*>(sh.hist);
  const uint4* m4 = reinterpret_cast<const uint4*>(maxima);
  // the smallest candidate maximum
  uint32_t least = top_key;
  for (int i = threadIdx.x; i < groups / 4; i += kRowThreads) {
    const uint4 q = m4[i];
    least = min(min(least, q.x ? q.x : top_key), min(min(q.y ? q.y : top_key, q.z ? q.z : top_key), q.w ? q.w : top_key));
  }
  least = __reduce_min_sync(0xffffffffu, least);
  if (lane == 0) sh.top[warp] = least;
  counts[threadIdx.x] = counts[threadIdx.x + kRowThreads] = 0;
  if (threadIdx.x == 0) sh.found[0] = ~0ull;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) least = min(least, sh.top[w]);
  uint32_t lo = least, hi = top_key;  // the bound is in [lo, hi]
  uint32_t above = 0;                 // maxima above hi
  const uint32_t want = k, enough = k + k / 4 + 16;
  while (true) {
    int shift = 0;
    while (((hi - lo) >> shift) >= BINS) ++shift;
    for (int i = threadIdx.x; i < groups / 4; i += kRowThreads) {
      const uint4 q = m4[i];
      const uint32_t m[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (m[e] >= lo && m[e] <= hi) atomicAdd(&counts[(hi - m[e]) >> shift], 1u);
    }
    __syncthreads();
    // bin b holds the keys hi - (b << shift) downwards; thread t has the bins 2t and 2t + 1
    const uint32_t c0 = counts[2 * threadIdx.x], c1 = counts[2 * threadIdx.x + 1];
    uint32_t inc = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) sh.top[warp] = inc;
    __syncthreads();
    uint32_t run = above + inc - c0 - c1;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) run += w < warp ? sh.top[w] : 0u;
    if (run < want && want <= run + c0) {
      sh.found[0] = 2 * threadIdx.x;
      sh.found[1] = (static_cast<uint64_t>(run) << 32) | (run + c0);
    } else if (run + c0 < want && want <= run + c0 + c1) {
      sh.found[0] = 2 * threadIdx.x + 1;
      sh.found[1] = (static_cast<uint64_t>(run + c0) << 32) | (run + c0 + c1);
    }
    counts[2 * threadIdx.x] = counts[2 * threadIdx.x + 1] = 0;
    __syncthreads();
    if (sh.found[0] == ~0ull) {  // fewer than k groups hold a candidate
      lo = 1u;
      break;
    }
    const uint32_t b = static_cast<uint32_t>(sh.found[0]), have = static_cast<uint32_t>(sh.found[1]);
    const uint32_t from = hi - (b << shift), depth = (1u << shift) - 1u;
    above = static_cast<uint32_t>(sh.found[1] >> 32);
    lo = from - lo > depth ? from - depth : lo;
    hi = from;
    if (have <= enough || shift == 0) break;
  }
  __syncthreads();  // found and the counts are free again
  return lo;
}

// Appends the entries of the lanes with `take` to the list, one atomic a warp. Every lane calls it.
template <typename E>
__device__ __forceinline__ void row_append(bool take, E entry, E* list, uint32_t* count) {
  const uint32_t who = __ballot_sync(0xffffffffu, take);
  if (who == 0) return;
  const int lane = threadIdx.x & 31, first = __ffs(who) - 1;
  uint32_t at = 0;
  if (lane == first) at = atomicAdd(count, static_cast<uint32_t>(__popc(who)));
  at = __shfl_sync(0xffffffffu, at, first) + __popc(who & ((1u << lane) - 1u));
  if (take && at < kRowList) list[at] = entry;
}

// Reads the groups at or above `low` again and lists their entries with low <= key; returns their
// number, or more than kRowList if they do not fit. Ends with a barrier; listed is left at 0.
template <typename T>
__device__ int row_gather(const RowView<T>& v, const uint32_t* maxima, int groups, uint32_t low, RowScratch& sh) {
  constexpr int VEC = RowView<T>::VEC, LANES = kRowGroup / VEC;
  const int lane = threadIdx.x & 31;
  for (int i0 = 0; i0 < groups; i0 += kRowThreads) {
    const int i = i0 + static_cast<int>(threadIdx.x);
    row_append(i < groups && maxima[i] >= low, static_cast<uint32_t>(i), sh.groups, &sh.ngroups);
  }
  __syncthreads();
  const int ng = static_cast<int>(sh.ngroups);  // every group holds at least one entry
  // LANES neighbouring lanes a group
  if (ng <= kRowList)
    for (int i0 = 0; i0 < ng; i0 += kRowThreads / LANES) {
      const int i = i0 + static_cast<int>(threadIdx.x) / LANES;
      uint32_t k[VEC];
      int b = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) k[e] = 0u;
      if (i < ng) {
        b = static_cast<int>(sh.groups[i]) * LANES + lane % LANES;
        v.keys(b, k);
      }
      __syncwarp();
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        row_append(k[e] >= low, (static_cast<uint64_t>(k[e]) << 32) | ~static_cast<uint32_t>(v.first(b) + e), sh.list,
                   &sh.listed);
    }
  __syncthreads();
  const int n = ng <= kRowList ? static_cast<int>(sh.listed) : kRowList + 1;
  __syncthreads();
  if (threadIdx.x == 0) sh.ngroups = sh.listed = 0;
  __syncthreads();
  return n;
}

// Descending bitonic sort of a[0, n2), n2 a power of two.
__device__ __forceinline__ void row_sort_desc(uint64_t* a, int n2) {
  for (int size = 2; size <= n2; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n2 / 2; i += kRowThreads) {
        const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const uint64_t x = a[lo], y = a[hi];
        if ((x < y) == ((lo & size) == 0)) {
          a[lo] = y;
          a[hi] = x;
        }
      }
    }
  __syncthreads();
}

// Orders `in` (n <= kRowList different entries) descending into `out` (not the same array): by rank
// counting for a few entries, several threads an entry; else by a sorting network on `in`.
__device__ __forceinline__ void row_order(uint64_t* in, uint64_t* out, int n) {
  if (n <= kRowThreads) {
    int parts = 32;
    while (parts > 1 && parts * n > kRowThreads) parts >>= 1;
    const int e = threadIdx.x / parts, part = threadIdx.x % parts;
    const uint64_t x = e < n ? in[e] : 0;
    int rank = 0;
    if (e < n)
      for (int j = part; j < n; j += parts) rank += in[j] > x;
    for (int o = parts >> 1; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (e < n && part == 0) out[rank] = x;
    __syncthreads();
    return;
  }
  int n2 = 1;
  while (n2 < n) n2 <<= 1;
  for (int i = n + threadIdx.x; i < n2; i += kRowThreads) in[i] = 0;
  row_sort_desc(in, n2);
  for (int i = threadIdx.x; i < n; i += kRowThreads) out[i] = in[i];
  __syncthreads();
}

// ------------------------------------------------------------------------------------------------
// Going over the whole row
// ------------------------------------------------------------------------------------------------

// f(index, key) for every candidate of the row, each by one thread.
template <typename T, typename F>
__device__ __forceinline__ void row_visit(const RowView<T>& v, F f) {
  constexpr int VEC = RowView<T>::VEC, UNROLL = 32 / VEC;
  for (int b0 = threadIdx.x; b0 < v.blocks; b0 += UNROLL * kRowThreads) {
    uint4 q[UNROLL];
    const bool inside = v.whole(b0) && v.whole(b0 + (UNROLL - 1) * kRowThreads);
#pragma unroll
    for (int j = 0; j < UNROLL; ++j)
      if (inside) q[j] = v.load(b0 + j * kRowThreads);
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      uint32_t k[VEC];
      if (inside)
        RowView<T>::keys_of(q[j], k);
      else
        v.keys(b0 + j * kRowThreads, k);
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (k[e]) f(v.first(b0 + j * kRowThreads) + e, k[e]);
    }
  }
}

// Finds, among the candidates with key >= floor_key in descending order of key, the key whose
// entries hold position `target` of the running measure: the measure (MASS: the sum of weights;
// otherwise the count) of all larger keys is `before` <= target < before + its own. The caller
// makes sure that target is below the total. Every thread gets the result.
template <typename T, bool MASS>
__device__ uint32_t row_radix_select(const RowView<T>& v, uint32_t floor_key, uint64_t target, const RowWeight& weight,
                                     RowScratch& sh, uint64_t& before) {
  constexpr int BITS = RowKey<T>::BITS;
  uint32_t prefix = 0;
  int shift = BITS;
  before = 0;
  uint32_t* counts = reinterpret_cast<uint32_t*>(sh.hist);
  while (shift > 0) {
    const int width = shift < 11 ? shift : 11;
    const int next = shift - width;
    const uint32_t mask = (1u << width) - 1u;
    for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) {
      if constexpr (MASS) sh.hist[i] = 0;
      else counts[i] = 0;
    }
    __syncthreads();
    row_visit<T>(v, [&](int, uint32_t k) {
      if (k < floor_key || (shift < BITS && (k >> shift) != prefix)) return;
      const uint32_t d = (k >> next) & mask;
      if constexpr (MASS) {
        const uint64_t w = weight(RowKey<T>::value(k));
        if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[d]), static_cast<unsigned long long>(w));
      } else {
        atomicAdd(&counts[d], 1u);
      }
    });
    __syncthreads();
    // thread t takes the bins 2047 - 4t .. 2044 - 4t
    constexpr int PER = kRowBins / kRowThreads;
    uint64_t h[PER], own = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int b = kRowBins - 1 - (static_cast<int>(threadIdx.x) * PER + j);
      h[j] = MASS ? sh.hist[b] : counts[b];
      own += h[j];
    }
    uint64_t total;
    uint64_t run = before + block_exclusive_u64(own, sh, total);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (run <= target && target < run + h[j]) {
        sh.found[0] = kRowBins - 1 - (threadIdx.x * PER + j);
        sh.found[1] = run;
      }
      run += h[j];
    }
    __syncthreads();
    prefix = (prefix << width) | static_cast<uint32_t>(sh.found[0]);
    before = sh.found[1];
    shift = next;
    __syncthreads();  // found is read before the next level sets it
  }
  return prefix;
}

// Steps of 32 blocks (512 bytes) that a warp goes through in index order: warp w has the steps from
// w * row_warp_steps on.
__device__ __forceinline__ int row_warp_steps(int blocks) { return ((blocks + 31) / 32 + kRowWarps - 1) / kRowWarps; }

// f(block, keys of this lane's block) for each step, by every lane of the warp, until f returns false
// (the same in every lane). Blocks whose group lies below `low` are not read (maxima null: all are);
// their keys are 0, as past the end. Loads run four steps ahead.
template <typename T, typename F>
__device__ __forceinline__ void row_warp_walk(const RowView<T>& v, const uint32_t* maxima, uint32_t low, F f) {
  constexpr int VEC = RowView<T>::VEC, LANES = kRowGroup / VEC, AHEAD = 4;
  const int lane = threadIdx.x & 31, per = row_warp_steps(v.blocks);
  const int s0 = static_cast<int>(threadIdx.x >> 5) * per, s1 = min((v.blocks + 31) / 32, s0 + per);
  for (int s = s0; s < s1; s += AHEAD) {
    uint4 q[AHEAD];
    bool whole[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int b = (s + j) * 32 + lane;
      whole[j] = s + j < s1 && v.whole(b) && (maxima == nullptr || maxima[b / LANES] >= low);
      if (whole[j]) q[j] = v.load(b);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (s + j >= s1) return;
      const int b = (s + j) * 32 + lane;
      uint32_t k[VEC];
      if (whole[j]) {
        RowView<T>::keys_of(q[j], k);
      } else if (b < v.blocks && !v.whole(b)) {
        v.edge(b, k);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) k[e] = 0u;
      }
      __syncwarp();
      if (!f(b, k)) return;
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Top-k
// ------------------------------------------------------------------------------------------------

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2)
    topk_rows_kernel(const T* __restrict__ x, int64_t ldx, int V, int k, float temperature, RowScan scan,
                     float* __restrict__ values, int64_t* __restrict__ ids, float* __restrict__ lse) {
  using K = RowKey<T>;
  extern __shared__ __align__(16) uint32_t row_maxima[];
  __shared__ RowScratch sh;
  griddep_wait();  // launched as a programmatic dependent of the scan
  const int64_t row = blockIdx.x;
  const RowView<T> v(x + row * ldx, V);
  const uint32_t top_key = row_open(scan, row, row_maxima, sh);
  if (threadIdx.x >= kRowThreads - 32) {  // the last warp joins the slices' sums at the row's maximum
    const double top = K::value(top_key);
    double s = 0.0;
    for (int i = threadIdx.x & 31; i < scan.slices; i += 32) {
      const RowSlice a = scan.slice[row * scan.slices + i];
      if (a.top) s += a.sum * exp((static_cast<double>(K::value(a.top)) - top) / temperature);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0)
      lse[row] = top_key == 0 ? -INFINITY : !(top < INFINITY) ? INFINITY : static_cast<float>(top / temperature + log(s));
  }
  int kk = 0;  // entries given
  if (top_key > 0) {
    const uint32_t bound = row_bound(row_maxima, scan.groups, k, top_key, sh);
    int n = row_gather<T>(v, row_maxima, scan.groups, bound, sh);
    kk = min(n, k);
    if (n > kRowList) {
      // the kk-th largest key, then the larger ones and of its equals the first in index order
      uint64_t n_gt;
      const RowWeight none{};
      const uint32_t cut = row_radix_select<T, false>(v, 1u, kk - 1, none, sh, n_gt);
      uint32_t eq = 0;
      row_warp_walk<T>(v, nullptr, 0u, [&](int, const uint32_t(&key)[RowView<T>::VEC]) {
#pragma unroll
        for (int e = 0; e < RowView<T>::VEC; ++e) eq += key[e] == cut;
        return true;
      });
      // equals of the warps before this one
      uint64_t total;
      uint64_t rank = block_exclusive_u64(eq, sh, total);
      rank = __shfl_sync(0xffffffffu, rank, 0);
      const uint64_t room = kk - n_gt;
      const int lane = threadIdx.x & 31;
      row_warp_walk<T>(v, nullptr, 0u, [&](int b, const uint32_t(&key)[RowView<T>::VEC]) {
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < RowView<T>::VEC; ++e) mine += key[e] == cut;
        uint32_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += u;
        }
        uint64_t r = rank + inc - mine;
        rank += __shfl_sync(0xffffffffu, inc, 31);
#pragma unroll
        for (int e = 0; e < RowView<T>::VEC; ++e)
          if (key[e] > cut || (key[e] == cut && r++ < room)) {
            const uint32_t at = atomicAdd(&sh.listed, 1u);
            sh.list[at] = (static_cast<uint64_t>(key[e]) << 32) | ~static_cast<uint32_t>(v.first(b) + e);
          }
        return true;
      });
      __syncthreads();
      n = kk;
    }
    row_order(sh.list, sh.hist, n);
  }
  for (int i = threadIdx.x; i < k; i += kRowThreads) {
    const uint64_t e = i < kk ? sh.hist[i] : 0;
    values[row * k + i] = i < kk ? K::value(static_cast<uint32_t>(e >> 32)) : -INFINITY;
    ids[row * k + i] = i < kk ? static_cast<int64_t>(~static_cast<uint32_t>(e)) : -1;
  }
}

// ------------------------------------------------------------------------------------------------
// Sampling
// ------------------------------------------------------------------------------------------------

// Order-preserving integer of a number, rounded down to the key's bits: every entry at or above x has a
// key at or above this.
template <typename T>
__device__ __forceinline__ uint32_t row_key_floor(float x) {
  const uint32_t b = __float_as_uint(x);
  return ((b & 0x80000000u) ? ~b : (b | 0x80000000u)) >> (32 - RowKey<T>::BITS);
}


// Filters the n listed entries and picks the token: the kept ones among the top_k largest and the ties
// of the last (top_k 0: among all). `mass` is the total that top-p refers to (0: the list's own); then
// the list is the head of the row's order, and the result is false if the border lies beyond it.
template <typename T>
__device__ bool row_pick_listed(int n, int top_k, float top_p, uint64_t mass, uint64_t least, float uniform,
                                const RowWeight& weight, RowScratch& sh, int64_t* __restrict__ token) {
  using K = RowKey<T>;
  constexpr int PER = kRowList / kRowThreads;
  uint64_t w[PER], own = 0, total;
  if (mass) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (threadIdx.x + j * kRowThreads < n)
        own += weight(K::value(static_cast<uint32_t>(sh.list[threadIdx.x + j * kRowThreads] >> 32)));
    if (floor_share(top_p, mass) >= block_sum_u64(own, sh)) return false;
    own = 0;
  }
  uint64_t* sorted = sh.hist;
  row_order(sh.list, sorted, n);
  const uint32_t kth = top_k ? static_cast<uint32_t>(sorted[top_k - 1] >> 32) : 0u;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int at = threadIdx.x * PER + j;
    const uint32_t key = at < n ? static_cast<uint32_t>(sorted[at] >> 32) : 0u;
    w[j] = at < n && key >= kth ? weight(K::value(key)) : 0;
    own += w[j];
  }
  uint64_t before = block_exclusive_u64(own, sh, total);
  const uint64_t target = top_p < 1.f ? floor_share(top_p, mass ? mass : total) : ~0ull;
  uint64_t* kept = sh.list;  // row_order has read the list
  own = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int at = threadIdx.x * PER + j;
    const uint64_t keep = before <= target && w[j] >= least ? w[j] : 0;
    before += w[j];
    own += keep;
    if (at < n) kept[at] = keep;
  }
  const uint64_t aim = floor_share(uniform, block_sum_u64(own, sh));
  // the running sum before an entry in index order is the weight of the kept entries of lower index
  int parts = 32;
  while (parts > 1 && parts * n > kRowThreads) parts >>= 1;
  const int stride = kRowThreads / parts, part = threadIdx.x % parts;
  for (int e0 = 0; e0 < n; e0 += stride) {
    const int e = e0 + threadIdx.x / parts;
    const uint32_t place = e < n ? static_cast<uint32_t>(sorted[e]) : 0u;
    const uint64_t mine = e < n ? kept[e] : 0;
    uint64_t run = 0;
    if (mine)
      for (int j = part; j < n; j += parts)
        if (static_cast<uint32_t>(sorted[j]) > place) run += kept[j];
    for (int o = parts >> 1; o > 0; o >>= 1) run += __shfl_xor_sync(0xffffffffu, run, o);
    if (mine && part == 0 && run <= aim && aim < run + mine) *token = ~place;
  }
  return true;
}

// A slice's weight at the row's maximum: as it is where the slice holds that maximum, else brought down.
__device__ __forceinline__ uint64_t row_slice_mass(const RowSlice& a, uint32_t top_key, float slice_top,
                                                   const RowWeight& weight, float temperature) {
  if (a.top == top_key || a.top == 0) return a.mass;
  return __double2ull_rn(static_cast<double>(a.mass) *
                         exp((static_cast<double>(slice_top) - static_cast<double>(weight.top)) / temperature));
}

// One step of a warp's walk to the token: the weights of each lane's block, in index order, on top of
// `run`; writes the token where `aim` falls and returns whether it lies further on.
template <int VEC>
__device__ __forceinline__ bool row_warp_find(const uint64_t (&w)[VEC], uint64_t& run, uint64_t aim, int first,
                                              int64_t* __restrict__ token) {
  const int lane = threadIdx.x & 31;
  uint64_t mine = 0;
#pragma unroll
  for (int e = 0; e < VEC; ++e) mine += w[e];
  uint64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  uint64_t at = run + inc - mine;
  run += __shfl_sync(0xffffffffu, inc, 31);
  if (at <= aim && aim < at + mine)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (at <= aim && aim < at + w[e]) *token = first + e;
      at += w[e];
    }
  return run <= aim;
}

// Samples from the nucleus of the whole row; `mass` is the weight of all candidates and `target` top-p's
// share of it. Entries that weigh at most (mass - target - 1) / V together weigh less than
// mass - target, so the border lies above them. The others are counted (32-bit counts, no weights) in
// 2048 bins even in x; as the entries of a bin weigh the same within a percent, the counts bound the
// running weight from both sides and leave a few bins that can hold the border. A second pass, in
// index order, sums what lies above those bins exactly and lists what lies in them. False where that
// list is too long (the caller then selects by radix).
template <typename T>
__device__ bool row_pick_nucleus(const RowView<T>& v, const uint32_t* maxima, float temperature, uint64_t mass,
                                 uint64_t target, uint64_t least, float uniform, const RowWeight& weight,
                                 RowScratch& sh, int64_t* __restrict__ token) {
  using K = RowKey<T>;
  constexpr int VEC = RowView<T>::VEC;
  const float top = weight.top;
  // how far below the maximum (times T) the border can lie, with a margin that covers the fp32 arithmetic;
  // weights are rounded, so one of light + 1 stands for light + 1/2 or more
  const uint64_t light = (mass - target - 1) / static_cast<uint64_t>(v.V);
  const float depth = (static_cast<float>(weight.S) - log2f(static_cast<float>(light) + 0.5f)) * kLn2 + 1e-3f;
  const float range = depth * temperature + 1e-5f * fabsf(top);
  if (!(top < INFINITY) || !(range < INFINITY)) return false;
  const float inv = static_cast<float>(kRowBins) / range, step = range / (temperature * kRowBins);
  const uint32_t low = row_key_floor<T>(top - range);
  auto bin = [&](uint32_t key) { return min(kRowBins - 1, static_cast<int>((top - K::value(key)) * inv)); };
  uint32_t* counts = reinterpret_cast<uint32_t*>(sh.hist);
  for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) counts[i] = 0;
  if (threadIdx.x == 0) {
    sh.found[0] = ~0ull;
    sh.found[1] = kRowBins - 1;
    sh.listed = 0;
  }
  __syncthreads();
  row_visit<T>(v, [&](int, uint32_t key) {
    if (key >= low) atomicAdd(&counts[bin(key)], 1u);
  });
  __syncthreads();
  // bounds of an entry's weight at a bin's ends, 2e-4 wider than the fp32 arithmetic needs, and of the
  // running weight
  constexpr int BINS = kRowBins / kRowThreads;
  uint32_t c[BINS];
  uint64_t most[BINS], fewest[BINS], sum_most = 0, sum_fewest = 0, total;
#pragma unroll
  for (int j = 0; j < BINS; ++j) {
    const int b = threadIdx.x * BINS + j;
    c[j] = counts[b];
    const double one = static_cast<double>(1ull << weight.S);
    most[j] = c[j] * (__double2ull_ru(expf(-step * b) * 1.0002 * one) + 1);
    fewest[j] = b == kRowBins - 1 ? 0 : c[j] * __double2ull_rd(expf(-step * (b + 1)) * 0.9998 * one);
    sum_most += most[j];
    sum_fewest += fewest[j];
  }
  uint64_t hi = block_exclusive_u64(sum_most, sh, total), lo = block_exclusive_u64(sum_fewest, sh, total);
#pragma unroll
  for (int j = 0; j < BINS; ++j) {
    if (hi <= target && target < hi + most[j]) sh.found[0] = threadIdx.x * BINS + j;
    if (lo <= target && target < lo + fewest[j]) sh.found[1] = threadIdx.x * BINS + j;
    hi += most[j];
    lo += fewest[j];
  }
  __syncthreads();
  if (sh.found[0] == ~0ull) return false;
  const int b1 = static_cast<int>(sh.found[0]), b2 = static_cast<int>(sh.found[1]);  // bins that can hold the border
  uint64_t inside = 0;
#pragma unroll
  for (int j = 0; j < BINS; ++j) {
    const int b = threadIdx.x * BINS + j;
    if (b >= b1 && b <= b2) inside += c[j];
  }
  if (block_sum_u64(inside, sh) > kRowList) return false;
  // no entry of those bins or above lies below this key
  const uint32_t floor_key = b2 == kRowBins - 1 ? low : max(low, row_key_floor<T>(top - (b2 + 1) * 1.00001f / inv - 1e-6f * fabsf(top)));
  uint64_t above = 0, kept = 0;
  row_warp_walk<T>(v, maxima, floor_key, [&](int b, const uint32_t(&key)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int at = key[e] >= floor_key ? bin(key[e]) : kRowBins;
      if (at < b1) {
        const uint64_t w = weight(K::value(key[e]));
        above += w;
        kept += w >= least ? w : 0;
      }
      row_append(at >= b1 && at <= b2, (static_cast<uint64_t>(key[e]) << 32) | ~static_cast<uint32_t>(v.first(b) + e),
                 sh.list, &sh.listed);
    }
    return true;
  });
  __syncthreads();
  const int n = static_cast<int>(sh.listed);
  uint64_t before = block_sum_u64(above, sh);
  if (n == 0 || target < before) return false;
  // the border: the listed entry at which the running weight passes the target
  uint64_t* sorted = sh.hist;
  if (threadIdx.x == 0) sh.found[0] = ~0ull;
  row_order(sh.list, sorted, n);
  constexpr int PER = kRowList / kRowThreads;
  uint64_t w[PER], own = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int at = threadIdx.x * PER + j;
    w[j] = at < n ? weight(K::value(static_cast<uint32_t>(sorted[at] >> 32))) : 0;
    own += w[j];
  }
  before += block_exclusive_u64(own, sh, total);
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (before <= target && target < before + w[j]) sh.found[0] = threadIdx.x * PER + j;
    before += w[j];
  }
  __syncthreads();
  if (sh.found[0] == ~0ull) return false;
  const int last = static_cast<int>(sh.found[0]);
  const uint64_t border = sorted[last];
  // the kept weight of each warp's range of the row
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = row_warp_steps(v.blocks);
  for (int j = lane; j <= last; j += 32) {
    const int i = static_cast<int>(~static_cast<uint32_t>(sorted[j]));
    if ((i + v.off) / VEC / 32 / per != warp) continue;
    const uint64_t wj = weight(K::value(static_cast<uint32_t>(sorted[j] >> 32)));
    kept += wj >= least ? wj : 0;
  }
  kept = warp_sum_u64(kept);
  uint64_t run = __shfl_sync(0xffffffffu, block_exclusive_u64(lane == 0 ? kept : 0, sh, total), 0);
  const uint64_t aim = floor_share(uniform, total);
  if (run > aim || aim >= run + kept) return true;
  row_warp_walk<T>(v, maxima, floor_key, [&](int b, const uint32_t(&key)[VEC]) {
    uint64_t we[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const uint64_t entry = (static_cast<uint64_t>(key[e]) << 32) | ~static_cast<uint32_t>(v.first(b) + e);
      we[e] = entry >= border && key[e] ? weight(K::value(key[e])) : 0;
      we[e] = we[e] >= least ? we[e] : 0;
    }
    return row_warp_find<VEC>(we, run, aim, v.first(b), token);
  });
  return true;
}

// Picks the token by going over the row in index order: kept are the entries above `cut` and the first
// `ties` equal to it, as far as they weigh `least`; no entry below the key `lowest` does.
template <typename T>
__device__ void row_pick_walk(const RowView<T>& v, const uint32_t* maxima, uint32_t cut, uint64_t ties, uint32_t lowest,
                              uint64_t least, float uniform, const RowWeight& weight, RowScratch& sh,
                              int64_t* __restrict__ token) {
  using K = RowKey<T>;
  constexpr int VEC = RowView<T>::VEC;
  const int lane = threadIdx.x & 31;
  const uint64_t cut_weight = weight(K::value(cut));
  if (cut_weight < least) ties = 0;
  const uint32_t low = max(cut, lowest);
  auto above = [&](uint32_t key) -> uint64_t {
    if (key <= cut || key < lowest) return 0;
    const uint64_t w = weight(K::value(key));
    return w >= least ? w : 0;
  };
  uint64_t sum = 0;
  uint32_t eq = 0;
  row_warp_walk<T>(v, maxima, low, [&](int, const uint32_t(&key)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sum += above(key[e]);
      eq += key[e] == cut;
    }
    return true;
  });
  // of each warp's range: its equals inside, its weight, the weight before it
  uint64_t all;
  uint64_t rank = __shfl_sync(0xffffffffu, block_exclusive_u64(eq, sh, all), 0);
  const uint64_t equals = __reduce_add_sync(0xffffffffu, eq);
  const uint64_t inside = rank < ties ? min(ties - rank, equals) : 0;
  sum = warp_sum_u64(sum) + inside * cut_weight;
  uint64_t run = __shfl_sync(0xffffffffu, block_exclusive_u64(lane == 0 ? sum : 0, sh, all), 0);
  const uint64_t aim = floor_share(uniform, all);
  if (run > aim || aim >= run + sum) return;
  row_warp_walk<T>(v, maxima, low, [&](int b, const uint32_t(&key)[VEC]) {
    uint32_t same = 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) same += key[e] == cut;
    uint32_t se = same;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, se, o);
      if (lane >= o) se += u;
    }
    uint64_t r = rank + se - same;
    rank += __shfl_sync(0xffffffffu, se, 31);
    uint64_t w[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[e] = key[e] == cut ? (r++ < ties ? cut_weight : 0) : above(key[e]);
    return row_warp_find<VEC>(w, run, aim, v.first(b), token);
  });
}

// Picks the token of an unfiltered row from the slices' weights: the slice that holds the uniform's
// share, and in it the entry, by the slice's own weights.
template <typename T, int BLOCKS>
__device__ void row_pick_slice(const RowView<T>& v, const RowScan& scan, int64_t row, uint32_t top_key,
                               float temperature, float uniform, const RowWeight& weight, RowScratch& sh,
                               int64_t* __restrict__ token) {
  using K = RowKey<T>;
  constexpr int VEC = RowView<T>::VEC, SLICE = BLOCKS * kScanThreads;
  RowSlice a{0u, 0u, 0ull};
  uint64_t own = 0, total;
  if (static_cast<int>(threadIdx.x) < scan.slices) {
    a = scan.slice[row * scan.slices + threadIdx.x];
    own = row_slice_mass(a, top_key, K::value(a.top), weight, temperature);
  }
  const uint64_t run = block_exclusive_u64(own, sh, total);
  uint64_t aim = floor_share(uniform, total);
  if (run <= aim && aim < run + own) {
    aim -= run;
    if (own != a.mass) {  // the share of the slice's own weight
      const double f = static_cast<double>(aim) / static_cast<double>(own) * static_cast<double>(a.mass);
      aim = min(static_cast<uint64_t>(__double2ull_rd(f)), a.mass - 1);
    }
    sh.found[0] = (static_cast<uint64_t>(a.top) << 32) | threadIdx.x;
    sh.found[1] = aim;
  }
  __syncthreads();
  const RowWeight local = row_weight(K::value(static_cast<uint32_t>(sh.found[0] >> 32)), temperature, weight.S, sh.exp_tab);
  const int b0 = static_cast<int>(sh.found[0] & 0xFFFFFFFFu) * SLICE;
  aim = sh.found[1];
  constexpr int PER = SLICE > kRowThreads ? SLICE / kRowThreads : 1;  // blocks of a thread, neighbours
  uint32_t key[PER][VEC];
  uint64_t mine = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int at = threadIdx.x * PER + j;
    if (at < SLICE) {
      v.keys(b0 + at, key[j]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) key[j][e] = 0u;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (key[j][e]) mine += local(K::value(key[j][e]));
  }
  uint64_t at = block_exclusive_u64(mine, sh, total);
  if (at <= aim && aim < at + mine)
#pragma unroll
    for (int j = 0; j < PER; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const uint64_t w = key[j][e] ? local(K::value(key[j][e])) : 0;
        if (at <= aim && aim < at + w) *token = v.first(b0 + threadIdx.x * PER + j) + e;
        at += w;
      }
}

template <typename T, int BLOCKS>
__global__ void __launch_bounds__(kRowThreads, 2)
    sample_logits_kernel(const T* __restrict__ x, int64_t ldx, int V, int S, const float* __restrict__ uniform,
                         SampleKnobs knobs, RowScan scan, int64_t* __restrict__ tokens) {
  using K = RowKey<T>;
  constexpr int LANES = kRowGroup / RowView<T>::VEC;
  extern __shared__ __align__(16) uint32_t row_maxima[];
  __shared__ RowScratch sh;
  const int64_t row = blockIdx.x;
  const RowView<T> v(x + row * ldx, V);
  row_exp_table(sh.exp_tab);
  griddep_wait();  // launched as a programmatic dependent of the scan
  const SampleRow knob(knobs, row);
  const float u = uniform[row], T_ = knob.temperature;
  const uint32_t top_key = row_open(scan, row, row_maxima, sh);
  if (top_key == 0) {
    if (threadIdx.x == 0) tokens[row] = -1;
    return;
  }
  if (knob.greedy) {  // the first group with the largest key, its first entry
    uint32_t g = 0xFFFFFFFFu;
    for (int i = threadIdx.x; i < scan.groups; i += kRowThreads)
      if (row_maxima[i] == top_key) g = min(g, static_cast<uint32_t>(i));
    g = __reduce_min_sync(0xffffffffu, g);
    if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = g;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    for (int w = 0; w < kRowWarps; ++w) g = min(g, static_cast<uint32_t>(sh.warp[w]));
    uint32_t at = 0xFFFFFFFFu;
    if (threadIdx.x < LANES) {
      uint32_t k[RowView<T>::VEC];
      const int b = static_cast<int>(g) * LANES + threadIdx.x;
      v.keys(b, k);
#pragma unroll
      for (int e = RowView<T>::VEC - 1; e >= 0; --e)
        if (k[e] == top_key) at = v.first(b) + e;
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (threadIdx.x == 0) tokens[row] = at;
    return;
  }
  const RowWeight weight = row_weight(K::value(top_key), T_, S, sh.exp_tab);
  // min-p: weights below `least` leave; no entry below the key `lowest` passes (lower by a margin that
  // covers fp32)
  const float floor_p = fminf(fmaxf(knob.min_p, 0.f), 1.f);
  const uint64_t least = __double2ull_ru(static_cast<double>(floor_p) * (1ull << S));
  uint32_t lowest = 1u;
  if (floor_p > 0.f)
    lowest = weight.top < INFINITY
                 ? max(1u, row_key_floor<T>(weight.top + T_ * (logf(floor_p) - 1e-3f) - 1e-5f * fabsf(weight.top)))
                 : top_key;

  // a top-k that is smaller than the number of candidates
  bool filtered = false;
  if (knob.top_k > kRowMaxK) {
    uint64_t candidates = 0;
    row_visit<T>(v, [&](int, uint32_t) { ++candidates; });
    filtered = static_cast<uint64_t>(knob.top_k) < block_sum_u64(candidates, sh);
  } else if (knob.top_k >= 1) {
    const uint32_t bound = row_bound(row_maxima, scan.groups, knob.top_k, top_key, sh);
    const int n = row_gather<T>(v, row_maxima, scan.groups, bound, sh);
    if (n <= kRowList) {  // with fewer than top_k entries, all there are
      row_pick_listed<T>(n, min(n, knob.top_k), knob.top_p, 0, least, u, weight, sh, tokens + row);
      return;
    }
    filtered = true;
  }
  uint32_t cut = 1u;
  uint64_t before, ties = ~0ull;
  if (filtered) cut = row_radix_select<T, false>(v, 1u, knob.top_k - 1, weight, sh, before);
  if (knob.top_p < 1.f) {
    uint64_t mass = 0;
    if (knob.wants_mass()) {
      if (static_cast<int>(threadIdx.x) < scan.slices) {
        const RowSlice a = scan.slice[row * scan.slices + threadIdx.x];
        mass = row_slice_mass(a, top_key, K::value(a.top), weight, T_);
      }
    } else {
      row_visit<T>(v, [&](int, uint32_t key) {
        if (key >= cut) mass += weight(K::value(key));
      });
    }
    mass = block_sum_u64(mass, sh);
    const uint64_t target = floor_share(knob.top_p, mass);
    if (!filtered) {
      // the head of the order first: a nucleus is usually a few hundred entries
      const uint32_t bound = row_bound(row_maxima, scan.groups, kRowMaxK, top_key, sh);
      const int n = row_gather<T>(v, row_maxima, scan.groups, bound, sh);
      const bool whole_row = n < kRowMaxK || bound == 1u;
      if (n <= kRowList && row_pick_listed<T>(n, 0, knob.top_p, whole_row ? 0 : mass, least, u, weight, sh, tokens + row))
        return;
      __syncthreads();
      if (row_pick_nucleus<T>(v, row_maxima, T_, mass, target, least, u, weight, sh, tokens + row)) return;
      __syncthreads();
    }
    cut = row_radix_select<T, true>(v, cut, target, weight, sh, before);
    ties = (target - before) / weight(K::value(cut)) + 1;
  } else if (!filtered && floor_p > 0.f) {
    const int n = row_gather<T>(v, row_maxima, scan.groups, lowest, sh);
    if (n <= kRowList) {
      row_pick_listed<T>(n, 0, 1.f, 0, least, u, weight, sh, tokens + row);
      return;
    }
  } else if (!filtered && knob.wants_mass()) {
    row_pick_slice<T, BLOCKS>(v, scan, row, top_key, T_, u, weight, sh, tokens + row);
    return;
  }
  row_pick_walk<T>(v, row_maxima, cut, ties, lowest, least, u, weight, sh, tokens + row);
}

// ------------------------------------------------------------------------------------------------
// Launch
// ------------------------------------------------------------------------------------------------

struct RowPlan {
  int groups, slices, blocks;  // blocks: 16-byte blocks of a scan thread
  size_t off_slice, total;
};

// Slices of 8192 entries, 32 a thread in flight; of 2048 where that leaves SMs without a slice (a
// few rows). `aligned`: every row starts on a 16-byte boundary.
inline RowPlan row_plan(int64_t R, int64_t V, int elem, bool aligned) {
  RowPlan p{};
  const int vec = 16 / elem;
  p.groups = static_cast<int>(ceil_div(V + (aligned ? 0 : vec - 1), 4 * kRowGroup)) * 4;
  const bool small = R * ceil_div(V, 8192) < 2 * num_sms() && V <= (1 << 19);
  p.blocks = (small ? 2048 : 8192) / vec / kScanThreads;
  p.slices = static_cast<int>(ceil_div(static_cast<int64_t>(p.groups) * kRowGroup, static_cast<int64_t>(p.blocks) * kScanThreads * vec));
  p.off_slice = (static_cast<size_t>(R) * p.groups * 4 + 255) / 256 * 256;
  p.total = p.off_slice + static_cast<size_t>(R) * p.slices * sizeof(RowSlice);
  return p;
}

// Bytes that do for any alignment.
inline size_t row_ws_bytes(int64_t R, int64_t V, int elem) {
  return std::max(row_plan(R, V, elem, true).total, row_plan(R, V, elem, false).total);
}

template <typename T, bool SAMPLE>
int row_scan_launch(const RowPlan& p, const T* x, int64_t ldx, int64_t R, int V, float temperature, int S,
                    const SampleKnobs& knobs, const RowScan& scan, cudaStream_t stream) {
  constexpr int BIG = 8192 / RowView<T>::VEC / kScanThreads, SMALL = 2048 / RowView<T>::VEC / kScanThreads;
  const unsigned grid = static_cast<unsigned>(R * p.slices);
  if (p.blocks == BIG)
    row_scan_kernel<T, BIG, SAMPLE><<<grid, kScanThreads, 0, stream>>>(x, ldx, V, temperature, S, knobs, scan);
  else
    row_scan_kernel<T, SMALL, SAMPLE><<<grid, kScanThreads, 0, stream>>>(x, ldx, V, temperature, S, knobs, scan);
  ORTHRUS_CHECK_LAUNCH();
  return ORTHRUS_OK;
}

template <typename T>
inline int row_prepare(const T* x, int64_t ldx, int64_t R, int64_t V, void* ws, size_t ws_bytes, RowPlan& p,
                       RowScan& scan) {
  p = row_plan(R, V, sizeof(T), aligned16(x) && (ldx * sizeof(T)) % 16 == 0);
  ORTHRUS_CHECK_ARG(R * p.slices < (1ll << 31) && (reinterpret_cast<uintptr_t>(x) & (sizeof(T) - 1)) == 0);
  if (ws == nullptr || ws_bytes < p.total) return ORTHRUS_EWORKSPACE;
  scan = {static_cast<uint32_t*>(ws), reinterpret_cast<RowSlice*>(static_cast<uint8_t*>(ws) + p.off_slice), p.groups,
          p.slices};
  return ORTHRUS_OK;
}

constexpr int kRowSmem = (kRowMaxV + 8) / kRowGroup * 4 + 32;  // the group maxima of the longest row

template <typename T>
int topk_rows_impl(const T* x, int64_t ldx, int64_t R, int64_t V, int k, float temperature, float* values, int64_t* ids,
                   float* lse, void* ws, size_t ws_bytes, cudaStream_t stream) {
  RowPlan p;
  RowScan scan;
  int rc = row_prepare(x, ldx, R, V, ws, ws_bytes, p, scan);
  if (rc != ORTHRUS_OK) return rc;
  rc = row_scan_launch<T, false>(p, x, ldx, R, static_cast<int>(V), temperature, 0, SampleKnobs{}, scan, stream);
  if (rc != ORTHRUS_OK) return rc;
  ORTHRUS_CHECK_CUDA(ensure_smem(topk_rows_kernel<T>, kRowSmem));
  ORTHRUS_CHECK_CUDA(launch_pdl(topk_rows_kernel<T>, dim3(static_cast<unsigned>(R)), dim3(kRowThreads),
                                p.groups * 4, stream, x, ldx, static_cast<int>(V), k, temperature, scan, values,
                                ids, lse));
  ORTHRUS_CHECK_LAUNCH();
  return ORTHRUS_OK;
}

template <typename T, int BLOCKS>
int sample_finish_launch(const RowPlan& p, const T* x, int64_t ldx, int64_t R, int V, int S, const float* uniform,
                         const SampleKnobs& knobs, const RowScan& scan, int64_t* tokens, cudaStream_t stream) {
  auto kernel = sample_logits_kernel<T, BLOCKS>;
  ORTHRUS_CHECK_CUDA(ensure_smem(kernel, kRowSmem));
  ORTHRUS_CHECK_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(R)), dim3(kRowThreads), p.groups * 4,
                                stream, x, ldx, V, S, uniform, knobs, scan, tokens));
  ORTHRUS_CHECK_LAUNCH();
  return ORTHRUS_OK;
}

template <typename T>
int sample_logits_impl(const T* x, int64_t ldx, int64_t R, int64_t V, const float* uniform, const SampleKnobs& knobs,
                       int64_t* tokens, void* ws, size_t ws_bytes, cudaStream_t stream) {
  RowPlan p;
  RowScan scan;
  int rc = row_prepare(x, ldx, R, V, ws, ws_bytes, p, scan);
  if (rc != ORTHRUS_OK) return rc;
  const int n = static_cast<int>(V), S = row_weight_bits(n);
  rc = row_scan_launch<T, true>(p, x, ldx, R, n, 1.f, S, knobs, scan, stream);
  if (rc != ORTHRUS_OK) return rc;
  constexpr int BIG = 8192 / RowView<T>::VEC / kScanThreads, SMALL = 2048 / RowView<T>::VEC / kScanThreads;
  return p.blocks == BIG ? sample_finish_launch<T, BIG>(p, x, ldx, R, n, S, uniform, knobs, scan, tokens, stream)
                         : sample_finish_launch<T, SMALL>(p, x, ldx, R, n, S, uniform, knobs, scan, tokens, stream);
}

}  // namespace orthrus
