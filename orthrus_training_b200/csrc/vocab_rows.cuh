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
//   - A nucleus without top-k is looked for among the 256 largest entries.
//   - Without a filter the slices' weights say which slice holds the uniform's share.
// Sampled rows that keep more than fits a CTA's shared memory (wide rows: nuclei of thousands of entries)
// get more launches: a scan that bins their weights and so finds a narrow window of values with the
// nucleus' border, one that sums what lies above the window and lists what lies in it, and a pick. Where
// even that does not do, a CTA goes over the whole row again: a radix selection that is right for every
// row, and a walk in index order. Those are rows of many equal values, wide rows past the first 2048 of a
// call (50257 entries, top-p 0.95 at T = 1.5: 2048 rows 750 us, 2100 rows 1113), a top-k above 1024, and
// rows with more than 2048 candidates in fewer than k groups, which give no bound: k = 300 with V from
// 2049 to 9600, k = 1024 to 32768, a nucleus (k = 256) to 8192, longer rows whose candidates stand
// together (256 rows fp32: top-300 at V = 8000 80 us, at 12000 43; top-p 0.9 at V = 8000 125, at 9000 99).
//
// What bounds it, and what it measured (us; V = 151936 where not given; floor: each logit read once at
// 6540 GB/s):
//   top-64, 1024 rows fp32           127 (floor 95): the scan 96 (6.5 TB/s), then the finish, whose one and a
//                                    half waves of CTAs wait for memory and barriers, 25
//   top-300, 333 x 50257 bf16         37 (5.3): the finish
//   top-8, 2 x 1024; top-64, 32 rows  18, 18: the call's host time (7 and 18 on the device)
//   plain sampling, 1 row             16: the call's host time (10 on the device)
//   top-p 0.95, 256 rows fp32        247 (24), every row wide: scan 69, finish 38, bins 43, window 6, sums 50,
//                                    pick 25. The scan is bound by instructions, 42 an entry, 15 of them
//                                    fp64 at half rate for the integer weight, the bins and sums by
//                                    those of passing over the entries (28 and 31)
//   mixed filters, 1024 rows bf16    258 (48): scan 96, finish 54, wide rows the rest
//   min-p 0.05, 77 x 32003 fp32       23 (1.5): latency of two dependent launches
// One CTA per row for all of it (a cluster, or a CTA going over its row again) took 576 us for the first,
// and 1490 against 254 for the wide nuclei: few bytes in flight. The finish is mostly code that runs once
// per row, so that fetching instructions costs more than executing them: what is not a hot loop is kept
// rolled and out of line.
//
// Candidates are the entries that are neither -inf nor NaN. Entries are ordered by (descending
// value, ascending index); -0 counts as +0.
#pragma once

#include <cuda_bf16.h>

#include "sm100.cuh"

namespace orthrus {

constexpr int kRowThreads = 256;          // of the CTA that finishes a row
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kScanThreads = 256;
constexpr int kRowGroup = 32;             // entries behind one group maximum
constexpr int kRowBins = 2048;
constexpr int kRowMaxK = 1024;            // largest k of topk_rows
constexpr int kRowList = 2048;            // most entries gathered into shared memory
constexpr int kRowWideShare = 8;          // a wide row's window lists at most one in so many of a slice's entries
constexpr int kRowWideBins = 512;         // weight bins of a wide row
constexpr int kRowWideRows = 2048;        // most wide rows of a call
constexpr int kRowHead = 256;             // entries among which a nucleus is looked for first
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

// Key of entry i, 0 outside the row. Out of line: only a row's ends need it, and in line it would be most
// of the code of every loop over a row (whose instruction fetches are what such a loop waits for).
template <typename T>
__device__ __noinline__ uint32_t row_key_at(const T* p, int V, int i) {
  if (i < 0 || i >= V) return 0u;
  if constexpr (sizeof(T) == 4)
    return RowKey<T>::of_bits(__ldg(reinterpret_cast<const uint32_t*>(p) + i));
  else
    return RowKey<T>::of_bits(__ldg(reinterpret_cast<const uint16_t*>(p) + i));
}

// The 16 bytes of a block that is not all within the row, with -inf outside it. Out of line, as above.
template <typename T>
__device__ __noinline__ uint4 row_raw_edge(const T* p, int V, int first) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 4) {
      const int i = first + e;
      w[e] = i < 0 || i >= V ? 0xFF800000u : __ldg(reinterpret_cast<const uint32_t*>(p) + i);
    } else {
      const int i = first + 2 * e;
      const uint32_t a = i < 0 || i >= V ? 0xFF80u : __ldg(reinterpret_cast<const uint16_t*>(p) + i);
      const uint32_t b = i + 1 < 0 || i + 1 >= V ? 0xFF80u : __ldg(reinterpret_cast<const uint16_t*>(p) + i + 1);
      w[e] = a | b << 16;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

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
  // block b as it is in memory, -inf outside the row
  __device__ __forceinline__ uint4 raw(int b) const {
    if (b < blocks) return whole(b) ? load(b) : row_raw_edge<T>(p, V, first(b));
    constexpr uint32_t none = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
    return make_uint4(none, none, none, none);
  }
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
  __device__ __forceinline__ uint32_t key(int i) const { return row_key_at<T>(p, V, i); }
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
  union {
    uint64_t list[kRowList];   // gathered entries, (key << 32 | ~index)
    uint32_t counts[kRowBins]; // histograms; done with before entries are gathered
  };
  uint64_t warp[kRowWarps];
  uint32_t top[kRowWarps];
  uint64_t found[2];         // result of a block-wide search
  union {
    uint64_t hist[kRowBins];           // weights of a radix selection
    uint64_t sorted[kRowList];         // the list in order
    uint32_t groups[kRowList];         // numbers of the groups to read again
  };
  uint32_t ngroups, listed;
};

// The finishing CTA's shared memory: the scratch, then the row's group maxima. The functions below
// reach it by name rather than through a reference, so that those kept out of line (the finish is
// long, and mostly run once per row: instruction fetches are what it waits for most) still use
// shared-memory instructions.
extern __shared__ __align__(16) uint8_t row_smem[];
__device__ __forceinline__ RowScratch& row_scratch() { return *reinterpret_cast<RowScratch*>(row_smem); }
__device__ __forceinline__ uint32_t* row_maxima() {
  return reinterpret_cast<uint32_t*>(row_smem + (sizeof(RowScratch) + 15) / 16 * 16);
}

__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct uint2x64 {
  uint64_t x, y;
};

// Block-wide sum; every thread gets it.
__device__ __noinline__ uint64_t block_sum_u64(uint64_t v) {
  RowScratch& sh = row_scratch();
  v = warp_sum_u64(v);
  const int lane = threadIdx.x & 31;
  if (lane == 0) sh.warp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < kRowWarps ? sh.warp[lane] : 0;
  __syncthreads();
  return warp_sum_u64(v);
}

// Exclusive prefix sum over the block's threads, and the block's sum.
__device__ __noinline__ uint2x64 block_exclusive2(uint64_t v) {
  RowScratch& sh = row_scratch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) sh.warp[warp] = inc;
  __syncthreads();
  const uint64_t w = lane < kRowWarps ? sh.warp[lane] : 0;
  __syncthreads();
  return {inc - v + warp_sum_u64(lane < warp ? w : 0), warp_sum_u64(w)};
}
__device__ __forceinline__ uint64_t block_exclusive_u64(uint64_t v, uint64_t& total) {
  const uint2x64 r = block_exclusive2(v);
  total = r.y;
  return r.x;
}

// ------------------------------------------------------------------------------------------------
// Softmax weights as 64-bit integers
// ------------------------------------------------------------------------------------------------

// w(x) = round(2^S exp((x - top) / T)). Integer weights make sums exact, so running sums do not
// depend on how a slice is split over threads. S = min(44, 62 - ceil(log2 V)) keeps a row's sum below
// 2^62; a weight is off by at most half a unit plus 2^-44 of itself, V of them by V / 2 units of a total
// of 2^S or more. What depends on where slices end: the scan weighs a slice against its own maximum,
// so that its units are finer than the row's, and brings its sum down in fp64.
//
// The exponential: y = (top - x) log2(e) / T = n - f with |f| <= 1/2, 2^f = 1 + f q(f) with q of degree
// 8 through the Chebyshev nodes of [-1/2, 1/2] (error below 4e-14), 2^(S - n) by the exponent. A table
// would save some of the fp64 products, but its lookups, of random banks, take longer. No branch, and
// what can be is left to fp32: the loops over rows are bound by the instructions that they issue.
__constant__ double kRowExp2[9] = {6.931471805599453e-01,  2.402265069581299e-01,  5.5504108664760424e-02,
                                   9.618129159402558e-03,  1.3333558179043112e-03, 1.5403455852453838e-04,
                                   1.525268684626772e-05,  1.3255224878668817e-06, 1.0203121063391729e-07};

struct RowWeight {
  float top;            // the maximum the weights refer to
  float floor;          // entries below are deeper than S + 3/2 bits: they weigh 0. +inf if top is
  int S;
  double from, scale;   // top, if finite; log2(e) / T

  __device__ __forceinline__ uint64_t operator()(float x) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    constexpr double kInt = 4503599627370496.0;    // 2^52
    const double y = (from - static_cast<double>(fminf(x, 3.4028234663852886e38f))) * scale;
    const double r = y + kRound;
    const double f = (r - kRound) - y;
    double q = kRowExp2[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) q = fma(q, f, kRowExp2[i]);
    const double p = fma(q, f, 1.0);
    const double w = __hiloint2double(__double2hiint(p) + ((S - __double2loint(r)) << 20), __double2loint(p)) + kInt;
    return x >= floor ? static_cast<uint64_t>(__double_as_longlong(w)) & 0xFFFFFFFFFFFFFull : 0ull;
  }
};

__host__ __device__ inline int row_weight_bits(int V) {
  int b = 0;
  while ((1ll << b) < V) ++b;
  return 62 - b < 44 ? 62 - b : 44;
}

__device__ __forceinline__ RowWeight row_weight(float top, float temperature, int S) {
  const double scale = 1.4426950408889634 / static_cast<double>(temperature);
  if (top == INFINITY) return {top, top, S, 3.4028234663852886e38, scale};
  const double from = static_cast<double>(top);
  return {top, __double2float_ru(from - (S + 1.5) / scale), S, from, scale};
}

// The same out of line, for the finish, which has many places that weigh an entry.
__device__ __noinline__ uint64_t row_weigh(float x, float floor, int S, double from, double scale) {
  return RowWeight{0.f, floor, S, from, scale}(x);
}
struct RowWeigher {
  float top, floor;
  int S;
  double from, scale;
  __device__ __forceinline__ explicit RowWeigher(const RowWeight& w)
      : top(w.top), floor(w.floor), S(w.S), from(w.from), scale(w.scale) {}
  __device__ __forceinline__ uint64_t operator()(float x) const { return row_weigh(x, floor, S, from, scale); }
};

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
  uint32_t* wide_count;  // cleared by the scan; may be null
};

// What a wide row's slice leaves: the weight above the window, the part of it that passes min-p, and the
// number of entries in the window.
struct RowSums {
  uint64_t above, kept;
  uint32_t listed;
};

// A wide row: the border of its nucleus lies in the window [lo, hi) of values, or (nucleus false) all
// entries from lo = hi on are kept. `bins`: the weights from the maximum down to lo, for the window.
struct RowWideRow {
  int64_t row;
  float top, lo, hi;
  uint64_t target;  // the weight at which the border lies
  bool nucleus;
  uint64_t bins[kRowWideBins];
  __device__ __forceinline__ float per_value() const { return static_cast<float>(kRowWideBins) / fmaxf(top - lo, 1e-30f); }
};

// The wide rows of a call: their records, sums [most, slices] and lists [most, slices, room].
struct RowWideRows {
  uint32_t* count;
  RowWideRow* rows;
  RowSums* sums;
  uint64_t* lists;
  int most, room;
};

struct SampleKnobs {
  const float* temperature;  // [R], or null: one value for every row
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature1, top_p1, min_p1;
  int top_k1;
};

// min-p as the least weight that passes.
__device__ __forceinline__ uint64_t row_least(float min_p, int S) {
  return __double2ull_ru(static_cast<double>(fminf(fmaxf(min_p, 0.f), 1.f)) * static_cast<double>(1ull << S));
}

// How a row is sampled, from its knobs.
struct SampleRow {
  float temperature, top_p, min_p;
  int top_k;
  bool greedy;
  __device__ __forceinline__ SampleRow(const SampleKnobs& k, int64_t row)
      : temperature(fminf(k.temperature ? k.temperature[row] : k.temperature1, 3e38f)),
        top_p(k.top_p ? k.top_p[row] : k.top_p1),
        min_p(k.min_p ? k.min_p[row] : k.min_p1),
        top_k(k.top_k ? k.top_k[row] : k.top_k1),
        greedy(!((k.temperature ? k.temperature[row] : k.temperature1) >= 1e-5f)) {}
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
  __shared__ float wtop[kScanThreads / 32], wsum[kScanThreads / 32];
  __shared__ uint64_t wmass[kScanThreads / 32];
  griddep_launch_dependents();
  if (SAMPLE && blockIdx.x == 0 && threadIdx.x == 0 && out.wide_count) *out.wide_count = 0;
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
  float m[BLOCKS], top = -INFINITY;
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) {
    m[j] = val[j][0];
#pragma unroll
    for (int e = 1; e < VEC; ++e) m[j] = fmaxf(m[j], val[j][e]);
    top = fmaxf(top, m[j]);
  }
  // the groups' maxima: halves of a group's lanes exchange halves of the blocks while there are several,
  // so that a lane ends with one group (block `held`) rather than every lane with all of its
  static_assert(BLOCKS <= LANES, "");
  int held = 0;
#pragma unroll
  for (int o = LANES / 2, n = BLOCKS; o > 0; o >>= 1) {
    if (n > 1) {
      n /= 2;
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < BLOCKS / 2; ++i)
        if (i < n) {
          const float other = __shfl_xor_sync(0xffffffffu, up ? m[i] : m[i + n], o);
          m[i] = fmaxf(up ? m[i + n] : m[i], other);
        }
      held += up ? n : 0;
    } else {
      m[0] = fmaxf(m[0], __shfl_xor_sync(0xffffffffu, m[0], o));
    }
  }
  const int g = (b0 + held * kScanThreads + static_cast<int>(threadIdx.x)) / LANES;
  if (lane % (LANES / BLOCKS) == 0 && g < out.groups) out.group[row * out.groups + g] = K::of(m[0]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) wtop[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kScanThreads / 32; ++w) top = fmaxf(top, wtop[w]);
  uint64_t mass = 0;
  float sum = 0.f;
  if constexpr (SAMPLE) {
    // the slice again, from L1: weighing it from registers would take 32 copies of the weight's code
    if (mass_wanted && top > -INFINITY) {
      const RowWeight weight = row_weight(top, temperature, S);
#pragma unroll 1
      for (int j = 0; j < BLOCKS; ++j) {
        float x[VEC];
        v.values(b0 + j * kScanThreads + threadIdx.x, x);
#pragma unroll
        for (int e = 0; e < VEC; ++e) mass += weight(x[e]);
      }
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
__device__ __forceinline__ uint32_t row_open(const RowScan& scan, int64_t row) {
  RowScratch& sh = row_scratch();
  uint32_t* maxima = row_maxima();
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
  return __reduce_max_sync(0xffffffffu, sh.top[threadIdx.x % kRowWarps]);
}

// A key with at least k entries of the row at or above it, and not many more: between the k-th largest
// maximum of a group and a little below it; 1 if fewer than k groups hold a candidate. Histograms of the maxima over the range of keys that
// can hold the bound, 512 bins at a time.
__device__ __noinline__ uint32_t row_bound(int groups, int k, uint32_t top_key) {
  RowScratch& sh = row_scratch();
  const uint32_t* maxima = row_maxima();
  constexpr int BIN_BITS = 9;  // two bins a thread
  static_assert(1 << BIN_BITS == 2 * kRowThreads, "");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t* counts = sh.counts;
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
  least = __reduce_min_sync(0xffffffffu, sh.top[lane % kRowWarps]);
  uint32_t lo = least, hi = top_key;  // the bound is in [lo, hi]
  uint32_t above = 0;                 // maxima above hi
  const uint32_t want = k, enough = k + k / 4 + 16;
  while (true) {
    const int shift = max(0, 32 - __clz(hi - lo) - BIN_BITS);
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
    const uint32_t run = above + inc - c0 - c1 + __reduce_add_sync(0xffffffffu, lane < warp ? sh.top[lane] : 0u);
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
__device__ __noinline__ int row_gather(const T* row, int V, int groups, uint32_t low) {
  RowScratch& sh = row_scratch();
  const uint32_t* maxima = row_maxima();
  const RowView<T> v(row, V);
  constexpr int LANES = kRowGroup / RowView<T>::VEC;
  const int lane = threadIdx.x & 31;
  // each thread marks its groups, 32 at a time, and takes their places with one atomic
#pragma unroll 1
  for (int i0 = threadIdx.x; i0 < groups / 4; i0 += 8 * kRowThreads) {
    uint32_t mine = 0;
#pragma unroll 1
    for (int j = 0; j < 8 && i0 + j * kRowThreads < groups / 4; ++j) {
      const uint4 q = reinterpret_cast<const uint4*>(maxima)[i0 + j * kRowThreads];
      mine |= ((q.x >= low) | (q.y >= low) << 1 | (q.z >= low) << 2 | (q.w >= low) << 3) << (4 * j);
    }
    uint32_t at = mine ? atomicAdd(&sh.ngroups, static_cast<uint32_t>(__popc(mine))) : 0u;
#pragma unroll 1
    for (; mine; mine &= mine - 1, ++at) {
      const int bit = __ffs(mine) - 1;
      if (at < kRowList) sh.groups[at] = 4 * (i0 + bit / 4 * kRowThreads) + bit % 4;
    }
  }
  __syncthreads();
  const int ng = static_cast<int>(sh.ngroups);  // every group holds at least one entry
  // LANES neighbouring lanes a group, four loads ahead; each thread marks its entries and takes their places
  // with one atomic. Values compare as their keys do from the lowest number up.
  if (ng <= kRowList) {
    using K = RowKey<T>;
    constexpr int AHEAD = 4, STEP = kRowThreads / LANES, VEC = RowView<T>::VEC;
    const float least = K::value(max(low, 0x00800000u >> (32 - K::BITS)));
    auto block = [&](int i) { return i < ng ? static_cast<int>(sh.groups[i]) * LANES + lane % LANES : v.blocks; };
#pragma unroll 1
    for (int i0 = static_cast<int>(threadIdx.x) / LANES; i0 < ng; i0 += AHEAD * STEP) {
      uint4 q[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) q[j] = v.raw(block(i0 + j * STEP));
      uint32_t mine = 0;
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        float x[VEC];
        RowView<T>::values_of(q[j], x);
#pragma unroll
        for (int e = 0; e < VEC; ++e) mine |= static_cast<uint32_t>(x[e] >= least) << (j * VEC + e);
      }
      uint32_t at = mine ? atomicAdd(&sh.listed, static_cast<uint32_t>(__popc(mine))) : 0u;
#pragma unroll 1
      for (; mine; mine &= mine - 1, ++at) {
        const int bit = __ffs(mine) - 1;
        const int i = v.first(block(i0 + bit / VEC * STEP)) + bit % VEC;
        if (at < kRowList) sh.list[at] = (static_cast<uint64_t>(v.key(i)) << 32) | ~static_cast<uint32_t>(i);
      }
    }
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

// Orders the scratch's list (n <= kRowList different entries) descending into `sorted`: by rank
// counting for a few entries, several threads an entry; else by a sorting network (top-64 of 16 rows of V
// = 151936 16.4 us by ranks, 18.5 by the network; top-120 18.8, 20.5; top-200 24.6, 22.6).
__device__ __noinline__ void row_order(int n) {
  uint64_t *in = row_scratch().list, *out = row_scratch().sorted;
  if (n <= 160) {
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

// f(index, key) for every candidate of the row, each by one thread, four loads at a time.
template <typename T, typename F>
__device__ __forceinline__ void row_visit(const RowView<T>& v, F f) {
  constexpr int VEC = RowView<T>::VEC, AHEAD = 4;
#pragma unroll 1
  for (int b0 = threadIdx.x; b0 < v.blocks; b0 += AHEAD * kRowThreads) {
    uint32_t k[AHEAD][VEC];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) v.keys(b0 + j * kRowThreads, k[j]);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (k[j][e]) f(v.first(b0 + j * kRowThreads) + e, k[j][e]);
  }
}

// Finds, among the candidates with key >= floor_key in descending order of key, the key whose
// entries hold position `target` of the running measure: the measure (MASS: the sum of weights;
// otherwise the count) of all larger keys is `before` <= target < before + its own; 1, less than any
// candidate's key, if target is not below the total (a mass summed over slices can exceed it by its
// rounding). Every thread gets the result.
template <typename T, bool MASS>
__device__ __noinline__ uint32_t row_radix_select(const RowView<T> v, uint32_t floor_key, uint64_t target,
                                                  const RowWeigher weight, uint64_t& before) {
  RowScratch& sh = row_scratch();
  constexpr int BITS = RowKey<T>::BITS;
  uint32_t prefix = 0;
  int shift = BITS;
  before = 0;
  uint32_t* counts = sh.counts;
  while (shift > 0) {
    const int width = shift < 11 ? shift : 11;
    const int next = shift - width;
    const uint32_t mask = (1u << width) - 1u;
    for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) {
      if constexpr (MASS) sh.hist[i] = 0;
      else counts[i] = 0;
    }
    if (threadIdx.x == 0) sh.found[0] = ~0ull;
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
    uint64_t run = before + block_exclusive_u64(own, total);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (run <= target && target < run + h[j]) {
        sh.found[0] = kRowBins - 1 - (threadIdx.x * PER + j);
        sh.found[1] = run;
      }
      run += h[j];
    }
    __syncthreads();
    const uint64_t bin = sh.found[0];
    if (bin == ~0ull) return 1u;
    prefix = (prefix << width) | static_cast<uint32_t>(bin);
    before = sh.found[1];
    shift = next;
    __syncthreads();  // found is read before the next level clears it
  }
  return prefix;
}

// Steps of 32 blocks (512 bytes) that a warp goes through in index order: warp w has the steps from
// w * row_warp_steps on.
__device__ __forceinline__ int row_warp_steps(int blocks) { return ((blocks + 31) / 32 + kRowWarps - 1) / kRowWarps; }

// f(block, keys of this lane's block) for each step, by every lane of the warp, until f returns false
// (the same in every lane); keys of 0 past the end. The next step's load is ahead of the one in hand.
template <typename T, typename F>
__device__ __forceinline__ void row_key_walk(const RowView<T>& v, F f) {
  constexpr int VEC = RowView<T>::VEC;
  const int lane = threadIdx.x & 31, per = row_warp_steps(v.blocks);
  const int s0 = static_cast<int>(threadIdx.x >> 5) * per, s1 = min((v.blocks + 31) / 32, s0 + per);
  uint32_t k[VEC], next[VEC];
  if (s0 < s1) v.keys(s0 * 32 + lane, k);
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    const int b = s * 32 + lane;
    v.keys(s + 1 < s1 ? b + 32 : v.blocks, next);
    __syncwarp();
    if (!f(b, k)) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e) k[e] = next[e];
  }
}

// ------------------------------------------------------------------------------------------------
// Top-k
// ------------------------------------------------------------------------------------------------

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 4)
    topk_rows_kernel(const T* __restrict__ x, int64_t ldx, int V, int k, float temperature, RowScan scan,
                     float* __restrict__ values, int64_t* __restrict__ ids, float* __restrict__ lse) {
  using K = RowKey<T>;
  RowScratch& sh = row_scratch();
  griddep_wait();  // launched as a programmatic dependent of the scan
  const int64_t row = blockIdx.x;
  const RowView<T> v(x + row * ldx, V);
  const uint32_t top_key = row_open(scan, row);
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
    const uint32_t bound = row_bound(scan.groups, k, top_key);
    int n = row_gather<T>(v.p, V, scan.groups, bound);
    kk = min(n, k);
    if (n > kRowList) {
      // the kk-th largest key, then the larger ones and of its equals the first in index order
      uint64_t n_gt;
      const RowWeigher none{RowWeight{}};
      const uint32_t cut = row_radix_select<T, false>(v, 1u, kk - 1, none, n_gt);
      uint32_t eq = 0;
      row_key_walk<T>(v, [&](int, const uint32_t(&key)[RowView<T>::VEC]) {
#pragma unroll
        for (int e = 0; e < RowView<T>::VEC; ++e) eq += key[e] == cut;
        return true;
      });
      // equals of the warps before this one
      uint64_t total;
      uint64_t rank = block_exclusive_u64(eq, total);
      rank = __shfl_sync(0xffffffffu, rank, 0);
      const uint64_t room = kk - n_gt;
      const int lane = threadIdx.x & 31;
      row_key_walk<T>(v, [&](int b, const uint32_t(&key)[RowView<T>::VEC]) {
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
    row_order(n);
  }
  for (int i = threadIdx.x; i < k; i += kRowThreads) {
    const uint64_t e = i < kk ? sh.sorted[i] : 0;
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
__device__ __noinline__ bool row_pick_listed(int n, int V, int top_k, float top_p, uint64_t mass, uint64_t least,
                                             float uniform, const RowWeigher weight, int64_t* __restrict__ token) {
  RowScratch& sh = row_scratch();
  using K = RowKey<T>;
  constexpr int PER = kRowList / kRowThreads;
  uint64_t w[PER], own = 0, total;
  if (mass) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (threadIdx.x + j * kRowThreads < n)
        own += weight(K::value(static_cast<uint32_t>(sh.list[threadIdx.x + j * kRowThreads] >> 32)));
    own = block_sum_u64(own);
    if (floor_share(top_p, mass) >= own) return false;
    own = 0;
  }
  // only top-k and top-p ask for the order
  const bool order = top_k || top_p < 1.f;
  if (order) row_order(n);
  const uint64_t* entries = order ? sh.sorted : sh.list;
  const uint32_t kth = top_k ? static_cast<uint32_t>(entries[top_k - 1] >> 32) : 0u;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int at = threadIdx.x * PER + j;
    const uint32_t key = at < n ? static_cast<uint32_t>(entries[at] >> 32) : 0u;
    w[j] = at < n && key >= kth ? weight(K::value(key)) : 0;
    own += w[j];
  }
  uint64_t before = block_exclusive_u64(own, total);
  const uint64_t target = top_p < 1.f ? floor_share(top_p, mass ? mass : total) : ~0ull;
  own = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint64_t keep = before <= target && w[j] >= least ? w[j] : 0;
    before += w[j];
    own += w[j] = keep;
  }
  const uint64_t aim = floor_share(uniform, block_sum_u64(own));
  // the token: the lowest index up to which the kept entries weigh more than `aim`
  // Up to 256 entries: the running sum before each, over all pairs (16 rows of V = 151936, us: top-k 60 20.5,
  // by bisection 31; top-k 200 35 and 39; top-k 400 71 and 47).
  if (n <= kRowThreads) {
    uint64_t* kept = order ? sh.list : sh.sorted;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (threadIdx.x * PER + j < n) kept[threadIdx.x * PER + j] = w[j];
    __syncthreads();
    const int parts = n <= kRowThreads / 2 ? 2 : 1;  // threads an entry
    const int e = min(static_cast<int>(threadIdx.x) / parts, n - 1);
    const uint32_t place = static_cast<uint32_t>(entries[e]);
    uint64_t run = 0;
    for (int j = threadIdx.x % parts; j < n; j += parts) run += static_cast<uint32_t>(entries[j]) > place ? kept[j] : 0;
    if (parts == 2) run += __shfl_xor_sync(0xffffffffu, run, 1);
    if (run <= aim && aim < run + kept[e]) *token = ~place;
    return true;
  }
  uint32_t place[PER];  // more: by bisection
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int at = threadIdx.x * PER + j;
    place[j] = at < n ? ~static_cast<uint32_t>(entries[at]) : 0xFFFFFFFFu;
  }
  uint32_t lo = 0, hi = V - 1;
#pragma unroll 1
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    own = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) own += place[j] <= mid ? w[j] : 0;
    if (block_sum_u64(own) > aim) hi = mid;
    else lo = mid + 1;
  }
  if (threadIdx.x == 0) *token = lo;
  return true;
}

// A slice's weight at the row's maximum: as it is where the slice holds that maximum, else brought down.
__device__ __forceinline__ uint64_t row_slice_mass(const RowSlice& a, uint32_t top_key, float slice_top,
                                                   const RowWeigher& weight, float temperature) {
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

// A value that the border of a row's nucleus does not lie below. `mass` is the weight of all candidates,
// `target` top-p's share of it. Entries that weigh at most (mass - target - 1) / V together weigh less than
// mass - target, so the border lies above them; weights are rounded, so one of light + 1 stands for
// light + 1/2 or more. The margin covers the fp32 arithmetic.
__device__ __forceinline__ float row_border_floor(int V, float temperature, uint64_t mass, uint64_t target, float top,
                                                  int S) {
  const uint64_t light = (mass - target - 1) / static_cast<uint64_t>(V);
  const float depth = (static_cast<float>(S) - log2f(static_cast<float>(light) + 0.5f)) * kLn2 + 1e-3f;
  return fmaxf(top - depth * temperature - 1e-5f * fabsf(top), -3.4e38f);
}

// Picks the token by going over the row in index order: kept are the entries above `cut` and the first
// `ties` equal to it, as far as they weigh `least`; no entry below the key `lowest` does.
template <typename T>
__device__ void row_pick_walk(const RowView<T>& v, uint32_t cut, uint64_t ties, uint32_t lowest, uint64_t least,
                              float uniform, const RowWeigher& weight, int64_t* __restrict__ token) {
  using K = RowKey<T>;
  constexpr int VEC = RowView<T>::VEC;
  const int lane = threadIdx.x & 31;
  const uint64_t cut_weight = weight(K::value(cut));
  if (cut_weight < least) ties = 0;
  auto above = [&](uint32_t key) -> uint64_t {
    if (key <= cut || key < lowest) return 0;
    const uint64_t w = weight(K::value(key));
    return w >= least ? w : 0;
  };
  uint64_t sum = 0;
  uint32_t eq = 0;
  row_key_walk<T>(v, [&](int, const uint32_t(&key)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sum += above(key[e]);
      eq += key[e] == cut;
    }
    return true;
  });
  // of each warp's range: its equals inside, its weight, the weight before it
  uint64_t all;
  uint64_t rank = __shfl_sync(0xffffffffu, block_exclusive_u64(eq, all), 0);
  const uint64_t equals = __reduce_add_sync(0xffffffffu, eq);
  const uint64_t inside = rank < ties ? min(ties - rank, equals) : 0;
  sum = warp_sum_u64(sum) + inside * cut_weight;
  uint64_t run = __shfl_sync(0xffffffffu, block_exclusive_u64(lane == 0 ? sum : 0, all), 0);
  const uint64_t aim = floor_share(uniform, all);
  if (run > aim || aim >= run + sum) return;
  row_key_walk<T>(v, [&](int b, const uint32_t(&key)[VEC]) {
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

// A slice's values staged in the list's and the histogram's memory, a thread's blocks neighbours. What
// goes over them are loops that stay loops: unrolled code would run once, at the speed of its
// instructions' fetches.
template <typename T, int BLOCKS>
struct RowStage {
  static constexpr int VEC = RowView<T>::VEC, SLICE = BLOCKS * kScanThreads;
  static constexpr int PER = SLICE > kRowThreads ? SLICE / kRowThreads : 1;  // blocks of a thread
  static constexpr int ENTRIES = PER * VEC;
  static_assert(SLICE * 16 <= static_cast<int>(sizeof(RowScratch::list) + sizeof(RowScratch::hist)) &&
                (PER & (PER - 1)) == 0 && ENTRIES <= 32 && SLICE % kRowThreads == 0, "");
  // block j of a thread; the exchange keeps a warp's 16-byte accesses off one another's banks
  __device__ static __forceinline__ uint4* place(int thread, int j) {
    RowScratch& sh = row_scratch();
    const int at = thread * PER + (j ^ (thread % PER));
    return at < kRowList / 2 ? reinterpret_cast<uint4*>(sh.list) + at : reinterpret_cast<uint4*>(sh.hist) + at - kRowList / 2;
  }
  __device__ static __forceinline__ void fill(const RowView<T>& v, int b0) {
#pragma unroll 4
    for (int j = 0; j < PER; ++j) *place(threadIdx.x, j) = v.raw(b0 + static_cast<int>(threadIdx.x) * PER + j);
  }
  __device__ static __forceinline__ float value(int thread, int e) {
    return fmaxf(static_cast<float>(reinterpret_cast<const T*>(place(thread, e / VEC))[e % VEC]), -INFINITY);
  }
  // The index of the entry in which `aim` falls, given each thread's sum of weights w(thread, e); -1 where aim
  // is not below their total. For the lanes of warp 0; the others get -1.
  template <typename W>
  __device__ static __forceinline__ int find(const RowView<T>& v, int b0, uint64_t sum, uint64_t aim, W w) {
    RowScratch& sh = row_scratch();
    const int lane = threadIdx.x & 31;
    uint64_t total;
    const uint64_t at = block_exclusive_u64(sum, total);
    if (at <= aim && aim < at + sum) {
      sh.found[0] = threadIdx.x;
      sh.found[1] = aim - at;
    }
    __syncthreads();
    if (threadIdx.x >= 32 || aim >= total) return -1;
    const int owner = static_cast<int>(sh.found[0]);  // its entries, one a lane
    const uint64_t rest = sh.found[1], own = lane < ENTRIES ? w(owner, lane) : 0;
    uint64_t inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const uint32_t who = __ballot_sync(0xffffffffu, inc - own <= rest && rest < inc);
    return v.first(b0 + owner * PER) + __ffs(who) - 1;
  }
};

// Picks the token of an unfiltered row from the slices' weights: the slice that holds the uniform's
// share, and in it the entry, by the slice's own weights.
template <typename T, int BLOCKS>
__device__ void row_pick_slice(const RowView<T>& v, const RowScan& scan, int64_t row, uint32_t top_key,
                               float temperature, float uniform, const RowWeigher& weight,
                               int64_t* __restrict__ token) {
  RowScratch& sh = row_scratch();
  using K = RowKey<T>;
  using View = RowView<T>;
  constexpr int VEC = View::VEC, SLICE = BLOCKS * kScanThreads;
  RowSlice a{0u, 0u, 0ull};
  uint64_t own = 0, total;
  if (static_cast<int>(threadIdx.x) < scan.slices) {
    a = scan.slice[row * scan.slices + threadIdx.x];
    own = row_slice_mass(a, top_key, K::value(a.top), weight, temperature);
  }
  const uint64_t run = block_exclusive_u64(own, total);
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
  const RowWeigher local{row_weight(K::value(static_cast<uint32_t>(sh.found[0] >> 32)), temperature, weight.S)};
  const int b0 = static_cast<int>(sh.found[0] & 0xFFFFFFFFu) * SLICE;
  aim = sh.found[1];
  __syncthreads();  // found is read
  using Stage = RowStage<T, BLOCKS>;
  Stage::fill(v, b0);
  const RowWeight inline_local{local.top, local.floor, local.S, local.from, local.scale};
  uint64_t sum = 0;
#pragma unroll 1
  for (int j = 0; j < Stage::PER; ++j) {
    float x[VEC];
    View::values_of(*Stage::place(threadIdx.x, j), x);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum += inline_local(x[e]);
  }
  const int i = Stage::find(v, b0, sum, aim, [&](int thread, int e) { return local(Stage::value(thread, e)); });
  if (threadIdx.x == 0 && i >= 0) *token = i;
}

template <typename T, int BLOCKS>
__global__ void __launch_bounds__(kRowThreads, 4)
    sample_logits_kernel(const T* __restrict__ x, int64_t ldx, int V, int S, const float* __restrict__ uniform,
                         SampleKnobs knobs, RowScan scan, RowWideRows wide, int64_t* __restrict__ tokens) {
  using K = RowKey<T>;
  constexpr int LANES = kRowGroup / RowView<T>::VEC;
  RowScratch& sh = row_scratch();
  const int64_t row = blockIdx.x;
  const RowView<T> v(x + row * ldx, V);
  griddep_launch_dependents();
  griddep_wait();  // launched as a programmatic dependent of the scan
  const SampleRow knob(knobs, row);
  const float u = uniform[row], T_ = knob.temperature;
  const uint32_t top_key = row_open(scan, row);
  if (top_key == 0) {
    if (threadIdx.x == 0) tokens[row] = -1;
    return;
  }
  if (knob.greedy) {  // the first group with the largest key, its first entry
    uint32_t g = 0xFFFFFFFFu;
    for (int i = threadIdx.x; i < scan.groups; i += kRowThreads)
      if (row_maxima()[i] == top_key) g = min(g, static_cast<uint32_t>(i));
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
  const RowWeigher weight{row_weight(K::value(top_key), T_, S)};
  // min-p: weights below `least` leave; no entry below the key `lowest` passes (lower by a margin that
  // covers fp32)
  const float floor_p = fminf(fmaxf(knob.min_p, 0.f), 1.f);
  const uint64_t least = row_least(floor_p, S);
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
    filtered = static_cast<uint64_t>(knob.top_k) < block_sum_u64(candidates);
  } else if (knob.top_k >= 1) {
    const uint32_t bound = row_bound(scan.groups, knob.top_k, top_key);
    const int n = row_gather<T>(v.p, V, scan.groups, bound);
    if (n <= kRowList) {  // with fewer than top_k entries, all there are
      row_pick_listed<T>(n, V, min(n, knob.top_k), knob.top_p, 0, least, u, weight, tokens + row);
      return;
    }
    filtered = true;
  }
  // the row's number among the wide rows, or -1: no room
  auto enlist = [&](float lo, float hi, uint64_t target, bool nucleus) {
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t slot = wide.count ? atomicAdd(wide.count, 1u) : 0xFFFFFFFFu;
      if (slot < static_cast<uint32_t>(wide.most)) {
        RowWideRow& r = wide.rows[slot];
        r.row = row;
        r.top = weight.top;
        r.lo = lo;
        r.hi = hi;
        r.target = target;
        r.nucleus = nucleus;
      }
      sh.found[0] = slot;
    }
    __syncthreads();
    if (sh.found[0] >= static_cast<uint64_t>(wide.most)) return false;
    for (int i = threadIdx.x; i < kRowWideBins; i += kRowThreads) wide.rows[sh.found[0]].bins[i] = 0;
    return true;
  };
  uint32_t cut = 1u;
  uint64_t before, ties = ~0ull;
  if (filtered) cut = row_radix_select<T, false>(v, 1u, knob.top_k - 1, weight, before);
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
    mass = block_sum_u64(mass);
    const uint64_t target = floor_share(knob.top_p, mass);
    if (!filtered) {
      // the head of the order first: most nuclei are a few hundred entries at most
      const uint32_t bound = row_bound(scan.groups, kRowHead, top_key);
      const int n = row_gather<T>(v.p, V, scan.groups, bound);
      if (n <= kRowList) {
        const bool whole_row = n < kRowHead || bound == 1u;
        if (row_pick_listed<T>(n, V, 0, knob.top_p, whole_row ? 0 : mass, least, u, weight, tokens + row)) return;
        if (weight.top < INFINITY &&
            enlist(row_border_floor(V, T_, mass, target, weight.top, S), INFINITY, target, true))
          return;
      }
      __syncthreads();
    }
    cut = row_radix_select<T, true>(v, cut, target, weight, before);
    ties = cut > 1u ? (target - before) / weight(K::value(cut)) + 1 : ~0ull;
  } else if (!filtered && floor_p > 0.f) {
    const int n = row_gather<T>(v.p, V, scan.groups, lowest);
    if (n <= kRowList) {
      row_pick_listed<T>(n, V, 0, 1.f, 0, least, u, weight, tokens + row);
      return;
    }
    if (weight.top < INFINITY && enlist(K::value(lowest), K::value(lowest), 0, false)) return;
  } else if (!filtered && knob.wants_mass()) {
    row_pick_slice<T, BLOCKS>(v, scan, row, top_key, T_, u, weight, tokens + row);
    return;
  }
  row_pick_walk<T>(v, cut, ties, lowest, least, u, weight, tokens + row);
}

// ------------------------------------------------------------------------------------------------
// Wide rows
// ------------------------------------------------------------------------------------------------

// f(index, value, live) for the entries at or above `lo` of a slice, 32 at a time by a whole warp: a warp
// queues its entries, so that the few that matter do not each cost a warp's arithmetic.
template <typename T, int BLOCKS, typename F>
__device__ __forceinline__ void row_slice_entries(const RowView<T>& v, int b0, float lo, uint2* queue, F f) {
  constexpr int VEC = RowView<T>::VEC;
  const int lane = threadIdx.x & 31;
  const uint32_t below = (1u << lane) - 1u;
  int queued = 0;
#pragma unroll 1
  for (int j = 0; j < BLOCKS; ++j) {
    const int b = b0 + j * kScanThreads + static_cast<int>(threadIdx.x);
    float xs[VEC];
    v.values(b, xs);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const uint32_t who = __ballot_sync(0xffffffffu, xs[e] >= lo);
      if (xs[e] >= lo) queue[queued + __popc(who & below)] = make_uint2(v.first(b) + e, __float_as_uint(xs[e]));
      queued += __popc(who);
    }
    __syncwarp();
#pragma unroll 1
    while (queued >= 32) {
      queued -= 32;
      const uint2 e = queue[queued + lane];
      f(e.x, __uint_as_float(e.y), true);
      __syncwarp();
    }
  }
  if (queued) {
    const uint2 e = queue[lane];
    f(e.x, __uint_as_float(e.y), lane < queued);
  }
}

// Persistent over the slices of the wide rows with a nucleus: the weights from the maximum down to lo, in
// bins even in x. They only say where to look for the border, so fp32 does: an entry counts as
// 2^18 times its weight over that of its bin's upper end, which keeps a slice's 8192 entries in 32
// bits (whose shared-memory atomics cost a fifth of those on 64).
template <typename T, int BLOCKS>
__global__ void __launch_bounds__(kScanThreads)
    row_wide_bins_kernel(const T* __restrict__ x, int64_t ldx, int V, SampleKnobs knobs, int slices, RowWideRows wide) {
  constexpr int VEC = RowView<T>::VEC;
  static_assert(BLOCKS * kScanThreads * VEC <= 8192, "a slice's sums exceed 32 bits");
  __shared__ uint32_t bins[kRowWideBins];
  griddep_launch_dependents();
  griddep_wait();
  const int64_t units = static_cast<int64_t>(min(*wide.count, static_cast<uint32_t>(wide.most))) * slices;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    RowWideRow& r = wide.rows[unit / slices];
    if (!r.nucleus) continue;
    for (int i = threadIdx.x; i < kRowWideBins; i += kScanThreads) bins[i] = 0;
    __syncthreads();
    const RowView<T> v(x + r.row * ldx, V);
    const float top = r.top, lo = r.lo, inv = r.per_value();
    const float bits = kLog2e / SampleRow(knobs, r.row).temperature / inv;  // of a bin
    const int b0 = static_cast<int>(unit % slices) * BLOCKS * kScanThreads;
#pragma unroll 1
    for (int j = 0; j < BLOCKS; ++j) {
      float xs[VEC];
      v.values(b0 + j * kScanThreads + static_cast<int>(threadIdx.x), xs);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = (top - xs[e]) * inv;
        const int b = min(kRowWideBins - 1, static_cast<int>(d));
        const uint32_t w = __float2uint_rn(ex2_approx(18.f - (d - static_cast<float>(b)) * bits));
        if (xs[e] >= lo) atomicAdd(&bins[b], w);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRowWideBins; i += kScanThreads)
      if (bins[i]) atomicAdd(reinterpret_cast<unsigned long long*>(&r.bins[i]), static_cast<unsigned long long>(bins[i]));
    __syncthreads();
  }
}

// One warp per wide row: the window becomes the bin that holds the border, a little wider than the fp32
// arithmetic needs, with the next bin where the border lies close to it. (Bins are off by 512 roundings
// of a bin's part of at most 2^-3 bits, the sums that run over them by less than 2^-15 of themselves.)
__global__ void __launch_bounds__(256) row_wide_window_kernel(int S, SampleKnobs knobs, RowWideRows wide) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t count = min(*wide.count, static_cast<uint32_t>(wide.most));
  for (uint32_t slot = blockIdx.x * 8 + (threadIdx.x >> 5); slot < count; slot += gridDim.x * 8) {
    RowWideRow& r = wide.rows[slot];
    if (!r.nucleus) continue;
    constexpr int PER = kRowWideBins / 32;
    const float lo = r.lo, inv = r.per_value();
    const float bits = kLog2e / SampleRow(knobs, r.row).temperature / inv;
    const double unit = static_cast<double>(1ull << (S - 18));
    double h[PER], sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      h[j] = static_cast<double>(r.bins[lane * PER + j]) * unit * exp2f(-bits * static_cast<float>(lane * PER + j));
      sum += h[j];
    }
    double run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += u;
    }
    run -= sum;
    const double target = static_cast<double>(r.target), near = target * 0x1p-15;
    int first = kRowWideBins, last = -1;  // bins that may hold the border
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (h[j] > 0.0 && run - near <= target && target <= run + h[j] + near) {
        first = min(first, lane * PER + j);
        last = lane * PER + j;
      }
      run += h[j];
    }
    first = __reduce_min_sync(0xffffffffu, first);
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0 && last >= 0) {
      const float slack = 1e-6f * (fabsf(r.top) + (r.top - lo));
      r.hi = first == 0 ? INFINITY : r.top - static_cast<float>(first) / inv + slack;
      r.lo = last == kRowWideBins - 1 ? lo : fmaxf(lo, r.top - static_cast<float>(last + 1) / inv - slack);
    }
    __syncwarp();
  }
}

// Persistent over the slices of the wide rows: per slice the weight of the entries above the window, all
// of them and those that pass min-p, and the window's entries.
template <typename T, int BLOCKS>
__global__ void __launch_bounds__(kScanThreads)
    row_wide_kernel(const T* __restrict__ x, int64_t ldx, int V, int S, SampleKnobs knobs, int slices,
                    RowWideRows wide) {
  using K = RowKey<T>;
  constexpr int WARPS = kScanThreads / 32;
  __shared__ uint2 queues[WARPS][32 * (RowView<T>::VEC + 1)];  // (index, value)
  __shared__ uint64_t wabove[WARPS], wkept[WARPS];
  __shared__ uint32_t listed;
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t below = (1u << lane) - 1u;
  const int64_t units = static_cast<int64_t>(min(*wide.count, static_cast<uint32_t>(wide.most))) * slices;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const RowWideRow& r = wide.rows[unit / slices];
    uint64_t* const list = wide.lists + unit * wide.room;
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    const float hi = r.hi;
    const RowView<T> v(x + r.row * ldx, V);
    const SampleRow knob(knobs, r.row);
    const RowWeight weight = row_weight(r.top, knob.temperature, S);
    const uint64_t least = row_least(knob.min_p, S);
    uint64_t above = 0, kept = 0;
    row_slice_entries<T, BLOCKS>(
        v, static_cast<int>(unit % slices) * BLOCKS * kScanThreads, r.lo, queues[warp], [&](uint32_t i, float xe, bool live) {
          const bool inside = live && !(xe >= hi);
          if (live && !inside) {
            const uint64_t w = weight(xe);
            above += w;
            kept += w >= least ? w : 0;
          }
          const uint32_t who = __ballot_sync(0xffffffffu, inside);
          if (who == 0) return;
          uint32_t at = 0;
          if (lane == 0) at = atomicAdd(&listed, static_cast<uint32_t>(__popc(who)));
          at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & below);
          if (inside && at < static_cast<uint32_t>(wide.room)) list[at] = (static_cast<uint64_t>(K::of(xe)) << 32) | ~i;
        });
    above = warp_sum_u64(above);
    kept = warp_sum_u64(kept);
    if (lane == 0) {
      wabove[warp] = above;
      wkept[warp] = kept;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      RowSums s{0, 0, listed};
      for (int w = 0; w < WARPS; ++w) {
        s.above += wabove[w];
        s.kept += wkept[w];
      }
      wide.sums[unit] = s;
    }
    __syncthreads();
  }
}

// Per slice, after the scratch: its kept weight and the entries that it listed.
struct RowWideSlices {
  uint64_t kept[kRowThreads];
  uint32_t listed[kRowThreads];
};

// One CTA per wide row at a time: the border among the window's entries, the slice that holds the
// uniform's share of the kept weight, and in it the entry.
template <typename T, int BLOCKS>
__global__ void __launch_bounds__(kRowThreads, 4)
    row_wide_pick_kernel(const T* __restrict__ x, int64_t ldx, int V, int S, const float* __restrict__ uniform,
                         SampleKnobs knobs, int slices, RowWideRows wide, int64_t* __restrict__ tokens) {
  using K = RowKey<T>;
  constexpr int VEC = RowView<T>::VEC, SLICE = BLOCKS * kScanThreads;
  RowScratch& sh = row_scratch();
  RowWideSlices& win = *reinterpret_cast<RowWideSlices*>(row_smem + (sizeof(RowScratch) + 15) / 16 * 16);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  griddep_wait();
  const uint32_t count = min(*wide.count, static_cast<uint32_t>(wide.most));
  for (uint32_t slot = blockIdx.x; slot < count; slot += gridDim.x) {
    __syncthreads();
    const RowWideRow& r = wide.rows[slot];
    const RowView<T> v(x + r.row * ldx, V);
    const SampleRow knob(knobs, r.row);
    const RowWeigher weight{row_weight(r.top, knob.temperature, S)};
    const uint64_t least = row_least(knob.min_p, S);
    const float u = uniform[r.row], lo = r.lo;
    const uint64_t border_at = r.target;
    uint64_t total;
    RowSums own{0, 0, 0};
    if (static_cast<int>(threadIdx.x) < slices) own = wide.sums[static_cast<int64_t>(slot) * slices + threadIdx.x];
    win.kept[threadIdx.x] = own.kept;
    win.listed[threadIdx.x] = own.listed;
    if (threadIdx.x == 0) {
      sh.listed = 0;
      sh.found[0] = ~0ull;
    }
    for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) sh.hist[i] = 0;
    uint64_t border = 0;  // of the kept entries the last in the order; 0: all are kept
    // f(entry or 0) for the listed entries of the warp's slices, 32 at a time; then g(slice)
    auto each = [&](auto f, auto g) {
      for (int s = warp; s < slices; s += kRowWarps) {
        const uint64_t* list = wide.lists + (static_cast<int64_t>(slot) * slices + s) * wide.room;
        const int n = static_cast<int>(win.listed[s]);
#pragma unroll 1
        for (int i = lane; i - lane < n; i += 128) {  // four loads at a time
          uint64_t e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) e[j] = i + 32 * j < n ? list[i + 32 * j] : 0ull;
#pragma unroll
          for (int j = 0; j < 4; ++j) f(e[j]);
        }
        g(s);
      }
    };
    if (r.nucleus) {
      const uint64_t above = block_sum_u64(own.above);
      bool ok = !__syncthreads_or(own.listed > static_cast<uint32_t>(wide.room)) && above <= border_at;
      if (ok) {
        // weights in 2048 bins even in x, the bin that holds the target, its entries in order
        const float xhi = fminf(r.hi, r.top), inv = static_cast<float>(kRowBins) / fmaxf(xhi - lo, 1e-30f);
        auto bin = [&](float x) { return min(kRowBins - 1, max(0, static_cast<int>((xhi - x) * inv))); };
        each(
            [&](uint64_t e) {
              if (e == 0) return;
              const float x = K::value(static_cast<uint32_t>(e >> 32));
              atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[bin(x)]), static_cast<unsigned long long>(weight(x)));
            },
            [](int) {});
        __syncthreads();
        constexpr int BINS = kRowBins / kRowThreads;
        uint64_t h[BINS], sum = 0;
#pragma unroll
        for (int j = 0; j < BINS; ++j) sum += h[j] = sh.hist[threadIdx.x * BINS + j];
        uint64_t run = above + block_exclusive_u64(sum, total);
#pragma unroll
        for (int j = 0; j < BINS; ++j) {
          if (run <= border_at && border_at < run + h[j]) {
            sh.found[0] = threadIdx.x * BINS + j;
            sh.found[1] = run;
          }
          run += h[j];
        }
        __syncthreads();
        ok = sh.found[0] != ~0ull;
        if (ok) {
          const int at = static_cast<int>(sh.found[0]);
          const uint64_t before = sh.found[1];
          each(
              [&](uint64_t e) {
                row_append(e && bin(K::value(static_cast<uint32_t>(e >> 32))) == at, e, sh.list, &sh.listed);
              },
              [](int) {});
          __syncthreads();
          const int m = static_cast<int>(min(sh.listed, static_cast<uint32_t>(kRowList) + 1u));
          ok = m <= kRowList;
          if (ok) {
            row_order(m);
            constexpr int PER = kRowList / kRowThreads;
            uint64_t w[PER], mine = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
              const int k = threadIdx.x * PER + j;
              w[j] = k < m ? weight(K::value(static_cast<uint32_t>(sh.sorted[k] >> 32))) : 0;
              mine += w[j];
            }
            run = before + block_exclusive_u64(mine, total);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
              if (run <= border_at && border_at < run + w[j]) sh.found[0] = sh.sorted[threadIdx.x * PER + j];
              run += w[j];
            }
            __syncthreads();
            border = sh.found[0];
          }
        }
      }
      if (!ok) {  // the border is not in the window, or the window holds too much: the whole row
        __syncthreads();
        uint64_t before;
        const uint32_t cut = row_radix_select<T, true>(v, 1u, border_at, weight, before);
        const uint64_t ties = cut > 1u ? (border_at - before) / weight(K::value(cut)) + 1 : ~0ull;
        row_pick_walk<T>(v, cut, ties, 1u, least, u, weight, tokens + r.row);
        continue;
      }
      // the kept entries of the window join their slices
      uint64_t sum = 0;
      each(
          [&](uint64_t e) {
            if (e < border || e == 0) return;
            const uint64_t w = weight(K::value(static_cast<uint32_t>(e >> 32)));
            sum += w >= least ? w : 0;
          },
          [&](int s) {
            sum = warp_sum_u64(sum);
            if (lane == 0) win.kept[s] += sum;
            sum = 0;
          });
    }
    __syncthreads();
    const uint64_t mine = win.kept[threadIdx.x];
    uint64_t run = block_exclusive_u64(mine, total);
    const uint64_t aim = floor_share(u, total);
    if (run <= aim && aim < run + mine) {
      sh.found[0] = threadIdx.x;
      sh.found[1] = aim - run;
    }
    __syncthreads();
    const int b0 = static_cast<int>(sh.found[0]) * SLICE;
    const uint64_t rest = sh.found[1];
    __syncthreads();
    using Stage = RowStage<T, BLOCKS>;
    Stage::fill(v, b0);
    uint32_t some = 0;  // the thread's entries at or above lo
#pragma unroll 1
    for (int j = 0; j < Stage::PER; ++j) {
      float xs[VEC];
      RowView<T>::values_of(*Stage::place(threadIdx.x, j), xs);
#pragma unroll
      for (int e = 0; e < VEC; ++e) some |= static_cast<uint32_t>(xs[e] >= lo) << (j * VEC + e);
    }
    auto kept = [&](int thread, int e) -> uint64_t {  // weight of a thread's e-th entry if it is kept
      const float xe = Stage::value(thread, e);
      const uint32_t i = v.first(b0 + thread * Stage::PER) + e;
      if (!(xe >= lo) || ((static_cast<uint64_t>(K::of(xe)) << 32) | ~i) < border) return 0;
      const uint64_t w = weight(xe);
      return w >= least ? w : 0;
    };
    uint64_t sum = 0;
#pragma unroll 1
    for (; some; some &= some - 1) sum += kept(threadIdx.x, __ffs(some) - 1);
    const int i = Stage::find(v, b0, sum, rest, kept);
    if (threadIdx.x == 0) tokens[r.row] = i;
  }
}

// ------------------------------------------------------------------------------------------------
// Launch
// ------------------------------------------------------------------------------------------------

struct RowPlan {
  int groups, slices, blocks;  // blocks: 16-byte blocks of a scan thread
  int wide, room;              // most wide rows; entries a slice of one may list
  size_t off_slice, off_count, off_rows, off_sums, off_lists, total;
};

// Slices of 8192 entries, 32 a thread in flight, or of 2048 where those would leave SMs idle. (Top-64 of V =
// 151936 fp32, us with slices of 8192 / 2048: 1 row 13.3 / 12.3, 16 rows 16.5 / 16.5, 64 rows 20.7 /
// 22.8.) Sampling weighs each entry in fp64, which small slices spread better, and the finish weighs one
// slice again: without filters that need more, 2048 up to some 120 such rows (1 row 16.5 / 10.3, 64 rows
// 41.2 / 34.9, 128 rows 57.9 / 55.4, 256 rows 94.3 / 100.4); wide rows cost launches' work per slice
// (top-p 0.95, 64 rows: 124 / 139, 256 rows: 251 / 324). `aligned`: every row starts on a 16-byte
// boundary. `wide`: rows can turn out wide.
inline RowPlan row_plan(int64_t R, int64_t V, int elem, bool aligned, bool sample, bool wide) {
  RowPlan p{};
  const int vec = 16 / elem;
  p.groups = static_cast<int>(ceil_div(V + (aligned ? 0 : vec - 1), 4 * kRowGroup)) * 4;
  const bool small = R * ceil_div(V, 8192) < (sample && !wide ? 16 : 2) * num_sms() && V <= (1 << 18);
  p.blocks = (small ? 2048 : 8192) / vec / kScanThreads;
  p.slices = static_cast<int>(ceil_div(static_cast<int64_t>(p.groups) * kRowGroup, static_cast<int64_t>(p.blocks) * kScanThreads * vec));
  p.wide = wide ? static_cast<int>(std::min<int64_t>(R, kRowWideRows)) : 0;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = (off + bytes + 255) / 256 * 256;
    return o;
  };
  take(static_cast<size_t>(R) * p.groups * 4);
  p.off_slice = take(static_cast<size_t>(R) * p.slices * sizeof(RowSlice));
  p.off_count = take(wide ? 4 : 0);
  p.off_rows = take(static_cast<size_t>(p.wide) * sizeof(RowWideRow));
  p.off_sums = take(static_cast<size_t>(p.wide) * p.slices * sizeof(RowSums));
  p.room = p.blocks * kScanThreads * vec / kRowWideShare;
  p.off_lists = take(static_cast<size_t>(p.wide) * p.slices * p.room * 8);
  p.total = off;
  return p;
}

// Bytes that do for any alignment.
inline size_t row_ws_bytes(int64_t R, int64_t V, int elem, bool sample, bool wide) {
  return std::max(row_plan(R, V, elem, true, sample, wide).total, row_plan(R, V, elem, false, sample, wide).total);
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
inline int row_prepare(const T* x, int64_t ldx, int64_t R, int64_t V, bool sample, bool wide, void* ws, size_t ws_bytes, RowPlan& p,
                       RowScan& scan) {
  p = row_plan(R, V, sizeof(T), aligned16(x) && (ldx * sizeof(T)) % 16 == 0, sample, wide);
  ORTHRUS_CHECK_ARG(R * p.slices < (1ll << 31) && (reinterpret_cast<uintptr_t>(x) & (sizeof(T) - 1)) == 0);
  if (ws == nullptr || ws_bytes < p.total) return ORTHRUS_EWORKSPACE;
  ORTHRUS_CHECK_ARG(aligned16(ws));
  uint8_t* w = static_cast<uint8_t*>(ws);
  scan = {reinterpret_cast<uint32_t*>(w), reinterpret_cast<RowSlice*>(w + p.off_slice), p.groups, p.slices,
          wide ? reinterpret_cast<uint32_t*>(w + p.off_count) : nullptr};
  return ORTHRUS_OK;
}

// Shared memory of a finish: the scratch and the group maxima (kRowSmem: of the longest row); of a pick.
constexpr int kRowScratch = (sizeof(RowScratch) + 15) / 16 * 16;
constexpr int kRowSmem = kRowScratch + (kRowMaxV + 8) / kRowGroup * 4 + 512;
constexpr int kRowWideSmem = kRowScratch + static_cast<int>(sizeof(RowWideSlices));

template <typename T>
int topk_rows_impl(const T* x, int64_t ldx, int64_t R, int64_t V, int k, float temperature, float* values, int64_t* ids,
                   float* lse, void* ws, size_t ws_bytes, cudaStream_t stream) {
  RowPlan p;
  RowScan scan;
  int rc = row_prepare(x, ldx, R, V, false, false, ws, ws_bytes, p, scan);
  if (rc != ORTHRUS_OK) return rc;
  rc = row_scan_launch<T, false>(p, x, ldx, R, static_cast<int>(V), temperature, 0, SampleKnobs{}, scan, stream);
  if (rc != ORTHRUS_OK) return rc;
  ORTHRUS_CHECK_CUDA(ensure_smem(topk_rows_kernel<T>, kRowSmem));
  ORTHRUS_CHECK_CUDA(launch_pdl(topk_rows_kernel<T>, dim3(static_cast<unsigned>(R)), dim3(kRowThreads),
                                kRowScratch + p.groups * 4, stream, x, ldx, static_cast<int>(V), k, temperature, scan, values,
                                ids, lse));
  ORTHRUS_CHECK_LAUNCH();
  return ORTHRUS_OK;
}

// Whether rows can turn out wide: a nucleus or min-p without a top-k that fits a list.
inline bool sample_can_be_wide(const SampleKnobs& k) {
  return (k.top_k || k.top_k1 < 1 || k.top_k1 > kRowMaxK) && (k.top_p || k.top_p1 < 1.f || k.min_p || k.min_p1 > 0.f);
}

template <typename T, int BLOCKS>
int sample_finish_launch(const RowPlan& p, const T* x, int64_t ldx, int64_t R, int V, int S, const float* uniform,
                         const SampleKnobs& knobs, const RowScan& scan, uint8_t* ws, int64_t* tokens,
                         cudaStream_t stream) {
  const RowWideRows wide{scan.wide_count, reinterpret_cast<RowWideRow*>(ws + p.off_rows),
                         reinterpret_cast<RowSums*>(ws + p.off_sums), reinterpret_cast<uint64_t*>(ws + p.off_lists),
                         p.wide, p.room};
  auto finish = sample_logits_kernel<T, BLOCKS>;
  ORTHRUS_CHECK_CUDA(ensure_smem(finish, kRowSmem));
  ORTHRUS_CHECK_CUDA(launch_pdl(finish, dim3(static_cast<unsigned>(R)), dim3(kRowThreads), kRowScratch + p.groups * 4,
                                stream, x, ldx, V, S, uniform, knobs, scan, wide, tokens));
  ORTHRUS_CHECK_LAUNCH();
  if (p.wide == 0) return ORTHRUS_OK;
  const int64_t units = static_cast<int64_t>(p.wide) * p.slices;
  if (knobs.top_p || knobs.top_p1 < 1.f) {
    ORTHRUS_CHECK_CUDA(launch_pdl(row_wide_bins_kernel<T, BLOCKS>,
                                  dim3(static_cast<unsigned>(std::min<int64_t>(units, 8 * num_sms()))), dim3(kScanThreads),
                                  0, stream, x, ldx, V, knobs, p.slices, wide));
    ORTHRUS_CHECK_LAUNCH();
    ORTHRUS_CHECK_CUDA(launch_pdl(row_wide_window_kernel,
                                  dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(p.wide, 8), num_sms()))),
                                  dim3(256), 0, stream, S, knobs, wide));
    ORTHRUS_CHECK_LAUNCH();
  }
  ORTHRUS_CHECK_CUDA(launch_pdl(row_wide_kernel<T, BLOCKS>,
                                dim3(static_cast<unsigned>(std::min<int64_t>(units, 6 * num_sms()))), dim3(kScanThreads), 0,
                                stream, x, ldx, V, S, knobs, p.slices, wide));
  ORTHRUS_CHECK_LAUNCH();
  auto pick = row_wide_pick_kernel<T, BLOCKS>;
  ORTHRUS_CHECK_CUDA(ensure_smem(pick, kRowWideSmem));
  ORTHRUS_CHECK_CUDA(launch_pdl(pick, dim3(static_cast<unsigned>(std::min(p.wide, 4 * num_sms()))), dim3(kRowThreads),
                                kRowWideSmem, stream, x, ldx, V, S, uniform, knobs, p.slices, wide, tokens));
  ORTHRUS_CHECK_LAUNCH();
  return ORTHRUS_OK;
}

template <typename T>
int sample_logits_impl(const T* x, int64_t ldx, int64_t R, int64_t V, const float* uniform, const SampleKnobs& knobs,
                       int64_t* tokens, void* ws, size_t ws_bytes, cudaStream_t stream) {
  RowPlan p;
  RowScan scan;
  int rc = row_prepare(x, ldx, R, V, true, sample_can_be_wide(knobs), ws, ws_bytes, p, scan);
  if (rc != ORTHRUS_OK) return rc;
  const int n = static_cast<int>(V), S = row_weight_bits(n);
  rc = row_scan_launch<T, true>(p, x, ldx, R, n, 1.f, S, knobs, scan, stream);
  if (rc != ORTHRUS_OK) return rc;
  constexpr int BIG = 8192 / RowView<T>::VEC / kScanThreads, SMALL = 2048 / RowView<T>::VEC / kScanThreads;
  uint8_t* w = static_cast<uint8_t*>(ws);
  return p.blocks == BIG ? sample_finish_launch<T, BIG>(p, x, ldx, R, n, S, uniform, knobs, scan, w, tokens, stream)
                         : sample_finish_launch<T, SMALL>(p, x, ldx, R, n, S, uniform, knobs, scan, w, tokens, stream);
}

}  // namespace orthrus
