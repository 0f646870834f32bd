// Row operators over vocabulary logits [R, V]: the k largest entries of a row with its
// log-sum-exp, and sampling from a row's filtered softmax with a given uniform.
//
// One cluster of CS CTAs owns one row. Each CTA reads its contiguous slice of the row once from
// HBM and keeps it in shared memory as order-preserving integer keys (32 bits for fp32, 16 for
// bf16); every later pass runs on shared memory, and the CTAs exchange maxima, sums and histograms
// through distributed shared memory. So the bytes moved are the row itself, whatever the filters
// need.
//
// Candidates are the entries that are neither -inf nor NaN. Entries are ordered by (descending
// value, ascending index); -0 counts as +0.
#pragma once

#include <cuda_bf16.h>

#include "sm100.cuh"

namespace orthrus {

constexpr int kRowThreads = 512;
constexpr int kRowBins = 2048;
constexpr int kRowMaxCluster = 8;  // portable cluster size
constexpr int kRowMaxK = 1024;     // largest k of topk_rows

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
// Cluster and block helpers
// ------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t ld_cluster_u64(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// Cluster barrier of every thread, also after loops whose lanes leave at different iterations.
__device__ __forceinline__ void row_cluster_sync() {
  __syncwarp();
  cluster_sync_all();
}

// The same object's value in CTA `rank` of the cluster.
__device__ __forceinline__ uint64_t peer_u64(const uint64_t* p, uint32_t rank) {
  return ld_cluster_u64(mapa_shared(smem_u32(p), rank));
}
__device__ __forceinline__ uint32_t peer_u32(const uint32_t* p, uint32_t rank) {
  return ld_cluster_u32(mapa_shared(smem_u32(p), rank));
}

struct RowShared {
  uint64_t hist[kRowBins];   // counts (as the low 32-bit words of the first half) or masses
  uint64_t list[kRowMaxK];   // leader: (key << 32 | ~index) of the chosen entries, then sorted
  double exp_tab[64];        // 2^(-j/64)
  uint64_t warp_u64[kRowThreads / 32];
  uint64_t slot[8];          // this CTA's published partials, one use each between barriers
  uint64_t found[2];         // result of a block-wide search
};

__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Block-wide sum; every thread gets it. Leaves warp_u64 free for reuse.
__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, RowShared& sh) {
  v = warp_sum_u64(v);
  if ((threadIdx.x & 31) == 0) sh.warp_u64[threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) t += sh.warp_u64[w];
  __syncthreads();
  return t;
}

__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, RowShared& sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  if ((threadIdx.x & 31) == 0) sh.warp_u64[threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) t = sh.warp_u64[w] > t ? sh.warp_u64[w] : t;
  __syncthreads();
  return t;
}

// Exclusive prefix sum over the block's threads; `total` is the block's sum.
__device__ __forceinline__ uint64_t block_exclusive_u64(uint64_t v, RowShared& sh, uint64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) sh.warp_u64[warp] = inc;
  __syncthreads();
  uint64_t before = 0, t = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) {
    if (w == warp) before = t;
    t += sh.warp_u64[w];
  }
  __syncthreads();
  total = t;
  return before + inc - v;
}

// ------------------------------------------------------------------------------------------------
// The row slice of a CTA
// ------------------------------------------------------------------------------------------------

// Index arithmetic of a slice: `lo` its first index in the row, `n` its entries, `chunk` the
// contiguous entries of one thread in the index-ordered passes (odd, so that neighbouring threads
// read different banks).
struct RowSlice {
  int lo, n, chunk;
  __device__ __forceinline__ RowSlice(int V, int per, uint32_t rank) {
    const int64_t a = static_cast<int64_t>(per) * rank;
    lo = static_cast<int>(a < V ? a : V);
    n = V - lo < per ? V - lo : per;
    chunk = ((n + kRowThreads - 1) / kRowThreads) | 1;
  }
  __device__ __forceinline__ int begin() const { return min(n, static_cast<int>(threadIdx.x) * chunk); }
  __device__ __forceinline__ int end() const { return min(n, (static_cast<int>(threadIdx.x) + 1) * chunk); }
};

// Loads the slice into shared memory as keys. The keys start `off` elements into the buffer so that
// the 16-byte vectors of the (arbitrarily aligned) row land on 16-byte boundaries. Returns the
// thread's largest key and its number of candidates.
template <typename T>
__device__ __forceinline__ int row_stage_offset(const T* p) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
}

template <typename T>
__device__ __forceinline__ void row_stage(const T* __restrict__ p, int n, typename RowKey<T>::type* keys,
                                          uint32_t& best, uint32_t& count) {
  using K = RowKey<T>;
  constexpr int VEC = K::VEC;
  const int off = row_stage_offset(p);
  const int head = min(n, (VEC - off) % VEC);
  best = 0;
  count = 0;
  auto take = [&](uint32_t bits) {
    const uint32_t k = K::of_bits(bits);
    best = max(best, k);
    count += k != 0u;
    return k;
  };
  auto scalar = [&](int i) {
    uint32_t bits;
    if constexpr (sizeof(T) == 4)
      bits = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
    else
      bits = __ldg(reinterpret_cast<const uint16_t*>(p) + i);
    keys[i] = static_cast<typename K::type>(take(bits));
  };
  if (static_cast<int>(threadIdx.x) < head) scalar(threadIdx.x);
  const int nvec = (n - head) / VEC;
  const uint4* src = reinterpret_cast<const uint4*>(p + head);
  uint4* dst = reinterpret_cast<uint4*>(keys + head);
  constexpr int UNROLL = 4;
  for (int v0 = threadIdx.x; v0 < nvec; v0 += UNROLL * kRowThreads) {
    uint4 q[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (v0 + u * kRowThreads < nvec) q[u] = __ldg(src + v0 + u * kRowThreads);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (v0 + u * kRowThreads < nvec) {
        uint32_t w[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 4)
            w[e] = take(w[e]);
          else {
            const uint32_t a = take(w[e] & 0xFFFFu), b = take(w[e] >> 16);
            w[e] = a | (b << 16);
          }
        }
        dst[v0 + u * kRowThreads] = make_uint4(w[0], w[1], w[2], w[3]);
      }
  }
  const int tail = head + nvec * VEC;
  if (tail + static_cast<int>(threadIdx.x) < n) scalar(tail + threadIdx.x);  // fewer than VEC
}

// ------------------------------------------------------------------------------------------------
// Softmax weights as 64-bit integers
// ------------------------------------------------------------------------------------------------

// w(x) = round(2^S exp((x - max) / T)). Integer weights make every sum exact, so running sums do
// not depend on how a row is split over threads and CTAs, and comparisons with a uniform's share of
// the total fall the same way on every path. S = min(44, 62 - ceil(log2 V)) keeps a row's sum below
// 2^62; a weight is off by at most half a unit plus 2^-44 of itself.
//
// The exponential is the table method (P. T. P. Tang, "Table-driven implementation of the
// exponential function in IEEE floating-point arithmetic", ACM TOMS 15, 1989): y = 64 (max - x) log2(e) / T
// = n + f with |f| <= 1/2, exp = 2^-(n >> 6) * tab[n & 63] * e^(-f ln2 / 64), the last factor by
// its Taylor polynomial of degree 4 (error below (0.0055)^5 / 120 = 4e-14).
struct RowWeight {
  float top;     // the row's maximum
  double scale;  // 64 log2(e) / T
  int S;
  const double* tab;

  __device__ __forceinline__ uint64_t operator()(float x) const {
    constexpr double kRound = 6755399441055744.0;   // 1.5 * 2^52: adding it rounds to an integer
    constexpr double kInt = 4503599627370496.0;     // 2^52
    const double y = x == top ? 0.0 : (static_cast<double>(top) - static_cast<double>(x)) * scale;
    if (!(y < 64.0 * (S + 2))) return 0;  // rounds to 0; also an infinite maximum's other entries
    const double r = y + kRound;
    const int n = __double2loint(r);
    const double z = (y - (r - kRound)) * (-0.6931471805599453 / 64.0);
    const double p = fma(fma(fma(fma(z, 1.0 / 24.0, 1.0 / 6.0), z, 0.5), z, 1.0), z, 1.0);
    const double s = __hiloint2double((1023 + S - (n >> 6)) << 20, 0);  // 2^(S - n/64)
    const double w = fma(p * tab[n & 63], s, kInt);
    return static_cast<uint64_t>(__double_as_longlong(w)) & 0xFFFFFFFFFFFFFull;
  }
};

__host__ __device__ inline int row_weight_bits(int V) {
  int b = 0;
  while ((1ll << b) < V) ++b;
  return 62 - b < 44 ? 62 - b : 44;
}

__device__ __forceinline__ void row_exp_table(RowShared& sh) {
  if (threadIdx.x < 64) sh.exp_tab[threadIdx.x] = exp2(-static_cast<double>(threadIdx.x) / 64.0);
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
// Radix selection over the cluster
// ------------------------------------------------------------------------------------------------

// Finds, among the cluster's entries with key >= floor_key in descending order of key, the key
// whose entries hold position `target` of the running measure: the measure (MASS: the sum of
// weights; otherwise the count) of all larger keys is `before` <= target < before + its own. The
// caller makes sure that target is below the total. Every thread of the cluster gets the result.
template <typename T, bool MASS>
__device__ uint32_t row_radix_select(const typename RowKey<T>::type* keys, const RowSlice& sl, uint32_t floor_key,
                                     uint64_t target, const RowWeight& weight, RowShared& sh, uint32_t cs,
                                     uint64_t& before) {
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
    for (int i = threadIdx.x; i < sl.n; i += kRowThreads) {
      const uint32_t k = keys[i];
      if (k < floor_key || k == 0u || (shift < BITS && (k >> shift) != prefix)) continue;
      const uint32_t d = (k >> next) & mask;
      if constexpr (MASS) {
        const uint64_t w = weight(RowKey<T>::value(k));
        if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[d]), static_cast<unsigned long long>(w));
      } else {
        atomicAdd(&counts[d], 1u);
      }
    }
    row_cluster_sync();
    // thread t sums the cluster's bins 2047 - 4t .. 2044 - 4t
    constexpr int PER = kRowBins / kRowThreads;
    uint64_t h[PER], own = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int b = kRowBins - 1 - (static_cast<int>(threadIdx.x) * PER + j);
      h[j] = 0;
      for (uint32_t c = 0; c < cs; ++c) h[j] += MASS ? peer_u64(&sh.hist[b], c) : peer_u32(&counts[b], c);
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
    row_cluster_sync();  // found is set; no CTA clears its bins while another still reads them
    prefix = (prefix << width) | static_cast<uint32_t>(sh.found[0]);
    before = sh.found[1];
    shift = next;
    __syncthreads();  // found is read before the next level sets it
  }
  return prefix;
}

// ------------------------------------------------------------------------------------------------
// Top-k
// ------------------------------------------------------------------------------------------------

// Descending bitonic sort of sh.list[0, n2), n2 a power of two.
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

// Sum over the thread's staged entries of exp((x - top) / T), `c` = log2(e) / T.
template <typename T>
__device__ __forceinline__ float row_exp_sum(const typename RowKey<T>::type* keys, int n, float top, float c) {
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += kRowThreads) {
    const uint32_t k = keys[i];
    if (k) s += ex2_approx((RowKey<T>::value(k) - top) * c);
  }
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) topk_rows_kernel(const T* __restrict__ x, int64_t ldx, int V, int per,
                                                                 int k, float temperature, float* __restrict__ values,
                                                                 int64_t* __restrict__ ids, float* __restrict__ lse) {
  using K = RowKey<T>;
  extern __shared__ __align__(16) uint8_t row_smem[];
  __shared__ RowShared sh;
  uint32_t cs, rank;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(cs));
  rank = cluster_ctarank();
  const int64_t row = blockIdx.x / cs;
  const RowSlice sl(V, per, rank);
  const T* p = x + row * ldx + sl.lo;
  auto* keys = reinterpret_cast<typename K::type*>(row_smem) + row_stage_offset(p);
  uint32_t best, count;
  row_stage<T>(p, sl.n, keys, best, count);
  const uint64_t bmax = block_max_u64(best, sh), bcount = block_sum_u64(count, sh);
  if (threadIdx.x == 0) {
    sh.slot[0] = bmax;
    sh.slot[1] = bcount;
  }
  row_cluster_sync();
  uint32_t top_key = 0;
  uint64_t candidates = 0;
  for (uint32_t r = 0; r < cs; ++r) {
    top_key = max(top_key, static_cast<uint32_t>(peer_u64(&sh.slot[0], r)));
    candidates += peer_u64(&sh.slot[1], r);
  }
  const float top = K::value(top_key);
  // the row's exponential sum, published with the tie counts below (64 fractional bits of a double)
  const float part = top_key && top < INFINITY ? row_exp_sum<T>(keys, sl.n, top, kLog2e / temperature) : 0.f;
  const uint64_t fixed = block_sum_u64(__double2ull_rn(static_cast<double>(part) * 1099511627776.0), sh);  // 2^40
  const int kk = static_cast<int>(candidates < static_cast<uint64_t>(k) ? candidates : k);
  uint32_t cut = 0;
  uint64_t n_gt = 0;
  RowWeight none{};
  if (kk > 0) cut = row_radix_select<T, false>(keys, sl, 1u, kk - 1, none, sh, cs, n_gt);
  // index-ordered compaction: larger keys first, then the lowest-index equals
  uint32_t gt = 0, eq = 0;
  if (kk > 0)
    for (int i = sl.begin(); i < sl.end(); ++i) {
      const uint32_t key = keys[i];
      gt += key > cut;
      eq += key == cut;
    }
  uint64_t total;
  const uint64_t at = block_exclusive_u64((static_cast<uint64_t>(gt) << 32) | eq, sh, total);
  if (threadIdx.x == 0) {
    sh.slot[2] = total;
    sh.slot[3] = fixed;
  }
  row_cluster_sync();
  uint64_t base = 0;
  for (uint32_t r = 0; r < rank; ++r) base += peer_u64(&sh.slot[2], r);
  uint32_t at_gt = static_cast<uint32_t>((base + at) >> 32), at_eq = static_cast<uint32_t>(base + at);
  const uint32_t room = static_cast<uint32_t>(kk - n_gt);
  const uint32_t list0 = mapa_shared(smem_u32(sh.list), 0);
  if (kk > 0 && (gt || eq))
    for (int i = sl.begin(); i < sl.end(); ++i) {
      const uint32_t key = keys[i];
      if (key < cut) continue;
      uint32_t pos;
      if (key > cut)
        pos = at_gt++;
      else if (at_eq < room)
        pos = static_cast<uint32_t>(n_gt) + at_eq++;
      else
        continue;
      st_cluster_u64(list0 + pos * 8, (static_cast<uint64_t>(key) << 32) | ~static_cast<uint32_t>(sl.lo + i));
    }
  uint64_t sum = 0;
  if (rank == 0)
    for (uint32_t r = 0; r < cs; ++r) sum += peer_u64(&sh.slot[3], r);
  row_cluster_sync();  // the list is complete; nothing of another CTA is read after this
  if (rank != 0) return;
  int n2 = 1;
  while (n2 < kk) n2 <<= 1;
  for (int i = kk + threadIdx.x; i < n2; i += kRowThreads) sh.list[i] = 0;
  row_sort_desc(sh.list, n2);
  for (int i = threadIdx.x; i < k; i += kRowThreads) {
    const uint64_t e = i < kk ? sh.list[i] : 0;
    values[row * k + i] = i < kk ? K::value(static_cast<uint32_t>(e >> 32)) : -INFINITY;
    ids[row * k + i] = i < kk ? static_cast<int64_t>(~static_cast<uint32_t>(e)) : -1;
  }
  if (threadIdx.x == 0) {
    const double s = static_cast<double>(sum) / 1099511627776.0;
    lse[row] = top_key == 0 ? -INFINITY
               : !(top < INFINITY) ? INFINITY
                                   : static_cast<float>(static_cast<double>(top) / temperature + log(s));
  }
}

// ------------------------------------------------------------------------------------------------
// Sampling
// ------------------------------------------------------------------------------------------------

struct SampleKnobs {
  const float* temperature;  // [R], or null: one value for every row
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature1, top_p1, min_p1;
  int top_k1;
};

template <typename T>
__global__ void __launch_bounds__(kRowThreads) sample_logits_kernel(const T* __restrict__ x, int64_t ldx, int V, int per,
                                                                     int S, const float* __restrict__ uniform,
                                                                     SampleKnobs knobs, int64_t* __restrict__ tokens) {
  using K = RowKey<T>;
  extern __shared__ __align__(16) uint8_t row_smem[];
  __shared__ RowShared sh;
  uint32_t cs, rank;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(cs));
  rank = cluster_ctarank();
  const int64_t row = blockIdx.x / cs;
  const float temperature = knobs.temperature ? knobs.temperature[row] : knobs.temperature1;
  const int top_k = knobs.top_k ? knobs.top_k[row] : knobs.top_k1;
  const float top_p = knobs.top_p ? knobs.top_p[row] : knobs.top_p1;
  const float min_p = knobs.min_p ? knobs.min_p[row] : knobs.min_p1;
  const bool greedy = temperature < 1e-5f;

  const RowSlice sl(V, per, rank);
  const T* p = x + row * ldx + sl.lo;
  auto* keys = reinterpret_cast<typename K::type*>(row_smem) + row_stage_offset(p);
  uint32_t best, count;
  row_exp_table(sh);
  row_stage<T>(p, sl.n, keys, best, count);
  const uint64_t bmax = block_max_u64(best, sh), bcount = block_sum_u64(count, sh);  // both order the staging
  uint32_t first = 0;  // ~index of the slice's first entry with its largest key
  if (greedy)
    for (int i = threadIdx.x; i < sl.n; i += kRowThreads)
      if (keys[i] == bmax) first = max(first, ~static_cast<uint32_t>(sl.lo + i));
  const uint64_t bfirst = block_max_u64(first, sh);
  if (threadIdx.x == 0) {
    sh.slot[0] = (bmax << 32) | bfirst;
    sh.slot[1] = bcount;
  }
  row_cluster_sync();
  uint64_t top_entry = 0, candidates = 0;
  for (uint32_t r = 0; r < cs; ++r) {
    const uint64_t e = peer_u64(&sh.slot[0], r);
    top_entry = e > top_entry ? e : top_entry;
    candidates += peer_u64(&sh.slot[1], r);
  }
  const uint32_t top_key = static_cast<uint32_t>(top_entry >> 32);
  if (greedy || top_key == 0) {  // the same for the whole cluster
    if (rank == 0 && threadIdx.x == 0)
      tokens[row] = top_key == 0 ? -1 : static_cast<int64_t>(~static_cast<uint32_t>(top_entry));
    row_cluster_sync();  // every CTA has read the others' slots
    return;
  }
  RowWeight weight;
  weight.top = K::value(top_key);
  weight.scale = 92.33248261893567 / static_cast<double>(temperature);  // 64 log2(e) / T
  weight.S = S;
  weight.tab = sh.exp_tab;

  // top-k: keys below the k-th largest (ties kept) leave
  uint32_t cut = 1;
  uint64_t before;
  if (top_k >= 1 && static_cast<uint64_t>(top_k) < candidates)
    cut = row_radix_select<T, false>(keys, sl, 1u, top_k - 1, weight, sh, cs, before);
  // top-p: the key at the border of the nucleus and how many of its entries are inside
  uint64_t ties = ~0ull;
  if (top_p < 1.f) {
    uint64_t mass = 0;
    for (int i = threadIdx.x; i < sl.n; i += kRowThreads)
      if (keys[i] >= cut) mass += weight(K::value(keys[i]));
    mass = block_sum_u64(mass, sh);
    if (threadIdx.x == 0) sh.slot[2] = mass;
    row_cluster_sync();
    mass = 0;
    for (uint32_t r = 0; r < cs; ++r) mass += peer_u64(&sh.slot[2], r);
    const uint64_t target = floor_share(top_p, mass);
    cut = row_radix_select<T, true>(keys, sl, cut, target, weight, sh, cs, before);
    ties = (target - before) / weight(K::value(cut)) + 1;
  }
  // min-p: weights below this leave
  const uint64_t least = __double2ull_ru(static_cast<double>(fminf(fmaxf(min_p, 0.f), 1.f)) * (1ull << S));

  // walk in index order: the thread's kept weight, its offset in the row, the entry that holds u
  const uint64_t cut_weight = weight(K::value(cut));
  uint32_t eq = 0;
  uint64_t sum = 0;
  for (int i = sl.begin(); i < sl.end(); ++i) {
    const uint32_t key = keys[i];
    if (key > cut) {
      const uint64_t w = weight(K::value(key));
      if (w >= least) sum += w;
    } else if (key == cut) {
      ++eq;
    }
  }
  uint64_t eq_total = 0, eq_before = block_exclusive_u64(eq, sh, eq_total);
  if (threadIdx.x == 0) sh.slot[3] = eq_total;
  row_cluster_sync();
  for (uint32_t r = 0; r < rank; ++r) eq_before += peer_u64(&sh.slot[3], r);
  uint64_t eq_kept = eq_before < ties ? min(ties - eq_before, static_cast<uint64_t>(eq)) : 0;
  if (cut_weight < least) eq_kept = 0;
  sum += eq_kept * cut_weight;
  uint64_t cta_total;
  uint64_t run = block_exclusive_u64(sum, sh, cta_total);
  if (threadIdx.x == 0) sh.slot[4] = cta_total;
  row_cluster_sync();
  uint64_t total = 0;
  for (uint32_t r = 0; r < cs; ++r) {
    const uint64_t t = peer_u64(&sh.slot[4], r);
    if (r < rank) run += t;
    total += t;
  }
  const uint64_t target = floor_share(uniform[row], total);
  if (run <= target && target < run + sum) {
    for (int i = sl.begin(); i < sl.end(); ++i) {
      const uint32_t key = keys[i];
      uint64_t w = 0;
      if (key > cut) {
        w = weight(K::value(key));
        if (w < least) w = 0;
      } else if (key == cut && eq_kept > 0) {
        w = cut_weight;
        --eq_kept;
      }
      run += w;
      if (run > target) {
        tokens[row] = sl.lo + i;
        break;
      }
    }
  }
  row_cluster_sync();  // no CTA leaves while another reads its shared memory
}

// ------------------------------------------------------------------------------------------------
// Launch
// ------------------------------------------------------------------------------------------------

struct RowLaunch {
  int cs, per, smem;
};

// Cluster size: the fewest CTAs (a power of two up to 8) whose slices fit `limit` bytes of shared
// memory each; 0 if the row is too long for a cluster.
inline RowLaunch row_launch_plan(int64_t V, int elem) {
  const int64_t limit = 80 * 1024;       // two CTAs per SM beside their static shared memory
  const int64_t hard = 190 * 1024;       // one CTA per SM
  for (int64_t cap : {limit, hard})
    for (int cs = 1; cs <= kRowMaxCluster; cs *= 2) {
      const int64_t per = ceil_div(ceil_div(V, cs), 8) * 8;
      if (per * elem + 32 <= cap) return {cs, static_cast<int>(per), static_cast<int>(per * elem + 32)};
    }
  return {0, 0, 0};
}

template <typename Kern, typename... Args>
inline int row_launch(Kern kernel, const RowLaunch& lp, int64_t rows, cudaStream_t stream, Args... args) {
  ORTHRUS_CHECK_CUDA(ensure_smem(kernel, 192 * 1024));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * lp.cs));
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = lp.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = lp.cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ORTHRUS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  ORTHRUS_CHECK_LAUNCH();
  return ORTHRUS_OK;
}

template <typename T>
int topk_rows_impl(const T* x, int64_t ldx, int64_t R, int64_t V, int k, float temperature, float* values, int64_t* ids,
                   float* lse, cudaStream_t stream) {
  const RowLaunch lp = row_launch_plan(V, sizeof(T));
  ORTHRUS_CHECK_ARG(lp.cs > 0 && R <= (1ll << 31) / kRowMaxCluster - 1);
  return row_launch(topk_rows_kernel<T>, lp, R, stream, x, ldx, static_cast<int>(V), lp.per, k, temperature, values, ids, lse);
}

template <typename T>
int sample_logits_impl(const T* x, int64_t ldx, int64_t R, int64_t V, const float* uniform, const SampleKnobs& knobs,
                       int64_t* tokens, cudaStream_t stream) {
  const RowLaunch lp = row_launch_plan(V, sizeof(T));
  ORTHRUS_CHECK_ARG(lp.cs > 0 && R <= (1ll << 31) / kRowMaxCluster - 1);
  return row_launch(sample_logits_kernel<T>, lp, R, stream, x, ldx, static_cast<int>(V), lp.per,
                    row_weight_bits(static_cast<int>(V)), uniform, knobs, tokens);
}

}  // namespace orthrus
