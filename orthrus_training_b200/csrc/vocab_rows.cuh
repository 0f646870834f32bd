// Row operators over vocabulary logits [R, V]: the k largest entries of a row with its
// log-sum-exp, and sampling from a row's filtered softmax with a given uniform.
//
// One cluster of CS CTAs owns one row. Each CTA reads its contiguous slice of the row once from
// HBM and keeps it in shared memory as order-preserving integer keys (32 bits for fp32, 16 for
// bf16); every later pass runs on shared memory, and the CTAs exchange maxima, sums and histograms
// through distributed shared memory. So the bytes moved are the row itself, whatever the filters
// need.
//
// The k largest entries come from a bound: the k-th largest of the threads' own maxima (512 a CTA)
// is at most the k-th largest entry, and little below it unless the row is arranged against it, so
// the few entries above that bound are gathered into one CTA and ordered there. A nucleus without a
// top-k is found by a 512-bin histogram of weights over the values that can hold its border, then
// exactly among the border bin's entries. Where the gathered entries are too many (rows of equal
// values), a radix selection over the whole cluster, right for every row, takes over.
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
constexpr int kRowList = 2048;     // most entries gathered into one CTA
constexpr int kRowNucleusBins = 512;

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
  uint64_t hist[kRowBins];   // radix selection: counts (as 32-bit words) or masses; else a second list
  uint64_t list[kRowList];   // gathered entries, (key << 32 | ~index)
  double exp_tab[64];        // 2^(-j/64)
  uint64_t warp_u64[kRowThreads / 32];
  uint64_t warp_count[2][kRowThreads / 32];
  uint64_t slot[8];          // this CTA's published partials, one use each between barriers
  uint64_t found[2];         // result of a block-wide search
  uint32_t tmax[kRowThreads];  // the threads' largest keys
  uint32_t listed;           // entries in the list
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

// Visits the entries that row_stage gave this thread: f(index in the slice, key).
template <typename T, typename F>
__device__ __forceinline__ void row_own(const typename RowKey<T>::type* keys, int off, int n, F f) {
  constexpr int VEC = RowKey<T>::VEC;
  const int head = min(n, (VEC - off) % VEC);
  const int t = threadIdx.x;
  if (t < head) f(t, static_cast<uint32_t>(keys[t]));
  const int nvec = (n - head) / VEC;
  const uint4* src = reinterpret_cast<const uint4*>(keys + head);
  for (int v = t; v < nvec; v += kRowThreads) {
    const uint4 q = src[v];
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) {
        f(head + 4 * v + e, w[e]);
      } else {
        f(head + 8 * v + 2 * e, w[e] & 0xFFFFu);
        f(head + 8 * v + 2 * e + 1, w[e] >> 16);
      }
    }
  }
  const int tail = head + nvec * VEC;
  if (tail + t < n) f(tail + t, static_cast<uint32_t>(keys[tail + t]));
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
// The few largest entries
// ------------------------------------------------------------------------------------------------

// A key with at least k entries of the cluster's row at or above it, and not many more: between
// the k-th largest thread maximum and a little below it. Four-way search on counts of the maxima
// (published in tmax before the last cluster barrier), the same in every CTA.
__device__ __forceinline__ uint32_t row_bound(int k, uint32_t top_key, RowShared& sh, uint32_t cs) {
  uint32_t mk[kRowMaxCluster];
  uint32_t least = 0xFFFFFFFFu, some = 0;
#pragma unroll
  for (int c = 0; c < kRowMaxCluster; ++c) {
    mk[c] = c < static_cast<int>(cs) ? peer_u32(&sh.tmax[threadIdx.x], c) : 0u;
    if (mk[c]) {
      least = min(least, mk[c]);
      ++some;
    }
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // three counters of 21 bits a word; `buf` alternates, so one barrier an exchange is enough
  auto total = [&](uint32_t a, uint32_t b, uint32_t c, int buf) {
    a = __reduce_add_sync(0xffffffffu, a);
    b = __reduce_add_sync(0xffffffffu, b);
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) sh.warp_count[buf][warp] = a | (static_cast<uint64_t>(b) << 21) | (static_cast<uint64_t>(c) << 42);
    __syncthreads();
    uint64_t t = 0;
#pragma unroll
    for (int w = 0; w < kRowThreads / 32; ++w) t += sh.warp_count[buf][w];
    return t;
  };
  least = __reduce_min_sync(0xffffffffu, least);
  if (lane == 0) sh.warp_u64[warp] = least;
  uint32_t have = static_cast<uint32_t>(total(some, 0, 0, 0) & 0x1FFFFF);
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) least = min(least, static_cast<uint32_t>(sh.warp_u64[w]));
  if (have < static_cast<uint32_t>(k)) return 1u;
  uint32_t lo = least, hi = top_key + 1;  // at least k maxima at or above lo, fewer at or above hi
  const uint32_t enough = k + k / 4 + 16;
  for (int step = 1; have > enough && hi - lo > 1; ++step) {
    const uint32_t d = hi - lo;
    const uint32_t t1 = lo + (d + 3) / 4, t2 = lo + (d + 1) / 2, t3 = lo + d - d / 4;
    uint32_t a = 0, b = 0, c = 0;
#pragma unroll
    for (int i = 0; i < kRowMaxCluster; ++i) {
      a += mk[i] >= t1;
      b += mk[i] >= t2;
      c += mk[i] >= t3;
    }
    const uint64_t t = total(a, b, c, step & 1);
    a = static_cast<uint32_t>(t) & 0x1FFFFF;
    b = static_cast<uint32_t>(t >> 21) & 0x1FFFFF;
    c = static_cast<uint32_t>(t >> 42);
    const uint32_t want = k;
    if (c >= want) {
      lo = t3;
      have = c;
    } else if (b >= want) {
      lo = t2;
      hi = t3;
      have = b;
    } else if (a >= want) {
      lo = t1;
      hi = t2;
      have = a;
    } else {
      hi = t1;
    }
  }
  __syncthreads();  // warp_u64 and warp_count are free again
  return lo;
}

// Appends this thread's entries with low <= key < high to the CTA's list (listed counts them, past
// the list's end too). `listed` is 0 and visible before; a block barrier follows.
template <typename T>
__device__ __forceinline__ void row_gather(const typename RowKey<T>::type* keys, int off, const RowSlice& sl,
                                           uint32_t low, uint32_t high, RowShared& sh) {
  row_own<T>(keys, off, sl.n, [&](int i, uint32_t key) {
    if (key >= low && key < high) {
      const uint32_t at = atomicAdd(&sh.listed, 1u);
      if (at < kRowList) sh.list[at] = (static_cast<uint64_t>(key) << 32) | ~static_cast<uint32_t>(sl.lo + i);
    }
  });
}

// Entries listed in the whole cluster (after a cluster barrier).
__device__ __forceinline__ uint32_t row_listed(RowShared& sh, uint32_t cs) {
  uint32_t n = 0;
  for (uint32_t c = 0; c < cs; ++c) n += peer_u32(&sh.listed, c);
  return n;
}

// Leader: copies every CTA's list to `out`, at most kRowList entries in all.
__device__ __forceinline__ void row_collect(uint64_t* out, RowShared& sh, uint32_t cs) {
  uint32_t at = 0;
  for (uint32_t c = 0; c < cs; ++c) {
    const uint32_t n = peer_u32(&sh.listed, c);
    for (uint32_t j = threadIdx.x; j < n; j += kRowThreads) out[at + j] = peer_u64(&sh.list[j], c);
    at += n;
  }
  __syncthreads();
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

// Orders `in` (n <= kRowList different entries) descending into `out` (not the same array): by rank
// counting for a few entries, several threads an entry; else by a sorting network on `in`.
__device__ __forceinline__ void row_order(uint64_t* in, uint64_t* out, int n, RowShared& sh) {
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

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2)
    topk_rows_kernel(const T* __restrict__ x, int64_t ldx, int V, int per, int k, float temperature,
                     float* __restrict__ values, int64_t* __restrict__ ids, float* __restrict__ lse) {
  using K = RowKey<T>;
  extern __shared__ __align__(16) uint8_t row_smem[];
  __shared__ RowShared sh;
  uint32_t cs, rank;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(cs));
  rank = cluster_ctarank();
  const int64_t row = blockIdx.x / cs;
  const RowSlice sl(V, per, rank);
  const T* p = x + row * ldx + sl.lo;
  const int off = row_stage_offset(p);
  auto* keys = reinterpret_cast<typename K::type*>(row_smem) + off;
  uint32_t best, count;
  if (threadIdx.x == 0) sh.listed = 0;
  row_stage<T>(p, sl.n, keys, best, count);
  sh.tmax[threadIdx.x] = best;
  // maximum and count of the slice in one exchange: a key of 32 bits over a count of 32
  const uint32_t wbest = __reduce_max_sync(0xffffffffu, best), wcount = __reduce_add_sync(0xffffffffu, count);
  if ((threadIdx.x & 31) == 0) sh.warp_u64[threadIdx.x >> 5] = (static_cast<uint64_t>(wbest) << 32) | wcount;
  __syncthreads();
  uint32_t bmax = 0, bcount = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) {
    bmax = max(bmax, static_cast<uint32_t>(sh.warp_u64[w] >> 32));
    bcount += static_cast<uint32_t>(sh.warp_u64[w]);
  }
  // the slice's sum of exp((x - its maximum) / T)
  const float btop = K::value(bmax);
  const float c = kLog2e / temperature;
  float part = 0.f;
  if (bmax && btop < INFINITY)
    row_own<T>(keys, off, sl.n, [&](int, uint32_t key) {
      part += key ? ex2_approx((K::value(key) - btop) * c) : 0.f;
    });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if ((threadIdx.x & 31) == 0) sh.warp_count[1][threadIdx.x >> 5] = __float_as_uint(part);
  __syncthreads();
  if (threadIdx.x == 0) {
    float s = 0.f;
    for (int w = 0; w < kRowThreads / 32; ++w) s += __uint_as_float(static_cast<uint32_t>(sh.warp_count[1][w]));
    sh.slot[0] = (static_cast<uint64_t>(bmax) << 32) | bcount;
    sh.slot[1] = __float_as_uint(s);
  }
  row_cluster_sync();
  uint32_t top_key = 0, candidates = 0;
  for (uint32_t r = 0; r < cs; ++r) {
    const uint64_t e = peer_u64(&sh.slot[0], r);
    top_key = max(top_key, static_cast<uint32_t>(e >> 32));
    candidates += static_cast<uint32_t>(e);
  }
  const int kk = static_cast<int>(min(candidates, static_cast<uint32_t>(k)));
  if (rank == 0 && threadIdx.x < 32) {  // lane r brings CTA r's sum to the row's maximum
    const uint32_t r = threadIdx.x;
    const double top = K::value(top_key);
    double s = 0.0;
    const uint32_t m = r < cs ? static_cast<uint32_t>(peer_u64(&sh.slot[0], r) >> 32) : 0u;
    if (m)
      s = __uint_as_float(static_cast<uint32_t>(peer_u64(&sh.slot[1], r))) *
          exp((static_cast<double>(K::value(m)) - top) / temperature);
#pragma unroll
    for (int o = kRowMaxCluster / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (r == 0)
      lse[row] = top_key == 0 ? -INFINITY : !(top < INFINITY) ? INFINITY : static_cast<float>(top / temperature + log(s));
  }
  uint64_t* ordered = sh.hist;
  int have = 0;
  if (kk > 0) {
    const uint32_t bound = row_bound(kk, top_key, sh, cs);
    if (best >= bound) row_gather<T>(keys, off, sl, bound, 0xFFFFFFFFu, sh);
    row_cluster_sync();
    const uint32_t n = row_listed(sh, cs);
    if (n <= kRowList) {
      have = static_cast<int>(n);
      if (rank == 0) row_collect(sh.hist, sh, cs);
      row_cluster_sync();  // nothing of another CTA is read after this
      if (rank != 0) return;
      row_order(sh.hist, sh.list, have, sh);
      ordered = sh.list;
    } else {
      uint64_t n_gt;
      RowWeight none{};
      const uint32_t cut = row_radix_select<T, false>(keys, sl, 1u, kk - 1, none, sh, cs, n_gt);
      // index-ordered compaction: larger keys first, then the lowest-index equals
      uint32_t gt = 0, eq = 0;
      for (int i = sl.begin(); i < sl.end(); ++i) {
        const uint32_t key = keys[i];
        gt += key > cut;
        eq += key == cut;
      }
      uint64_t total;
      const uint64_t at = block_exclusive_u64((static_cast<uint64_t>(gt) << 32) | eq, sh, total);
      if (threadIdx.x == 0) sh.slot[2] = total;
      row_cluster_sync();
      uint64_t base = at;
      for (uint32_t r = 0; r < rank; ++r) base += peer_u64(&sh.slot[2], r);
      uint32_t at_gt = static_cast<uint32_t>(base >> 32), at_eq = static_cast<uint32_t>(base);
      const uint32_t room = static_cast<uint32_t>(kk - n_gt);
      const uint32_t list0 = mapa_shared(smem_u32(sh.list), 0);
      if (gt || eq)
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
      row_cluster_sync();  // the list is complete; nothing of another CTA is read after this
      if (rank != 0) return;
      have = kk;
      row_order(sh.list, sh.hist, have, sh);
      ordered = sh.hist;
    }
  } else {
    row_cluster_sync();  // the leader has read the slots
    if (rank != 0) return;
  }
  for (int i = threadIdx.x; i < k; i += kRowThreads) {
    const uint64_t e = i < kk ? ordered[i] : 0;
    values[row * k + i] = i < kk ? K::value(static_cast<uint32_t>(e >> 32)) : -INFINITY;
    ids[row * k + i] = i < kk ? static_cast<int64_t>(~static_cast<uint32_t>(e)) : -1;
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

// Order-preserving integer of a number, rounded down to the key's bits: every entry at or above x has a
// key at or above this.
template <typename T>
__device__ __forceinline__ uint32_t row_key_floor(float x) {
  const uint32_t b = __float_as_uint(x);
  return ((b & 0x80000000u) ? ~b : (b | 0x80000000u)) >> (32 - RowKey<T>::BITS);
}

// The border of the nucleus among all candidates: the key `cut` of its last entry and how many of
// the entries with that key are inside (`ties`); `mass` is the weight of all candidates. The entries
// that weigh at most (mass - target - 1) / V together weigh less than mass - target, so the border
// lies above them: only the others are counted, in bins even in x. False where the border's bin
// holds too many entries (the caller then selects by radix).
template <typename T>
__device__ bool row_nucleus(const typename RowKey<T>::type* keys, int off, const RowSlice& sl, int V, float T_,
                            uint64_t mass, uint64_t target, const RowWeight& weight, RowShared& sh, uint32_t cs,
                            uint32_t& cut, uint64_t& ties) {
  using K = RowKey<T>;
  const float top = weight.top;
  // how far below the maximum (times T) a border can lie, with a margin that covers the fp32 arithmetic;
  // weights are rounded, so one of light + 1 stands for light + 1/2 or more
  const uint64_t light = (mass - target - 1) / static_cast<uint64_t>(V);
  const float depth = (static_cast<float>(weight.S) - log2f(static_cast<float>(light) + 0.5f)) * kLn2 + 1e-3f;
  const float range = depth * T_ + 1e-5f * fabsf(top);
  if (!(top < INFINITY) || !(range < INFINITY)) return false;  // the same in every CTA
  const float inv = static_cast<float>(kRowNucleusBins) / range;
  const uint32_t low = row_key_floor<T>(top - range);
  auto bin = [&](uint32_t key) { return min(kRowNucleusBins - 1, static_cast<int>((top - K::value(key)) * inv)); };
  sh.hist[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.found[0] = ~0ull;
  __syncthreads();
  row_own<T>(keys, off, sl.n, [&](int, uint32_t key) {
    if (key < low || key == 0u) return;
    const uint64_t w = weight(K::value(key));
    if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[bin(key)]), static_cast<unsigned long long>(w));
  });
  row_cluster_sync();
  uint64_t h = 0, total;
  for (uint32_t c = 0; c < cs; ++c) h += peer_u64(&sh.hist[threadIdx.x], c);
  const uint64_t run = block_exclusive_u64(h, sh, total);
  if (run <= target && target < run + h) {
    sh.found[0] = threadIdx.x;
    sh.found[1] = run;
  }
  __syncthreads();
  const uint64_t border = sh.found[0];
  uint64_t before = sh.found[1];
  if (border != ~0ull)
    row_own<T>(keys, off, sl.n, [&](int i, uint32_t key) {
      if (key < low || key == 0u || bin(key) != static_cast<int>(border)) return;
      const uint32_t at = atomicAdd(&sh.listed, 1u);
      if (at < kRowList) sh.list[at] = (static_cast<uint64_t>(key) << 32) | ~static_cast<uint32_t>(sl.lo + i);
    });
  row_cluster_sync();
  const uint32_t n = row_listed(sh, cs);
  constexpr int MOST = kRowList / 2;
  if (border == ~0ull || n > MOST) {
    row_cluster_sync();  // nobody reads the bins any more
    return false;
  }
  // every CTA orders the border bin's entries for itself and finds the entry that holds the target
  row_collect(sh.hist, sh, cs);
  uint64_t* sorted = sh.hist + MOST;
  row_order(sh.hist, sorted, n, sh);
  constexpr int PER = MOST / kRowThreads;
  uint64_t w[PER], own = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint32_t at = threadIdx.x * PER + j;
    w[j] = at < n ? weight(K::value(static_cast<uint32_t>(sorted[at] >> 32))) : 0;
    own += w[j];
  }
  before += block_exclusive_u64(own, sh, total);
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (before <= target && target < before + w[j]) {
      const int at = threadIdx.x * PER + j;
      const uint32_t key = static_cast<uint32_t>(sorted[at] >> 32);
      int first = at;
      while (first > 0 && static_cast<uint32_t>(sorted[first - 1] >> 32) == key) --first;
      sh.found[0] = key;
      sh.found[1] = at - first + 1;
    }
    before += w[j];
  }
  __syncthreads();
  cut = static_cast<uint32_t>(sh.found[0]);
  ties = sh.found[1];
  return true;
}

// The leader's part of a top-k sample: `merged` holds n entries, the top_k largest and every tie of
// the last among them. Filters them and picks the token.
template <typename T>
__device__ void row_pick_listed(uint64_t* merged, uint64_t* sorted, int n, int top_k, float top_p, uint64_t least,
                                float uniform, const RowWeight& weight, RowShared& sh, int64_t* __restrict__ token) {
  using K = RowKey<T>;
  row_order(merged, sorted, n, sh);
  const uint32_t kth = static_cast<uint32_t>(sorted[top_k - 1] >> 32);
  constexpr int PER = kRowList / kRowThreads;
  uint64_t w[PER], own = 0, total;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int at = threadIdx.x * PER + j;
    const uint32_t key = at < n ? static_cast<uint32_t>(sorted[at] >> 32) : 0u;
    w[j] = at < n && key >= kth ? weight(K::value(key)) : 0;
    own += w[j];
  }
  uint64_t before = block_exclusive_u64(own, sh, total);
  const uint64_t target = top_p < 1.f ? floor_share(top_p, total) : ~0ull;
  own = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int at = threadIdx.x * PER + j;
    const uint64_t kept = before <= target && w[j] >= least ? w[j] : 0;
    before += w[j];
    own += kept;
    if (at < n) merged[at] = kept;  // merged has been read by row_order
  }
  const uint64_t all = block_sum_u64(own, sh);
  const uint64_t aim = floor_share(uniform, all);
  // the running sum before an entry in index order is the weight of the kept entries of lower index
  int parts = 32;
  while (parts > 1 && parts * n > kRowThreads) parts >>= 1;
  const int stride = kRowThreads / parts, part = threadIdx.x % parts;
  for (int e0 = 0; e0 < n; e0 += stride) {
    const int e = e0 + threadIdx.x / parts;
    const uint32_t place = e < n ? static_cast<uint32_t>(sorted[e]) : 0u;
    uint64_t run = 0;
    if (e < n)
      for (int j = part; j < n; j += parts)
        if (static_cast<uint32_t>(sorted[j]) > place) run += merged[j];
    for (int o = parts >> 1; o > 0; o >>= 1) run += __shfl_xor_sync(0xffffffffu, run, o);
    if (e < n && part == 0 && run <= aim && aim < run + merged[e]) *token = ~place;
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2)
    sample_logits_kernel(const T* __restrict__ x, int64_t ldx, int V, int per, int S,
                         const float* __restrict__ uniform, SampleKnobs knobs, int64_t* __restrict__ tokens) {
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
  const int off = row_stage_offset(p);
  auto* keys = reinterpret_cast<typename K::type*>(row_smem) + off;
  uint32_t best, count;
  row_exp_table(sh);
  if (threadIdx.x == 0) sh.listed = 0;
  row_stage<T>(p, sl.n, keys, best, count);
  sh.tmax[threadIdx.x] = best;
  const uint32_t wbest = __reduce_max_sync(0xffffffffu, best), wcount = __reduce_add_sync(0xffffffffu, count);
  if ((threadIdx.x & 31) == 0) sh.warp_u64[threadIdx.x >> 5] = (static_cast<uint64_t>(wbest) << 32) | wcount;
  __syncthreads();
  uint32_t bmax = 0, bcount = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) {
    bmax = max(bmax, static_cast<uint32_t>(sh.warp_u64[w] >> 32));
    bcount += static_cast<uint32_t>(sh.warp_u64[w]);
  }
  if (threadIdx.x == 0) {
    sh.slot[0] = (static_cast<uint64_t>(bmax) << 32) | bcount;
    sh.slot[1] = 0;
  }
  if (greedy) {  // the slice's first entry with its largest key
    __syncthreads();
    uint32_t first = 0;
    if (best == bmax)
      row_own<T>(keys, off, sl.n, [&](int i, uint32_t key) {
        if (key == bmax) first = max(first, ~static_cast<uint32_t>(sl.lo + i));
      });
    if (first) atomicMax(reinterpret_cast<unsigned long long*>(&sh.slot[1]), static_cast<unsigned long long>(first));
  }
  row_cluster_sync();
  uint32_t top_key = 0, candidates = 0, top_place = 0;
  for (uint32_t r = 0; r < cs; ++r) {
    const uint64_t e = peer_u64(&sh.slot[0], r);
    const uint32_t key = static_cast<uint32_t>(e >> 32);
    if (key > top_key) {  // of equal maxima the first CTA's
      top_key = key;
      top_place = greedy ? static_cast<uint32_t>(peer_u64(&sh.slot[1], r)) : 0u;
    }
    candidates += static_cast<uint32_t>(e);
  }
  if (greedy || top_key == 0) {  // the same for the whole cluster
    if (rank == 0 && threadIdx.x == 0) tokens[row] = top_key == 0 ? -1 : static_cast<int64_t>(~top_place);
    row_cluster_sync();  // every CTA has read the others' slots
    return;
  }
  RowWeight weight;
  weight.top = K::value(top_key);
  weight.scale = 92.33248261893567 / static_cast<double>(temperature);  // 64 log2(e) / T
  weight.S = S;
  weight.tab = sh.exp_tab;
  // min-p: weights below this leave
  const float floor_p = fminf(fmaxf(min_p, 0.f), 1.f);
  const uint64_t least = __double2ull_ru(static_cast<double>(floor_p) * (1ull << S));

  // top-k: keys below the k-th largest (ties kept) leave
  uint32_t cut = 1;
  uint64_t before;
  if (top_k >= 1 && static_cast<uint32_t>(top_k) < candidates) {
    if (top_k <= kRowMaxK) {
      const uint32_t bound = row_bound(top_k, top_key, sh, cs);
      if (best >= bound) row_gather<T>(keys, off, sl, bound, 0xFFFFFFFFu, sh);
      row_cluster_sync();
      const uint32_t n = row_listed(sh, cs);
      if (n <= kRowList) {  // everything else happens in one CTA
        if (rank == 0) row_collect(sh.hist, sh, cs);
        row_cluster_sync();  // nothing of another CTA is read after this
        if (rank == 0)
          row_pick_listed<T>(sh.hist, sh.list, n, top_k, top_p, least, uniform[row], weight, sh, tokens + row);
        return;
      }
    }
    cut = row_radix_select<T, false>(keys, sl, 1u, top_k - 1, weight, sh, cs, before);
  }
  // top-p: the key at the border of the nucleus and how many of its entries are inside
  uint64_t ties = ~0ull;
  if (top_p < 1.f) {
    uint64_t mass = 0;
    row_own<T>(keys, off, sl.n, [&](int, uint32_t key) {
      if (key >= cut) mass += weight(K::value(key));
    });
    mass = block_sum_u64(mass, sh);
    if (threadIdx.x == 0) sh.slot[2] = mass;
    row_cluster_sync();
    mass = 0;
    for (uint32_t r = 0; r < cs; ++r) mass += peer_u64(&sh.slot[2], r);
    const uint64_t target = floor_share(top_p, mass);
    if (cut > 1 ||
        !row_nucleus<T>(keys, off, sl, V, temperature, mass, target, weight, sh, cs, cut, ties)) {
      cut = row_radix_select<T, true>(keys, sl, cut, target, weight, sh, cs, before);
      ties = (target - before) / weight(K::value(cut)) + 1;
    }
  }
  // no entry below this key passes min-p (lower by a margin that covers fp32)
  uint32_t lowest = cut;
  if (floor_p > 0.f && weight.top < INFINITY)
    lowest = max(cut, row_key_floor<T>(weight.top + temperature * (logf(floor_p) - 1e-3f) - 1e-5f * fabsf(weight.top)));

  // walk in index order: the thread's kept weight, its offset in the row, the entry that holds u
  const uint64_t cut_weight = weight(K::value(cut));
  uint32_t eq = 0;
  uint64_t sum = 0;
  for (int i = sl.begin(); i < sl.end(); ++i) {
    const uint32_t key = keys[i];
    if (key < lowest) continue;
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
      if (key < lowest) continue;
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

// Cluster size: the fewest CTAs (a power of two up to 8) with at most 20480 entries each, about 40 a
// thread, so that two CTAs share an SM and a single row is spread wide; longer rows take up to one
// CTA's shared memory. 0 if the row is too long for a cluster.
inline RowLaunch row_launch_plan(int64_t V, int elem) {
  for (int cs = 1; cs <= kRowMaxCluster; cs *= 2) {
    const int64_t per = ceil_div(ceil_div(V, cs), 8) * 8;
    const int64_t bytes = per * elem + 32;
    if (per <= 20480 || (cs == kRowMaxCluster && bytes <= 190 * 1024))
      return {cs, static_cast<int>(per), static_cast<int>(bytes)};
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
