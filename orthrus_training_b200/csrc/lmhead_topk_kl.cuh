// Distillation from a teacher's top logits through the LM head: per student row h with the kept
// teacher logits (v_j, id_j) of its teacher row,
//
//   q_j = softmax over the kept v_j / T      (or exp(v_j / T - lse) with the teacher's normaliser)
//   p   = softmax(W h / T) over the whole vocabulary
//   kl  = sum_j q_j (log q_j - log p_{id_j})          total = sum_r w_r kl_r
//   d total / dh = (w / T) (Q p - q) W                Q = sum_j q_j
//
// The student's normaliser needs every logit, so forward and gradient are two products of
// [n, d] x [d, V]; the teacher costs its k entries per row. With z = sum_i exp(s_i / T - c) for any
// reference c of the row, e_i = exp(s_i / T - c),
//
//   grad = (w Q / (T z)) (e - q z / Q) W
//
// so one sweep over the vocabulary can write e before z is known: the row factor is applied to the
// finished product, and only the k kept entries are rewritten in between. bf16 passes, a chunk of rows
// at a time:
//   exp    logits tile in tensor memory (CTA pairs), e in bf16 to the chunk buffer [rows, V],
//          per-row partial z, sum of e times its exponent and maximum, and the fp32 logits at the kept
//          ids picked out of the tile;
//   finish z, kl, agreement, the kept entries e_j - q_j z / Q (one rounding of the difference, so
//          the gradient of a student near its teacher is not the difference of rounded numbers),
//          and the row factor;
//   grad   row factor * (chunk buffer @ W) on CTA pairs (gemm2_tc.cuh).
// The reference c is the student's logit at the teacher's first id. bf16 has fp32's exponent range, so
// a c within 60 bits of the row's maximum loses nothing. Rows where it is further below (another
// logit is the student's) or above (T so low that the roundings of that logit, over T, are many bits)
// are noticed, and swept again relative to their maximum, subtracted before the division by T, where
// nothing is lost at any T (whole tiles of 256 rows; that launch ends at once where there are none).
//
// The tensor cores' adder cuts where fp32 rounds, so a logit comes out short by a part delta of itself:
// with normal operands about 8e-10 d, up to 2.3e-9 d for products of one sign, nothing where the sums
// are exact. A common factor of the logits is to kl what its derivative says,
//   kl(s (1 + delta)) = kl(s) + delta (Q sum_i p_i s_i - sum_j q_j s_j) / T + O(delta^2),
// and delta is measured for each row, by least squares over the two logits whose fp32 products are at
// hand: the teacher's first and the student's largest. Relative error of kl_rows against 64 bits: 6.4e-7 at
// 1999 x 50257 x 768 (3.7e-6 without; torch's fp32 products 6.1e-7), 2.8e-7 at 512 x 151936 x 1024 (9e-7;
// 5.3e-7). It costs one more fp32 product per row and one FMA per exponential, 1 % of 512 rows.
//
// fp32 rows run on CUDA cores: logits = student @ W^T, a row kernel that turns a row of logits into
// its kl and the difference (w / T) (Q p - q), and grad = difference @ W.
#pragma once

#include "gemm2_tc.cuh"
#include "gemm_f32.cuh"
#include "lmhead_kl.cuh"

namespace orthrus {

constexpr int kTopkKlMaxK = 1024;
constexpr int kTopkKlThreads = 512;

// ------------------------------------------------------------------------------------------------
// fp32 rows
// ------------------------------------------------------------------------------------------------

// The kept teacher entries of one row in shared memory. Entries with id < 0 or value -inf are
// padding (q = 0, id = -1); an id past the vocabulary is recorded and counts as padding.
struct TopkTeacherRow {
  float q[kTopkKlMaxK];
  float logq[kTopkKlMaxK];
  int id[kTopkKlMaxK];
  float red[kTopkKlThreads / 32];
  int redi[kTopkKlThreads / 32];
};

__device__ __forceinline__ float tk_block_sum(float v, TopkTeacherRow& sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < kTopkKlThreads / 32; ++w) t += sh.red[w];
  return t;
}

// Largest value and the lowest index that holds it, over the block.
__device__ __forceinline__ void tk_block_argmax(float& v, int& i, TopkTeacherRow& sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, v, o);
    const int oi = __shfl_xor_sync(0xffffffffu, i, o);
    if (ov > v || (ov == v && oi < i)) {
      v = ov;
      i = oi;
    }
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    sh.red[threadIdx.x >> 5] = v;
    sh.redi[threadIdx.x >> 5] = i;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kTopkKlThreads / 32; ++w)
    if (sh.red[w] > v || (sh.red[w] == v && sh.redi[w] < i)) {
      v = sh.red[w];
      i = sh.redi[w];
    }
}

// Fills `sh` with the teacher row of student row r; returns Q and the id of the first largest value
// (-1 if nothing is kept).
__device__ inline float tk_load_teacher(const float* __restrict__ values, const int64_t* __restrict__ ids, int k,
                                        int64_t m, const int64_t* __restrict__ index,
                                        const float* __restrict__ teacher_lse, int V, float T, int64_t r,
                                        TopkTeacherRow& sh, int& top_id) {
  int64_t t = index ? index[r] : r;
  const bool row_ok = t >= 0 && t < m;
  if (!row_ok) {
    if (threadIdx.x == 0) record_error(ORTHRUS_ERR_BOUNDS);
    t = 0;
  }
  float best = -INFINITY;
  int at = INT_MAX;
  for (int j = threadIdx.x; j < k; j += kTopkKlThreads) {
    const float v = values[t * k + j];
    const int64_t id = ids[t * k + j];
    const bool past = id >= V;
    if (past) record_error(ORTHRUS_ERR_BOUNDS);
    const bool live = row_ok && id >= 0 && !past && v != -INFINITY;
    sh.id[j] = live ? static_cast<int>(id) : -1;
    sh.logq[j] = live ? v : -INFINITY;
    if (live && v > best) {
      best = v;
      at = j;
    }
  }
  tk_block_argmax(best, at, sh);
  top_id = at == INT_MAX ? -1 : sh.id[at];
  // log q from the distance to the largest value: v / T - (best / T + log z) would lose log z where
  // best / T is large
  float base = 0.f, norm;
  if (teacher_lse != nullptr) {
    norm = teacher_lse[t];
  } else {
    float z = 0.f;
    base = best;
    for (int j = threadIdx.x; j < k; j += kTopkKlThreads)
      if (sh.id[j] >= 0) z += expf((sh.logq[j] - base) / T);
    norm = logf(tk_block_sum(z, sh));
  }
  float Q = 0.f;
  for (int j = threadIdx.x; j < k; j += kTopkKlThreads) {
    const float lq = sh.id[j] >= 0 ? (sh.logq[j] - base) / T - norm : -INFINITY;
    sh.logq[j] = lq;
    sh.q[j] = expf(lq);
    Q += sh.q[j];
  }
  return tk_block_sum(Q, sh);
}

// One CTA per row of a chunk: logits [rows, ld] fp32 of student rows c0.. -> kl_rows, agree and, with
// `diff`, the difference (w / T) (Q p - q) (which may overwrite the logits).
__global__ void __launch_bounds__(kTopkKlThreads)
    topk_kl_rows_kernel(const float* logits, int64_t ld, int c0, int V, const float* __restrict__ values,
                        const int64_t* __restrict__ ids, int k, int64_t m, const int64_t* __restrict__ index,
                        const float* __restrict__ teacher_lse, const float* __restrict__ row_weight, float T,
                        float* __restrict__ kl_rows, uint8_t* __restrict__ agree, float* diff, int64_t ldd) {
  __shared__ TopkTeacherRow sh;
  const int64_t r = c0 + static_cast<int64_t>(blockIdx.x);
  const float* x = logits + blockIdx.x * ld;
  int top_id;
  const float Q = tk_load_teacher(values, ids, k, m, index, teacher_lse, V, T, r, sh, top_id);
  float top = -INFINITY;
  int at = INT_MAX;
  for (int i = threadIdx.x; i < V; i += kTopkKlThreads)
    if (x[i] > top) {
      top = x[i];
      at = i;
    }
  tk_block_argmax(top, at, sh);
  float z = 0.f;
  for (int i = threadIdx.x; i < V; i += kTopkKlThreads) z += expf((x[i] - top) / T);
  z = tk_block_sum(z, sh);
  const float logz = logf(z);
  float kl = 0.f;
  for (int j = threadIdx.x; j < k; j += kTopkKlThreads)
    if (sh.id[j] >= 0 && sh.q[j] > 0.f) kl += sh.q[j] * (sh.logq[j] - ((x[sh.id[j]] - top) / T - logz));
  kl = tk_block_sum(kl, sh);
  if (threadIdx.x == 0) {
    kl_rows[r] = kl;
    agree[r] = top_id >= 0 && top_id == at;
  }
  if (diff == nullptr) return;
  // the kept entries' differences first (they read the logits), then the sweep, then their stores
  const float w = (row_weight ? row_weight[r] : 1.f) / T;
  float* d = diff + blockIdx.x * ldd;
  if (w * Q == 0.f) {  // no mass or no weight: 0 whatever the row holds (the sum above is past its last reads)
    for (int i = threadIdx.x; i < V; i += kTopkKlThreads) d[i] = 0.f;
    return;
  }
  constexpr int PER = kTopkKlMaxK / kTopkKlThreads;
  float fix[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int j = threadIdx.x + u * kTopkKlThreads;
    if (j >= k || sh.id[j] < 0) continue;
    float q = 0.f;  // an id kept twice counts with its whole mass
    for (int i = 0; i < k; ++i) q += sh.id[i] == sh.id[j] ? sh.q[i] : 0.f;
    fix[u] = w * (Q * (expf((x[sh.id[j]] - top) / T) / z) - q);
  }
  __syncthreads();
  const float scale = w * Q / z;
  for (int i = threadIdx.x; i < V; i += kTopkKlThreads) d[i] = scale * expf((x[i] - top) / T);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int j = threadIdx.x + u * kTopkKlThreads;
    if (j < k && sh.id[j] >= 0) d[sh.id[j]] = fix[u];
  }
}

// ------------------------------------------------------------------------------------------------
// bf16 rows
// ------------------------------------------------------------------------------------------------

constexpr float kTopkExpLimit = 60.f;  // log2 of the largest e: z and Q / z stay normal numbers
constexpr int kTopkMaxSplits = 64;

// One CTA per teacher row: its entries sorted by id (sid [m, k], padding INT_MAX at the end) with log q
// beside them, the id of the first largest value and Q. Sorted ids let a sweep over the vocabulary meet
// them in its own order.
__global__ void __launch_bounds__(128)
    topk_teacher_kernel(const float* __restrict__ values, const int64_t* __restrict__ ids, int k, int V, float T,
                        const float* __restrict__ teacher_lse, int* __restrict__ sid, float* __restrict__ slogq,
                        int* __restrict__ top_id, float* __restrict__ mass) {
  __shared__ int id[kTopkKlMaxK];
  __shared__ float val[kTopkKlMaxK];
  __shared__ float red[4];
  __shared__ int redi[4];
  const int64_t t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_launch_dependents();
  int n2 = 1;
  while (n2 < k) n2 <<= 1;
  float best = -INFINITY;
  int at = INT_MAX;
  for (int j = threadIdx.x; j < n2; j += 128) {
    const float v = j < k ? values[t * k + j] : -INFINITY;
    const int64_t i = j < k ? ids[t * k + j] : -1;
    if (i >= V) record_error(ORTHRUS_ERR_BOUNDS);
    const bool live = i >= 0 && i < V && v != -INFINITY;
    id[j] = live ? static_cast<int>(i) : INT_MAX;
    val[j] = live ? v : -INFINITY;
    if (live && v > best) {
      best = v;
      at = j;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, best, o);
    const int oi = __shfl_xor_sync(0xffffffffu, at, o);
    if (ov > best || (ov == best && oi < at)) {
      best = ov;
      at = oi;
    }
  }
  if (lane == 0) {
    red[warp] = best;
    redi[warp] = at;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w)
    if (red[w] > best || (red[w] == best && redi[w] < at)) {
      best = red[w];
      at = redi[w];
    }
  const int first = at == INT_MAX ? -1 : id[at];
  for (int size = 2; size <= n2; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n2 / 2; i += 128) {
        const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const int x = id[lo], y = id[hi];
        if ((x > y) == ((lo & size) == 0)) {
          const float v = val[lo];
          id[lo] = y;
          id[hi] = x;
          val[lo] = val[hi];
          val[hi] = v;
        }
      }
    }
  __syncthreads();
  auto sum = [&](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
  };
  float base = 0.f, norm;  // as tk_load_teacher
  if (teacher_lse != nullptr) {
    norm = teacher_lse[t];
  } else {
    float z = 0.f;
    base = best;
    for (int j = threadIdx.x; j < k; j += 128)
      if (id[j] != INT_MAX) z += expf((val[j] - base) / T);
    norm = logf(sum(z));
  }
  float q = 0.f;
  for (int j = threadIdx.x; j < k; j += 128) {
    const float lq = id[j] != INT_MAX ? (val[j] - base) / T - norm : -INFINITY;
    sid[t * k + j] = id[j];
    slogq[t * k + j] = lq;
    q += expf(lq);
  }
  q = sum(q);
  if (threadIdx.x == 0) {
    top_id[t] = first;
    mass[t] = q;
  }
}

// The product of two rows of D bf16 numbers in fp32, by a warp; every lane has it.
__device__ __forceinline__ float topk_dot(const __nv_bfloat16* h, const __nv_bfloat16* w, int D) {
  const uint4* h4 = reinterpret_cast<const uint4*>(h);
  const uint4* w4 = reinterpret_cast<const uint4*>(w);
  float dot = 0.f;
  for (int i = threadIdx.x & 31; i < D / 8; i += 32) {
    const uint4 a = h4[i], b = w4[i];
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      dot = fmaf(__uint_as_float(x[e] << 16), __uint_as_float(y[e] << 16), dot);
      dot = fmaf(__uint_as_float(x[e] & 0xffff0000u), __uint_as_float(y[e] & 0xffff0000u), dot);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
  return dot;
}

// One warp per student row: its teacher row (-1 if the index is out of range) and its logit at the
// teacher's first id, whose log2(e) / T fold is the reference c; clears the rows' maxima and the second
// sweep's flags.
__global__ void __launch_bounds__(256)
    topk_student_kernel(const __nv_bfloat16* __restrict__ student, const __nv_bfloat16* __restrict__ W, int64_t n,
                        int64_t m, int D, const int64_t* __restrict__ index, const int* __restrict__ top_id,
                        int* __restrict__ trow, float* __restrict__ top_logit, unsigned* __restrict__ rowmax,
                        int* __restrict__ again) {
  const int64_t r = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  griddep_launch_dependents();
  griddep_wait();  // launched as a programmatic dependent
  if (r >= n) return;
  int64_t t = index ? index[r] : r;
  if (t < 0 || t >= m) {
    if (lane == 0) record_error(ORTHRUS_ERR_BOUNDS);
    t = -1;
  }
  const int id = t < 0 ? -1 : top_id[t];
  const float dot = id < 0 ? 0.f : topk_dot(student + r * D, W + static_cast<int64_t>(id) * D, D);
  if (lane == 0) {
    trow[r] = static_cast<int>(t);
    top_logit[r] = dot;
    rowmax[r] = 0;
    if (r % 256 == 0) again[r / 256] = 0;
  }
}

// A row's largest logit as an ordered integer (0: none yet).
__device__ __forceinline__ unsigned topk_max_key(float x) {
  const unsigned b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// How a row's exponents are formed: (x - shift) * alpha - ref. In the first sweep shift is 0; once the
// row's maximum is known, a reference too far from it (of a row with teacher entries) gives way to it.
struct TopkReference {
  float shift, ref;
  __device__ __forceinline__ float operator()(float x, float alpha) const { return fmaf(x - shift, alpha, -ref); }
};
__device__ __forceinline__ TopkReference topk_reference(float top_logit, unsigned max_key, float alpha, bool kept) {
  const float ref = top_logit * alpha;
  if (!kept || max_key == 0u) return {0.f, ref};
  const float m = __uint_as_float((max_key & 0x80000000u) ? (max_key & 0x7FFFFFFFu) : ~max_key);
  return fabsf(fmaf(m, alpha, -ref)) > kTopkExpLimit ? TopkReference{m, 0.f} : TopkReference{0.f, ref};
}

struct TopkExpTile {
  static constexpr int BM = 128, BK = 64, BN = 256;  // rows and columns of a pair: 256 x 256
  static constexpr int A_BYTES = BM * BK * 2;        // this CTA's 128 student rows
  static constexpr int B_BYTES = 128 * BK * 2;       // this CTA's 128 vocabulary rows of W
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 6;
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int STAGING = 32 * 64 * 2;  // per epilogue warp: 32 rows x 64 bf16 on their way out
  static constexpr int SMEM = STAGES * STAGE_BYTES + EPI_WARPS * STAGING + 1024 + 256;
};

struct TopkExpArgs {
  int rows, c0;  // rows of the chunk, its first student row
  int V, D, k;
  int vtiles, tiles_per_split, rtiles, units;
  float alpha;            // log2(e) / T
  const int* trow;        // [n]
  const float* top_logit; // [n]
  const int* sid;         // [m, k]
  const int* top_id;      // [m]
  unsigned* rowmax;       // [n]: topk_max_key of the row's maximum, from the first sweep
  int* again;             // [ceil(n / 256)]: tiles that may hold a row whose reference is too far off
  bool second;            // the second sweep takes the flagged tiles only
  float* kept;            // [chunk, k] student logits at the sorted ids
  float* part_z;          // [2 splits, chunk], as the three below
  float* part_y;          // sum of e_i times its exponent
  float* part_m;
  int* part_i;
  int64_t part_ld;
  bool write_e;           // the exponentials are wanted (tmE)
};

// One fp32 column of this warp's 32 TMEM lanes.
__device__ __forceinline__ float tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
  return __uint_as_float(r);
}

// The exp sweep: a persistent cluster of two CTAs walks units (tile of 256 student rows, range of the
// vocabulary). Warp 0 loads, warp 1 of the leader issues the MMAs of the pair, warps 2-9 are the
// epilogue: thread (quarter, half, lane) owns row quarter * 32 + lane of its CTA and 128 of the
// tile's 256 columns. Two accumulators of 256 columns let the epilogue of one tile run under the
// MMAs of the next.
__global__ void __launch_bounds__(TopkExpTile::THREADS, 1)
    topk_exp_kernel(const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmE, const TopkExpArgs a) {
  using T = TopkExpTile;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + T::STAGES * T::A_BYTES;
  uint8_t* staging = sB + T::STAGES * T::B_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + T::EPI_WARPS * T::STAGING);
  uint64_t* empty = full + T::STAGES;
  uint64_t* acc_full = empty + T::STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;      // [2], leader only: both CTAs' epilogue warps arrive
  uint64_t* mma_drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  const int KB = (a.D + T::BK - 1) / T::BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * T::EPI_WARPS);
    }
    mbar_init(mma_drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  __syncthreads();
  cluster_sync_all();  // the peer's barriers are initialised before anyone signals them
  // launched as a programmatic dependent: the set-up above overlaps the previous kernel's tail
  griddep_launch_dependents();
  griddep_wait();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // unit u = (row tile u % rtiles, vocabulary range u / rtiles); the same tiles for every role of
  // both CTAs (the flags do not change during the second sweep)
  auto unit_tiles = [&](int u, int& row0, int& split, int& t0) {
    const int rt = u % a.rtiles;
    split = u / a.rtiles;
    row0 = rt * 256 + static_cast<int>(rank) * T::BM;  // this CTA's first row in the chunk
    t0 = split * a.tiles_per_split;
    if (a.second && a.again[a.c0 / 256 + rt] == 0) return 0;
    return max(min(a.vtiles, t0 + a.tiles_per_split) - t0, 0);
  };

  if (warp == 0) {
    if (elect_one()) {
      prefetch_tensormap(&tmH);
      prefetch_tensormap(&tmW);
      int it = 0, issued = 0;
      for (int u = cluster; u < a.units && !*abort_flag; u += nclusters) {
        int row0, split, t0;
        const int ntiles = unit_tiles(u, row0, split, t0);
        for (int t = 0; t < ntiles && !*abort_flag; ++t) {
          const int v0 = (t0 + t) * T::BN + static_cast<int>(rank) * 128;
          for (int kb = 0; kb < KB; ++kb, ++it) {
            const int s = it % T::STAGES;
            if (!mbar_wait(&empty[s], ((it / T::STAGES) & 1) ^ 1)) {
              *abort_flag = 1;
              break;
            }
            const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
            if (leader) mbar_arrive_expect_tx(&full[s], 2 * T::STAGE_BYTES);
            tma_load_2d_pair(sA + s * T::A_BYTES, &tmH, bar, kb * T::BK, a.c0 + row0);
            tma_load_2d_pair(sB + s * T::B_BYTES, &tmW, bar, kb * T::BK, v0);
            issued = it + 1;
          }
        }
      }
      if (*abort_flag && leader)
        for (int i = max(0, issued - T::STAGES); i < issued; ++i)
          mbar_wait_short(&full[i % T::STAGES], (i / T::STAGES) & 1);
    }
  } else if (warp == 1) {
    if (leader && elect_one()) {
      constexpr uint32_t idesc = umma_idesc_bf16(256, T::BN, false, false);
      int it = 0, tt = 0;
      for (int u = cluster; u < a.units && !*abort_flag; u += nclusters) {
        int row0, split, t0;
        const int ntiles = unit_tiles(u, row0, split, t0);
        for (int t = 0; t < ntiles && !*abort_flag; ++t, ++tt) {
          const int b = tt & 1;
          if (!mbar_wait_cluster(&acc_empty[b], ((tt >> 1) & 1) ^ 1)) {
            *abort_flag = 1;
            break;
          }
          tc_fence_after();
          for (int kb = 0; kb < KB; ++kb, ++it) {
            const int s = it % T::STAGES;
            if (!mbar_wait(&full[s], (it / T::STAGES) & 1)) {
              *abort_flag = 1;
              break;
            }
            tc_fence_after();
            const uint32_t a_base = smem_u32(sA + s * T::A_BYTES);
            const uint32_t b_base = smem_u32(sB + s * T::B_BYTES);
#pragma unroll
            for (int kk = 0; kk < T::BK / 16; ++kk)
              umma_f16_pair(tmem + b * T::BN, g2_desc_k(a_base, kk), g2_desc_k(b_base, kk), idesc,
                            (kb > 0 || kk > 0) ? 1u : 0u);
            umma_commit_pair(&empty[s], 3);
          }
          umma_commit_pair(&acc_full[b], 3);
        }
      }
      // every MMA issued has completed (in both CTAs' TMEM) before either frees its columns
      umma_commit_pair(mma_drain, 3);
      mbar_wait(mma_drain, 0);
    } else if (!leader && elect_one()) {
      mbar_wait(mma_drain, 0);  // the leader's last MMAs also wrote this CTA's TMEM
    }
  } else {
    const int quarter = warp & 3;      // TMEM lanes this warp may read
    const int half = (warp - 2) >> 2;  // which half of the tile's columns it takes
    uint8_t* const stage = staging + (warp - 2) * T::STAGING;
    int tt = 0;
    for (int u = cluster; u < a.units && !*abort_flag; u += nclusters) {
      int row0, split, t0;
      const int ntiles = unit_tiles(u, row0, split, t0);
      if (ntiles == 0) continue;
      const int crow = row0 + quarter * 32 + lane;  // row in the chunk
      const bool live = crow < a.rows;
      const int trow = live ? a.trow[a.c0 + crow] : -1;
      const int top = trow < 0 ? -1 : a.top_id[trow];
      const TopkReference ref = topk_reference(live ? a.top_logit[a.c0 + crow] : 0.f,
                                               live && a.second ? a.rowmax[a.c0 + crow] : 0u, a.alpha, top >= 0);
      bool far = false;  // the row's largest logit may be too far from its reference
      // the row's sorted ids from this unit's first column on
      const int* sid = a.sid + static_cast<int64_t>(trow < 0 ? 0 : trow) * a.k;
      int p = 0;
      if (trow >= 0)
        for (int hi = a.k; p < hi;) {
          const int mid = (p + hi) / 2;
          if (sid[mid] < t0 * T::BN) p = mid + 1;
          else hi = mid;
        }
      int next = trow >= 0 && p < a.k ? sid[p] : INT_MAX;
      float z = 0.f, zy = 0.f, m = -INFINITY;
      int idx = INT_MAX;
      for (int t = 0; t < ntiles; ++t, ++tt) {
        const int b = tt & 1;
        if (*abort_flag || !mbar_wait(&acc_full[b], (tt >> 1) & 1)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const int v0 = (t0 + t) * T::BN;
        const int lo = v0 + half * 128;
        const uint32_t base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + b * T::BN;
        // kept ids among these columns: the warp loads one column at a time, the lanes whose id it is
        // take it
        while (next < lo) next = ++p < a.k ? sid[p] : INT_MAX;
        __syncwarp();
        for (uint32_t todo; (todo = __ballot_sync(0xffffffffu, next < lo + 128)) != 0;) {
          const int col = __shfl_sync(0xffffffffu, next, __ffs(todo) - 1);
          const float x = tmem_ld1(base + (col - v0));
          tmem_wait_ld();
          while (next == col) {  // an id kept twice stands twice
            a.kept[static_cast<int64_t>(crow) * a.k + p] = x;
            far |= col == top && ref(x, a.alpha) < -kTopkExpLimit;
            next = ++p < a.k ? sid[p] : INT_MAX;
          }
          __syncwarp();
        }
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          const int col0 = lo + c * 32;
          const int nvalid = min(32, a.V - col0);
          if (nvalid <= 0) break;  // uniform over the warp
          if (a.write_e && !(c & 1)) {  // the previous store has read the staging tile
            if (lane == 0) tma_store_wait_read_all();
            __syncwarp();
          }
          float x[32];
          tmem_ld32(base + half * 128 + c * 32, x);
          tmem_wait_ld();
          // first maximum, four independent chains (column j in chain j % 4), lower columns on ties
          float cmv[4];
          int civ[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            cmv[i] = -INFINITY;
            civ[i] = 32;
          }
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j < nvalid && x[j] > cmv[j & 3]) {
              cmv[j & 3] = x[j];
              civ[j & 3] = j;
            }
#pragma unroll
          for (int i = 1; i < 4; ++i)
            if (cmv[i] > cmv[0] || (cmv[i] == cmv[0] && civ[i] < civ[0])) {
              cmv[0] = cmv[i];
              civ[0] = civ[i];
            }
          if (cmv[0] > m) {
            m = cmv[0];
            idx = col0 + civ[0];
          }
          float zv[4] = {0.f, 0.f, 0.f, 0.f}, yv[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t packed[16];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float y = ref(x[j], a.alpha);
            y = y > kTopkExpLimit ? kTopkExpLimit : y;  // NaN stays
            x[j] = j < nvalid ? ex2_approx(y) : 0.f;
            zv[j & 3] += x[j];
            yv[j & 3] = fmaf(x[j], y, yv[j & 3]);
          }
          z += (zv[0] + zv[1]) + (zv[2] + zv[3]);
          zy += (yv[0] + yv[1]) + (yv[2] + yv[3]);
#pragma unroll
          for (int j = 0; j < 16; ++j) packed[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
          if (a.write_e) {
            // 64 columns of the warp's 32 rows leave by one TMA store, which cuts them at the chunk's
            // rows and at V. Stores straight from registers (16 bytes in each of 32 rows an
            // instruction) kept the load/store unit 65 % busy and the tensor pipe at 67 %.
#pragma unroll
            for (int q = 0; q < 4; ++q)
              st_shared_v4(smem_u32(stage) + sw128_offset(lane, (c & 1) * 4 + q), packed[4 * q], packed[4 * q + 1],
                           packed[4 * q + 2], packed[4 * q + 3]);
            if ((c & 1) || col0 + 32 >= a.V) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0 && row0 + quarter * 32 < a.rows) {
                tma_store_2d(&tmE, stage, col0 - (c & 1) * 32, row0 + quarter * 32);
                tma_store_commit();
              }
            }
          }
          __syncwarp();  // the tensor-memory loads take the whole warp
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[b]), 0));
      }
      if (live) {
        const int64_t o = static_cast<int64_t>(2 * split + half) * a.part_ld + crow;
        a.part_z[o] = z;
        a.part_y[o] = zy;
        a.part_m[o] = m;
        a.part_i[o] = idx;
        if (!a.second && top >= 0) {
          atomicMax(&a.rowmax[a.c0 + crow], topk_max_key(m));
          if (far || ref(m, a.alpha) > kTopkExpLimit) a.again[(a.c0 + crow) / 256] = 1;
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
  }
  __syncthreads();
  cluster_sync_all();  // neither CTA frees TMEM or leaves while the other may still signal it
  if (warp == 1) {
    tc_fence_after();
    tmem_free_pair(tmem, 512);
  }
}

// One warp per row of the chunk: z and the first maximum from the partials (a fixed order), the row's
// kl and agreement, the kept entries of the chunk buffer and the row factor of the gradient.
__global__ void __launch_bounds__(256)
    topk_finish_kernel(const float* __restrict__ part_z, const float* __restrict__ part_y, const float* __restrict__ part_m,
                       const int* __restrict__ part_i, int parts, int64_t part_ld, int rows, int c0, int k, float alpha,
                       float T, const __nv_bfloat16* __restrict__ student, const __nv_bfloat16* __restrict__ W, int D,
                       const int* __restrict__ trow, const float* __restrict__ top_logit,
                       const unsigned* __restrict__ rowmax, const int* __restrict__ sid,
                       const float* __restrict__ slogq, const int* __restrict__ top_id,
                       const float* __restrict__ mass, const float* __restrict__ kept,
                       const float* __restrict__ row_weight, float* __restrict__ kl_rows, uint8_t* __restrict__ agree,
                       __nv_bfloat16* __restrict__ e, int64_t lde, float* __restrict__ scale) {
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  griddep_launch_dependents();
  griddep_wait();  // launched as a programmatic dependent
  if (r >= rows) return;
  const int64_t g = c0 + r;
  float z = 0.f, zy = 0.f, m = -INFINITY;
  int at = INT_MAX;
  for (int s = lane; s < parts; s += 32) {
    z += part_z[s * part_ld + r];
    zy += part_y[s * part_ld + r];
    const float pm = part_m[s * part_ld + r];
    const int pi = part_i[s * part_ld + r];
    if (pm > m || (pm == m && pi < at)) {
      m = pm;
      at = pi;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, o);
    zy += __shfl_xor_sync(0xffffffffu, zy, o);
    const float om = __shfl_xor_sync(0xffffffffu, m, o);
    const int oi = __shfl_xor_sync(0xffffffffu, at, o);
    if (om > m || (om == m && oi < at)) {
      m = om;
      at = oi;
    }
  }
  const int t = trow[g], top = t >= 0 ? top_id[t] : -1;
  const float Q = t >= 0 ? mass[t] : 0.f;
  const float logz = logf(z);
  const TopkReference c = topk_reference(top_logit[g], rowmax[g], alpha, top >= 0);
  float kl = 0.f;
  if (top >= 0 && Q != 0.f) {
    const int* id = sid + static_cast<int64_t>(t) * k;
    const float* lq = slogq + static_cast<int64_t>(t) * k;
    float qy = 0.f, first = -INFINITY;  // sum of q_j times its exponent; the swept logit at the first id
    for (int j = lane; j < k; j += 32) {
      const int i = id[j];
      if (i == INT_MAX) continue;
      const float x = kept[static_cast<int64_t>(r) * k + j], y = c(x, alpha);
      if (i == top) first = x;
      const float q = expf(lq[j]);
      if (q != 0.f) {
        kl += q * (lq[j] - (y * kLn2 - logz));
        qy += q * y;
      }
      if (e == nullptr || (j > 0 && id[j - 1] == i)) continue;
      float all = q;  // an id kept twice counts with its whole mass
      for (int o = j + 1; o < k && id[o] == i; ++o) all += expf(lq[o]);
      e[r * lde + i] = __float2bfloat16_rn(ex2_approx(y > kTopkExpLimit ? kTopkExpLimit : y) - (all / Q) * z);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      kl += __shfl_xor_sync(0xffffffffu, kl, o);
      qy += __shfl_xor_sync(0xffffffffu, qy, o);
      first = fmaxf(first, __shfl_xor_sync(0xffffffffu, first, o));
    }
    if (at != INT_MAX) {
      // what the sweep's sums cut off (see the top of this file): at most a unit of fp32 every 16
      // products. More is no cut but logits that cancel, or NaN, and says nothing about the others.
      const float exact = at == top ? top_logit[g] : topk_dot(student + g * D, W + static_cast<int64_t>(at) * D, D);
      const float delta = ((exact - m) * m + (top_logit[g] - first) * first) / (m * m + first * first);
      const float add = fabsf(delta) <= static_cast<float>(D) * 0x1p-27f ? delta * kLn2 * (Q * (zy / z) - qy) : 0.f;
      if (fabsf(add) < INFINITY) kl += add;
    }
  }
  if (lane == 0) {
    kl_rows[g] = kl;
    agree[g] = top >= 0 && top == at;
    // a row of padding has no reference near its logits, so its z may be 0 (or anything)
    scale[r] = Q == 0.f ? 0.f : (row_weight ? row_weight[g] : 1.f) / T * (Q / z);
  }
}

// ------------------------------------------------------------------------------------------------
// Host orchestration
// ------------------------------------------------------------------------------------------------

struct TopkKlPlan {
  int64_t chunk, Vp;
  int splits;  // most vocabulary ranges of a chunk's sweep
  size_t off_buf, off_gemm, gemm_bytes;
  size_t off_sid, off_logq, off_top, off_mass, off_trow, off_logit, off_rowmax, off_again, off_kept, off_part, off_scale;
  size_t total;
};

// n, V and d up to 2^30: loops step past them in 32 bits.
inline bool topk_kl_sizes_ok(int64_t n, int64_t m, int64_t V, int64_t D, int64_t k) {
  return n >= 0 && m >= 0 && V >= 1 && D >= 1 && k >= 1 && k <= kTopkKlMaxK && n <= (1ll << 30) && m < (1ll << 31) &&
         V <= (1ll << 30) && D <= (1ll << 30);
}

// The chunk buffer holds fp32 logits (fp32 rows) or bf16 exponentials of p.chunk rows.
inline TopkKlPlan topk_kl_plan(int64_t n, int64_t m, int64_t V, int64_t D, int64_t k, int64_t chunk_rows, int dtype) {
  TopkKlPlan p{};
  const int64_t tile = dtype == ORTHRUS_BF16 ? 256 : 1;
  const int64_t chunk = std::min<int64_t>(chunk_rows <= 0 ? 4096 : chunk_rows, std::max<int64_t>(n, 1));
  p.chunk = ceil_div(chunk, tile) * tile;
  p.Vp = ceil_div(V, 8) * 8;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = align_up(off + bytes, 256);
    return o;
  };
  p.off_buf = take(static_cast<size_t>(p.chunk) * p.Vp * (dtype == ORTHRUS_BF16 ? 2 : 4));
  if (dtype == ORTHRUS_BF16) {
    // a short last chunk has fewer tiles and may split deeper: the larger of the two
    p.gemm_bytes = std::max(gemm2_rowscale_ws_bytes(std::min(n, p.chunk), D, V),
                            n % p.chunk ? gemm2_rowscale_ws_bytes(n % p.chunk, D, V) : size_t(0));
    p.splits = static_cast<int>(std::min<int64_t>(kTopkMaxSplits, ceil_div(V, 256)));
    p.off_sid = take(static_cast<size_t>(m) * k * 4);
    p.off_logq = take(static_cast<size_t>(m) * k * 4);
    p.off_top = take(static_cast<size_t>(m) * 4);
    p.off_mass = take(static_cast<size_t>(m) * 4);
    p.off_trow = take(static_cast<size_t>(n) * 4);
    p.off_logit = take(static_cast<size_t>(n) * 4);
    p.off_rowmax = take(static_cast<size_t>(n) * 4);
    p.off_again = take(static_cast<size_t>(ceil_div(n, 256)) * 4);
    p.off_kept = take(static_cast<size_t>(p.chunk) * k * 4);
    p.off_part = take(static_cast<size_t>(p.chunk) * 2 * p.splits * 16);
    p.off_scale = take(static_cast<size_t>(p.chunk) * 4);
  } else {
    for (int64_t rows : {std::min(n, p.chunk), n % p.chunk})  // a short last chunk may split deeper
      if (rows > 0) p.gemm_bytes = std::max({p.gemm_bytes, f32_plan(rows, V, D).bytes, f32_plan(rows, D, V).bytes});
  }
  p.off_gemm = take(p.gemm_bytes);
  p.total = off;
  return p;
}

struct TopkKlCall {
  int64_t n, m;
  int k;
  const float* values;
  const int64_t *ids, *index;
  const float *teacher_lse, *row_weight;
  int64_t V, D;
  float T;
  float* kl_rows;
  uint8_t* agree;
};

inline int topk_kl_rows_f32(const TopkKlCall& a, const TopkKlPlan& p, const float* student, const float* W, float* grad,
                            uint8_t* ws, cudaStream_t stream) {
  float* buf = reinterpret_cast<float*>(ws + p.off_buf);
  void* gws = ws + p.off_gemm;
  for (int64_t c0 = 0; c0 < a.n; c0 += p.chunk) {
    const int64_t rows = std::min<int64_t>(p.chunk, a.n - c0);
    int rc = f32_product<false>(student + c0 * a.D, a.D, W, a.D, buf, p.Vp, rows, a.V, a.D, gws, p.gemm_bytes, stream);
    if (rc != ORTHRUS_OK) return rc;
    topk_kl_rows_kernel<<<static_cast<unsigned>(rows), kTopkKlThreads, 0, stream>>>(
        buf, p.Vp, static_cast<int>(c0), static_cast<int>(a.V), a.values, a.ids, a.k, a.m, a.index, a.teacher_lse,
        a.row_weight, a.T, a.kl_rows, a.agree, grad ? buf : nullptr, p.Vp);
    ORTHRUS_CHECK_LAUNCH();
    if (grad == nullptr) continue;
    rc = f32_product<true>(buf, p.Vp, W, a.D, grad + c0 * a.D, a.D, rows, a.D, a.V, gws, p.gemm_bytes, stream);
    if (rc != ORTHRUS_OK) return rc;
  }
  return ORTHRUS_OK;
}

inline int topk_exp_launch(const CUtensorMap& th, const CUtensorMap& tw, const CUtensorMap& te, const TopkExpArgs& a,
                           cudaStream_t stream) {
  ORTHRUS_CHECK_CUDA(ensure_smem(topk_exp_kernel, TopkExpTile::SMEM));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min(a.units, num_sms() / 2)));
  cfg.blockDim = dim3(TopkExpTile::THREADS);
  cfg.dynamicSmemBytes = TopkExpTile::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  ORTHRUS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, topk_exp_kernel, th, tw, te, a));
  ORTHRUS_CHECK_LAUNCH();
  return ORTHRUS_OK;
}

inline int topk_kl_rows_bf16(const TopkKlCall& a, const TopkKlPlan& p, const __nv_bfloat16* student,
                             const __nv_bfloat16* W, __nv_bfloat16* grad, uint8_t* ws, cudaStream_t stream) {
  auto* e = reinterpret_cast<__nv_bfloat16*>(ws + p.off_buf);
  auto f = [&](size_t off) { return reinterpret_cast<float*>(ws + off); };
  auto i = [&](size_t off) { return reinterpret_cast<int*>(ws + off); };
  const float alpha = static_cast<float>(1.4426950408889634 / a.T);
  const int D = static_cast<int>(a.D), V = static_cast<int>(a.V);
  topk_teacher_kernel<<<static_cast<unsigned>(a.m), 128, 0, stream>>>(a.values, a.ids, a.k, V, a.T, a.teacher_lse,
                                                                      i(p.off_sid), f(p.off_logq), i(p.off_top),
                                                                      f(p.off_mass));
  ORTHRUS_CHECK_LAUNCH();
  auto* rowmax = reinterpret_cast<unsigned*>(ws + p.off_rowmax);
  ORTHRUS_CHECK_CUDA(launch_pdl(topk_student_kernel, dim3(static_cast<unsigned>(ceil_div(a.n, 8))), dim3(256), 0, stream,
                                student, W, a.n, a.m, D, a.index, static_cast<const int*>(i(p.off_top)),
                                i(p.off_trow), f(p.off_logit), rowmax, i(p.off_again)));
  ORTHRUS_CHECK_LAUNCH();
  CUtensorMap th, tw, te{};
  if (!make_tmap_2d_bf16(&th, student, a.D, a.n, a.D, 64, 128)) return ORTHRUS_ECUDA;
  if (!make_tmap_2d_bf16(&tw, W, a.D, a.V, a.D, 64, 128)) return ORTHRUS_ECUDA;
  TopkExpArgs x{};
  x.V = V;
  x.D = D;
  x.k = a.k;
  x.vtiles = static_cast<int>(ceil_div(a.V, 256));
  x.alpha = alpha;
  x.trow = i(p.off_trow);
  x.top_logit = f(p.off_logit);
  x.top_id = i(p.off_top);
  x.rowmax = rowmax;
  x.again = i(p.off_again);
  x.sid = i(p.off_sid);
  x.kept = f(p.off_kept);
  const size_t part = static_cast<size_t>(p.chunk) * 2 * p.splits;
  x.part_z = f(p.off_part);
  x.part_y = x.part_z + part;
  x.part_m = x.part_y + part;
  x.part_i = reinterpret_cast<int*>(x.part_m + part);
  x.part_ld = p.chunk;
  x.write_e = grad != nullptr;
  for (int64_t c0 = 0; c0 < a.n; c0 += p.chunk) {
    x.rows = static_cast<int>(std::min<int64_t>(p.chunk, a.n - c0));
    x.c0 = static_cast<int>(c0);
    x.rtiles = static_cast<int>(ceil_div(x.rows, 256));
    x.tiles_per_split =
        static_cast<int>(ceil_div(x.vtiles, pick_splits(x.rtiles, x.vtiles, num_sms() / 2, p.splits)));
    const int splits = static_cast<int>(ceil_div(x.vtiles, x.tiles_per_split));
    x.units = x.rtiles * splits;
    x.second = false;
    if (grad && !make_tmap_2d_bf16(&te, e, a.V, x.rows, p.Vp, 64, 32)) return ORTHRUS_ECUDA;
    int rc = topk_exp_launch(th, tw, te, x, stream);
    if (rc != ORTHRUS_OK) return rc;
    x.second = true;
    rc = topk_exp_launch(th, tw, te, x, stream);
    if (rc != ORTHRUS_OK) return rc;
    ORTHRUS_CHECK_CUDA(launch_pdl(
        topk_finish_kernel, dim3(static_cast<unsigned>(ceil_div(x.rows, 8))), dim3(256), 0, stream,
        static_cast<const float*>(x.part_z), static_cast<const float*>(x.part_y), static_cast<const float*>(x.part_m),
        static_cast<const int*>(x.part_i), 2 * splits, x.part_ld, x.rows, x.c0, a.k, alpha, a.T, student, W, D, x.trow,
        x.top_logit, static_cast<const unsigned*>(rowmax), x.sid, static_cast<const float*>(f(p.off_logq)), x.top_id,
        static_cast<const float*>(f(p.off_mass)), static_cast<const float*>(x.kept), a.row_weight, a.kl_rows, a.agree,
        grad ? e : nullptr, p.Vp, f(p.off_scale)));
    ORTHRUS_CHECK_LAUNCH();
    if (grad == nullptr) continue;
    rc = gemm2_rowscale_impl(e, p.Vp, W, grad + c0 * a.D, f(p.off_scale), x.rows, a.D, a.V, ws + p.off_gemm,
                             p.gemm_bytes, stream);
    if (rc != ORTHRUS_OK) return rc;
  }
  return ORTHRUS_OK;
}

template <typename E>
int lmhead_topk_kl_fwd_impl(const E* student, const E* weight, const TopkKlCall& a, const int64_t* offsets,
                            int num_offsets, float* total, E* grad, float* kl_by_offset, int64_t* agree_by_offset,
                            int64_t chunk_rows, void* ws_raw, size_t ws_bytes, cudaStream_t stream) {
  constexpr bool kBf16 = sizeof(E) == 2;
  ORTHRUS_CHECK_ARG(topk_kl_sizes_ok(a.n, a.m, a.V, a.D, a.k));
  ORTHRUS_CHECK_ARG(a.T >= 1e-30f && a.T <= 1e30f);
  ORTHRUS_CHECK_ARG(weight && total);
  ORTHRUS_CHECK_ARG(a.n == 0 || (student && a.values && a.ids && a.kl_rows && a.agree && a.m >= 1));
  ORTHRUS_CHECK_ARG(a.index != nullptr || a.n <= a.m);
  ORTHRUS_CHECK_ARG(offsets == nullptr || (kl_by_offset && agree_by_offset && num_offsets > 0));
  if (kBf16) ORTHRUS_CHECK_ARG(a.D % 8 == 0 && aligned16(student) && aligned16(weight) && (!grad || aligned16(grad)));
  const TopkKlPlan p = topk_kl_plan(a.n, a.m, a.V, a.D, a.k, chunk_rows, kBf16 ? ORTHRUS_BF16 : ORTHRUS_F32);
  if (ws_raw == nullptr || ws_bytes < p.total) return ORTHRUS_EWORKSPACE;
  ORTHRUS_CHECK_ARG(aligned16(ws_raw));
  if (a.n == 0) {
    ORTHRUS_CHECK_CUDA(cudaMemsetAsync(total, 0, sizeof(float), stream));
    if (kl_by_offset && agree_by_offset) {  // an empty offsets array may be NULL
      ORTHRUS_CHECK_CUDA(cudaMemsetAsync(kl_by_offset, 0, num_offsets * sizeof(float), stream));
      ORTHRUS_CHECK_CUDA(cudaMemsetAsync(agree_by_offset, 0, num_offsets * sizeof(int64_t), stream));
    }
    return ORTHRUS_OK;
  }
  int rc;
  if constexpr (kBf16)
    rc = topk_kl_rows_bf16(a, p, student, weight, grad, static_cast<uint8_t*>(ws_raw), stream);
  else
    rc = topk_kl_rows_f32(a, p, student, weight, grad, static_cast<uint8_t*>(ws_raw), stream);
  if (rc != ORTHRUS_OK) return rc;
  lmhead_finalize_kernel<<<1, 1024, 0, stream>>>(a.kl_rows, a.agree, a.row_weight, offsets, a.n, num_offsets, total,
                                                 kl_by_offset, agree_by_offset);
  ORTHRUS_CHECK_LAUNCH();
  return ORTHRUS_OK;
}

}  // namespace orthrus
