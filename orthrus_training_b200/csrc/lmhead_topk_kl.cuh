// Distillation from a teacher's top logits through the LM head: per student row h with the kept
// teacher logits (v_j, id_j) of its teacher row,
//
//   q_j = softmax over the kept v_j / T      (or exp(v_j / T - lse) with the teacher's normaliser)
//   p   = softmax(W h / T) over the whole vocabulary
//   kl  = sum_j q_j (log q_j - log p_{id_j})          total = sum_r w_r kl_r
//   d total / dh = (w / T) (Q p - q) W                Q = sum_j q_j
//
// The student's normaliser needs every logit, so forward and gradient are two products of
// [n, d] x [d, V]; the teacher costs its k entries per row.
//
// Passes, a chunk of rows at a time: logits = student @ W^T (fp32), a row kernel that turns a row of
// logits into its kl and the difference (w / T) (Q p - q), and grad = difference @ W.
#pragma once

#include "gemm_simt.cuh"
#include "gemm_tc.cuh"
#include "lmhead_kl.cuh"

namespace orthrus {

constexpr int kTopkKlMaxK = 1024;
constexpr int kTopkKlThreads = 512;

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
    sh.logq[j] = live ? v / T : -INFINITY;
    if (live && v > best) {
      best = v;
      at = j;
    }
  }
  tk_block_argmax(best, at, sh);
  top_id = at == INT_MAX ? -1 : sh.id[at];
  float norm;
  if (teacher_lse != nullptr) {
    norm = teacher_lse[t];
  } else {
    float z = 0.f;
    for (int j = threadIdx.x; j < k; j += kTopkKlThreads)
      if (sh.id[j] >= 0) z += expf(sh.logq[j] - best / T);
    norm = best / T + logf(tk_block_sum(z, sh));
  }
  float Q = 0.f;
  for (int j = threadIdx.x; j < k; j += kTopkKlThreads) {
    const float lq = sh.id[j] >= 0 ? sh.logq[j] - norm : -INFINITY;
    sh.logq[j] = lq;
    sh.q[j] = expf(lq);
    Q += sh.q[j];
  }
  return tk_block_sum(Q, sh);
}

// One CTA per row of a chunk: logits [rows, ld] fp32 of student rows c0.. -> kl_rows, agree and, with
// `diff`, the difference (w / T) (Q p - q) in T's type (which may overwrite the logits).
template <typename D>
__global__ void __launch_bounds__(kTopkKlThreads)
    topk_kl_rows_kernel(const float* logits, int64_t ld, int c0, int V, const float* __restrict__ values,
                        const int64_t* __restrict__ ids, int k, int64_t m, const int64_t* __restrict__ index,
                        const float* __restrict__ teacher_lse, const float* __restrict__ row_weight, float T,
                        float* __restrict__ kl_rows, uint8_t* __restrict__ agree, D* diff, int64_t ldd) {
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
  D* d = diff + blockIdx.x * ldd;
  const float scale = w * Q / z;
  for (int i = threadIdx.x; i < V; i += kTopkKlThreads) d[i] = from_f32<D>(scale * expf((x[i] - top) / T));
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int j = threadIdx.x + u * kTopkKlThreads;
    if (j < k && sh.id[j] >= 0) d[sh.id[j]] = from_f32<D>(fix[u]);
  }
}

// ------------------------------------------------------------------------------------------------
// Host orchestration
// ------------------------------------------------------------------------------------------------

struct TopkKlPlan {
  int64_t chunk, Vp;
  size_t off_logits, off_diff, off_gemm, gemm_bytes, total;
};

inline TopkKlPlan topk_kl_plan(int64_t n, int64_t V, int64_t D, int64_t chunk_rows, int dtype) {
  TopkKlPlan p{};
  p.chunk = std::min<int64_t>(chunk_rows <= 0 ? 4096 : chunk_rows, std::max<int64_t>(n, 1));
  p.Vp = ceil_div(V, 8) * 8;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = align_up(off + bytes, 256);
    return o;
  };
  p.off_logits = take(static_cast<size_t>(p.chunk) * p.Vp * 4);
  p.off_diff = dtype == ORTHRUS_BF16 ? take(static_cast<size_t>(p.chunk) * p.Vp * 2) : p.off_logits;
  p.gemm_bytes = dtype == ORTHRUS_BF16 ? std::max(gemm_ws_bytes(p.chunk, V, D), gemm_ws_bytes(p.chunk, D, V))
                                       : std::max(simt_ws_bytes(p.chunk, V, D), simt_ws_bytes(p.chunk, D, V));
  p.off_gemm = take(p.gemm_bytes);
  p.total = off;
  return p;
}

template <typename E>
int lmhead_topk_kl_fwd_impl(const E* student, int64_t n, const float* values, const int64_t* ids, int64_t m, int k,
                            const int64_t* index, const float* teacher_lse, const E* weight, int64_t V, int64_t D,
                            float temperature, const float* row_weight, const int64_t* offsets, int num_offsets,
                            float* total, float* kl_rows, uint8_t* agree, E* grad, float* kl_by_offset,
                            int64_t* agree_by_offset, int64_t chunk_rows, void* ws_raw, size_t ws_bytes,
                            cudaStream_t stream) {
  constexpr bool kBf16 = sizeof(E) == 2;
  ORTHRUS_CHECK_ARG(n >= 0 && m >= 0 && V >= 1 && D >= 1 && k >= 1 && k <= kTopkKlMaxK && temperature > 0.f);
  ORTHRUS_CHECK_ARG(n < (1ll << 31) && V < (1ll << 31) && D < (1ll << 31));
  ORTHRUS_CHECK_ARG(weight && total && (n == 0 || (student && values && ids && kl_rows && agree && m >= 1)));
  ORTHRUS_CHECK_ARG(index != nullptr || n <= m);
  ORTHRUS_CHECK_ARG(offsets == nullptr || (kl_by_offset && agree_by_offset && num_offsets > 0));
  if (kBf16) ORTHRUS_CHECK_ARG(D % 8 == 0 && aligned16(student) && aligned16(weight) && (!grad || aligned16(grad)));
  const TopkKlPlan p = topk_kl_plan(n, V, D, chunk_rows, kBf16 ? ORTHRUS_BF16 : ORTHRUS_F32);
  if (ws_raw == nullptr || ws_bytes < p.total) return ORTHRUS_EWORKSPACE;
  if (n == 0) {
    ORTHRUS_CHECK_CUDA(cudaMemsetAsync(total, 0, sizeof(float), stream));
    if (kl_by_offset && agree_by_offset) {  // an empty offsets array may be NULL
      ORTHRUS_CHECK_CUDA(cudaMemsetAsync(kl_by_offset, 0, num_offsets * sizeof(float), stream));
      ORTHRUS_CHECK_CUDA(cudaMemsetAsync(agree_by_offset, 0, num_offsets * sizeof(int64_t), stream));
    }
    return ORTHRUS_OK;
  }
  uint8_t* ws = static_cast<uint8_t*>(ws_raw);
  float* logits = reinterpret_cast<float*>(ws + p.off_logits);
  E* diff = reinterpret_cast<E*>(ws + p.off_diff);
  void* gws = ws + p.off_gemm;
  for (int64_t c0 = 0; c0 < n; c0 += p.chunk) {
    const int64_t rows = std::min<int64_t>(p.chunk, n - c0);
    int rc;
    if constexpr (kBf16)
      rc = gemm_bf16_impl(student + c0 * D, D, weight, D, logits, p.Vp, rows, V, D, 0, 1, gws, p.gemm_bytes, stream);
    else
      rc = gemm_simt_impl<E, false>(student + c0 * D, D, weight, D, logits, p.Vp, rows, V, D, gws, p.gemm_bytes, stream);
    if (rc != ORTHRUS_OK) return rc;
    topk_kl_rows_kernel<E><<<static_cast<unsigned>(rows), kTopkKlThreads, 0, stream>>>(
        logits, p.Vp, static_cast<int>(c0), static_cast<int>(V), values, ids, k, m, index, teacher_lse, row_weight,
        temperature, kl_rows, agree, grad ? diff : nullptr, p.Vp);
    ORTHRUS_CHECK_LAUNCH();
    if (grad != nullptr) {
      if constexpr (kBf16)
        rc = gemm_bf16_impl(diff, p.Vp, weight, D, grad + c0 * D, D, rows, D, V, 1, 0, gws, p.gemm_bytes, stream, false);
      else
        rc = gemm_simt_impl<E, true>(diff, p.Vp, weight, D, grad + c0 * D, D, rows, D, V, gws, p.gemm_bytes, stream);
      if (rc != ORTHRUS_OK) return rc;
    }
  }
  lmhead_finalize_kernel<<<1, 1024, 0, stream>>>(kl_rows, agree, row_weight, offsets, n, num_offsets, total,
                                                 kl_by_offset, agree_by_offset);
  ORTHRUS_CHECK_LAUNCH();
  return ORTHRUS_OK;
}

}  // namespace orthrus
