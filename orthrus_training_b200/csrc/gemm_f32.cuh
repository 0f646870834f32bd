// fp32 products of the distillation loss's exact path: C[M, N] = A[M, K] B with B given as [N, K] rows (the
// logits) or [K, N] rows (the gradient), any sizes and pitches.
//
// Bound by the FMA pipes for many rows and by latency for few (90 rows x 1024 entries x 256: 24 MFMA, a
// microsecond of work). A CTA of 16 x 16 threads holds a tile of (16 R)^2 sums in registers, R x R a thread,
// and goes through K in chunks of 16: the next chunk's elements are loaded into registers while this one's
// are multiplied out of shared memory (two buffers, one barrier a chunk). The larger the tile the
// fewer shared-memory reads a product takes (2 R for R^2); the smaller, the more SMs a small problem
// fills, so R is the largest of 8, 4 and 2 with a tile for three SMs in four, counting parts of K of 128 or
// more, which are summed in order by a second launch. Measured, us for the logits / the gradient with R =
// 2, 4 and 8: 90 x 1024 x 256: 10 / 12, 13 / 14, 24 / 25; 300 x 4000 x 256: 43 / 119, 33 / 41, 37 / 35;
// 600 x 8000 x 512: 289 / 426, 171 / 458, 193 / 156 (32 TFLOP/s); 2000 x 32000 x 1024: 7287 / 7319,
// 3947 / 4776, 3506 / 4015 (37 and 33 TFLOP/s). What bounds the large ones is
// the issue of FMAs beside one vector load of shared memory per 16.
#pragma once

#include "host_common.h"
#include "sm100.cuh"

namespace orthrus {

constexpr int kF32Chunk = 16;

template <int R, bool B_KN>
__global__ void __launch_bounds__(256)
    f32_product_kernel(const float* __restrict__ A, int64_t lda, const float* __restrict__ B, int64_t ldb,
                       float* __restrict__ C, int64_t ldc, float* __restrict__ part, int M, int N, int K, int tiles_m,
                       int k_per_split) {
  constexpr int TILE = 16 * R, VEC = R < 4 ? R : 4, QUADS = R / VEC;
  __shared__ __align__(16) float sA[2][kF32Chunk][TILE + 4];
  __shared__ __align__(16) float sB[2][kF32Chunk][TILE + 4];
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int m0 = static_cast<int>(blockIdx.x % tiles_m) * TILE;
  const int n0 = static_cast<int>(blockIdx.x / tiles_m) * TILE;
  const int k0 = static_cast<int>(blockIdx.y) * k_per_split, k1 = min(K, k0 + k_per_split);
  float fa[R], fb[R];  // a chunk's elements of this thread
  auto fetch = [&](int kk) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int k = kk + tx, m = m0 + ty + 16 * i;
      fa[i] = m < M && k < k1 ? A[static_cast<int64_t>(m) * lda + k] : 0.f;
      if constexpr (B_KN) {
        const int kb = kk + (tid + 256 * i) / TILE, n = n0 + (tid + 256 * i) % TILE;
        fb[i] = n < N && kb < k1 ? B[static_cast<int64_t>(kb) * ldb + n] : 0.f;
      } else {
        const int n = n0 + ty + 16 * i;
        fb[i] = n < N && k < k1 ? B[static_cast<int64_t>(n) * ldb + k] : 0.f;
      }
    }
  };
  float acc[R][R] = {};
  fetch(k0);
  int buf = 0;
  for (int kk = k0; kk < k1; kk += kF32Chunk, buf ^= 1) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      sA[buf][tx][ty + 16 * i] = fa[i];
      if constexpr (B_KN) sB[buf][(tid + 256 * i) / TILE][(tid + 256 * i) % TILE] = fb[i];
      else sB[buf][tx][ty + 16 * i] = fb[i];
    }
    __syncthreads();  // the other buffer's readers are behind the barrier before
    if (kk + kF32Chunk < k1) fetch(kk + kF32Chunk);
#pragma unroll
    for (int k = 0; k < kF32Chunk; ++k) {
      float a[R], b[R];
#pragma unroll
      for (int q = 0; q < QUADS; ++q)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {  // neighbouring elements: one vector load a quad
          a[q * VEC + e] = sA[buf][k][q * 64 + ty * VEC + e];
          b[q * VEC + e] = sB[buf][k][q * 64 + tx * VEC + e];
        }
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
  }
  float* out = part ? part + static_cast<int64_t>(blockIdx.y) * M * N : C;
  const int64_t pitch = part ? N : ldc;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int m = m0 + (i / VEC) * 64 + ty * VEC + i % VEC;
    if (m >= M) continue;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int n = n0 + (j / VEC) * 64 + tx * VEC + j % VEC;
      if (n < N) out[m * pitch + n] = acc[i][j];
    }
  }
}

// C = the sum of `splits` partial products, in their order.
__global__ void __launch_bounds__(256)
    f32_join_kernel(const float* __restrict__ part, float* __restrict__ C, int64_t ldc, int64_t M, int64_t N, int splits) {
  const int64_t total = M * N;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    float sum = part[i];
    for (int s = 1; s < splits; ++s) sum += part[s * total + i];
    C[i / N * ldc + i % N] = sum;
  }
}

struct F32Plan {
  int R, splits, per_split;
  int64_t tiles_m, tiles;
  size_t bytes;  // of the partial products
};

inline F32Plan f32_plan(int64_t M, int64_t N, int64_t K) {
  F32Plan p{};
  for (p.R = 8;; p.R /= 2) {
    p.tiles_m = ceil_div(M, 16 * p.R);
    p.tiles = p.tiles_m * ceil_div(N, 16 * p.R);
    p.splits = static_cast<int>(std::max<int64_t>(1, std::min(K / 128, num_sms() / p.tiles)));
    if (p.R == 2 || p.tiles * p.splits * 4 >= 3 * num_sms()) break;
  }
  p.per_split = static_cast<int>(ceil_div(ceil_div(K, p.splits), kF32Chunk) * kF32Chunk);
  p.splits = static_cast<int>(ceil_div(K, p.per_split));
  p.bytes = p.splits > 1 ? static_cast<size_t>(p.splits) * M * N * sizeof(float) : 0;
  return p;
}

template <bool B_KN>
int f32_product(const float* A, int64_t lda, const float* B, int64_t ldb, float* C, int64_t ldc, int64_t M, int64_t N,
                int64_t K, void* ws, size_t ws_bytes, cudaStream_t stream) {
  const F32Plan p = f32_plan(M, N, K);
  ORTHRUS_CHECK_ARG(p.tiles < (1ll << 31));
  if (p.bytes > ws_bytes) return ORTHRUS_EWORKSPACE;
  float* part = p.splits > 1 ? static_cast<float*>(ws) : nullptr;
  auto kernel = p.R == 8 ? f32_product_kernel<8, B_KN> : p.R == 4 ? f32_product_kernel<4, B_KN> : f32_product_kernel<2, B_KN>;
  kernel<<<dim3(static_cast<unsigned>(p.tiles), p.splits), 256, 0, stream>>>(
      A, lda, B, ldb, C, ldc, part, static_cast<int>(M), static_cast<int>(N), static_cast<int>(K),
      static_cast<int>(p.tiles_m), p.per_split);
  ORTHRUS_CHECK_LAUNCH();
  if (part) {
    const int64_t blocks = std::min<int64_t>(ceil_div(M * N, 256), 8 * num_sms());
    f32_join_kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(part, C, ldc, M, N, p.splits);
    ORTHRUS_CHECK_LAUNCH();
  }
  return ORTHRUS_OK;
}

}  // namespace orthrus
