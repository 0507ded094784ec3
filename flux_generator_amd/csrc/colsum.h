// Second stage of a column sum in a fixed order: float32 partial rows part[G][n][K][D] -> out_k[G][D] for k < K <= 2.
// A block owns 64 columns of one group's k; its 16 waves take the partial rows n = wave, wave + 16, .. and are added in wave order.
#pragma once
#include "elem.h"

namespace {

template <int T>
__global__ __launch_bounds__(1024) void colsum_final_kernel(const float* part, int64_t n, int K, int D, void* out0, void* out1) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = blockIdx.y, k = blockIdx.z, col = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (col < D) {
    const float* p = part + ((int64_t)g * n * K + k) * D + col;
    const int64_t step = (int64_t)K * D;
#pragma unroll 8
    for (int64_t i = w; i < n; i += 16) s += p[i * step];
  }
  lds[w][lane] = s;
  __syncthreads();
  if (w == 0 && col < D) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][lane];
    Elem<T>::put((typename Elem<T>::type*)(k ? out1 : out0) + (int64_t)g * D + col, s);
  }
}

void launch_colsum_final(const float* part, int64_t n, int64_t G, int K, int D, void* out0, void* out1, int dtype, hipStream_t st) {
  const dim3 grid((D + 63) / 64, (unsigned)G, K);
  if (dtype == 0) hipLaunchKernelGGL((colsum_final_kernel<0>), grid, dim3(1024), 0, st, part, n, K, D, out0, out1);
  else if (dtype == 1) hipLaunchKernelGGL((colsum_final_kernel<1>), grid, dim3(1024), 0, st, part, n, K, D, out0, out1);
  else hipLaunchKernelGGL((colsum_final_kernel<2>), grid, dim3(1024), 0, st, part, n, K, D, out0, out1);
}

}  // namespace
