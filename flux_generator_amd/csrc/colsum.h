// Second stage of a column sum in a fixed order: float32 partial rows part[G][n][K][D] -> out_k[G][D] for k < K <= 2.
// A block owns 64 columns of one group's k; its 16 waves take the partial rows n = wave, wave + 16, .. and are added in wave order.
// Columns of another matrix can be added up in the same launch (Extra: rows of T, or float32 partial rows): one launch less.
#pragma once
#include "elem.h"

namespace {

struct Extra {
  const void* x;                 // null: none
  void* out;
  int64_t ld, n;
  int D, f32;
};

template <int S, class Load>
DEVINL float column_total(int64_t n, Load load, float (*lds)[64]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float s = 0.f;
#pragma unroll S
  for (int64_t i = w; i < n; i += 16) s += load(i);
  lds[w][lane] = s;
  __syncthreads();
  s = 0.f;
  if (w == 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][lane];
  }
  return s;                      // of the first wave
}

template <int T>
__global__ __launch_bounds__(1024) void colsum_final_kernel(const float* part, int64_t n, int K, int D, void* out0, void* out1, Extra x) {
  typedef typename Elem<T>::type E;
  __shared__ float lds[16][64];
  const int g = blockIdx.y, k = blockIdx.z, col = blockIdx.x * 64 + (threadIdx.x & 63);
  if (k == K) {
    const int c = min(col, x.D - 1);
    const float s = x.f32 ? column_total<8>(x.n, [&](int64_t i) { return ((const float*)x.x)[i * x.ld + c]; }, lds)
                          : column_total<8>(x.n, [&](int64_t i) { return Elem<T>::get((const E*)x.x + i * x.ld + c); }, lds);
    if (threadIdx.x < 64 && col < x.D) Elem<T>::put((E*)x.out + col, s);
    return;
  }
  const float* p = part + ((int64_t)g * n * K + k) * D + min(col, D - 1);
  const int64_t step = (int64_t)K * D;
  const float s = column_total<8>(n, [&](int64_t i) { return p[i * step]; }, lds);
  if (threadIdx.x < 64 && col < D) Elem<T>::put((E*)(k ? out1 : out0) + (int64_t)g * D + col, s);
}

void launch_colsum_final(const float* part, int64_t n, int64_t G, int K, int D, void* out0, void* out1, int dtype, hipStream_t st, Extra x = Extra{}) {
  const dim3 grid(((x.x && x.D > D ? x.D : D) + 63) / 64, (unsigned)G, K + (x.x ? 1 : 0));   // (with an Extra, G is 1)
  if (dtype == 0) hipLaunchKernelGGL((colsum_final_kernel<0>), grid, dim3(1024), 0, st, part, n, K, D, out0, out1, x);
  else if (dtype == 1) hipLaunchKernelGGL((colsum_final_kernel<1>), grid, dim3(1024), 0, st, part, n, K, D, out0, out1, x);
  else hipLaunchKernelGGL((colsum_final_kernel<2>), grid, dim3(1024), 0, st, part, n, K, D, out0, out1, x);
}

}  // namespace
