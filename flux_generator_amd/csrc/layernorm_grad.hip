// LayerNorm with the statistics its gradient needs, and that gradient - for training adapters through the transformer blocks.
//
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh g + b          g = offset + gamma
//   backward  e = dy g, dx = r (e - mean(e) - xh mean(e xh)), dgamma = sum_rows dy xh, dbeta = sum_rows dy
//
// Both are HBM-bound: a row is read once into registers (8-element chunks, chunk c of a row on thread c mod (64 WPR) of the row's
// group, as in norm.hip), statistics are float32 and two-pass over the registers.  gamma / beta are [D], or one vector per
// sample ([B][D], adaLN) - then the reduction of their gradient stops at the sample.  Row starts need only element alignment:
// the 16-byte loads of this chip take any address, so an odd width costs its last chunk's element loads and nothing else.
// The parameter gradient is a two-stage sum in a fixed order: every block adds its rows' contributions in registers and
// writes one float32 partial row, ln_partial_sum_kernel adds those; no atomics, so the result is the same in every run.
#include "../../include/fluxhip.h"
#include "common.h"
#include "elem.h"
#include "colsum.h"

namespace {

struct LnArgs {
  const void *x, *dy, *gamma, *beta;
  void *y, *dgamma, *dbeta;           // y: forward result, or dx
  float *mean, *rstd, *part;
  int64_t x_bs, x_rs, dy_bs, dy_rs;   // element strides of sample / row
  int64_t T, p_bs;                    // rows per sample; elements between the samples' parameter vectors (0: shared)
  int D, p_f32, direct;               // direct: one block sees every row behind a gradient vector and writes it, no partial rows
  float eps, offset;
};

// sum over the WPR waves that share a row; red: two slots of 4 floats, used in turn (a slot is rewritten only behind the next
// barrier, which every reader of it has passed)
template <int WPR>
DEVINL float row_sum(float v, float (*red)[4], int& turn) {
  v = row16_sum(v);
  const int i = __builtin_bit_cast(int, v);
  v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 0)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 16)) +
      __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 32)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 48));
  if constexpr (WPR == 1) return v;
  const int s = turn;
  turn ^= 1;
  if ((threadIdx.x & 63) == 0) red[s][threadIdx.x >> 6] = v;
  __syncthreads();
  return red[s][0] + red[s][1] + red[s][2] + red[s][3];
}

template <int T, int NCH, int NT>
DEVINL void load_row(const typename Elem<T>::type* p, int tr, int D, float (&v)[NCH][8]) {
#pragma unroll
  for (int i = 0; i < NCH; ++i) Elem<T>::load8(p, (tr + i * NT) * 8, D, v[i]);
}

// parameters are the tensors' own type or float32
template <int T, int NCH, int NT>
DEVINL void load_param(const void* p, int64_t off, int f32, int tr, int D, float (&v)[NCH][8], float dflt, float add) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      for (int j = 0; j < 8; ++j) v[i][j] = dflt;
    return;
  }
  if (f32) load_row<2, NCH, NT>((const float*)p + off, tr, D, v);
  else load_row<T, NCH, NT>((const typename Elem<T>::type*)p + off, tr, D, v);
#pragma unroll
  for (int i = 0; i < NCH; ++i)
    for (int j = 0; j < 8; ++j) v[i][j] += add;
}

template <int T, int WPR, int NCH>
__global__ __launch_bounds__(256) void ln_fwd_kernel(LnArgs a) {
  using E = typename Elem<T>::type;
  constexpr int NT = 64 * WPR, RPB = 4 / WPR;
  __shared__ float red[2][4];
  int turn = 0;
  const int tr = threadIdx.x % NT, sub = threadIdx.x / NT;
  const int64_t b = blockIdx.y;
  float g[NCH][8], be[NCH][8];
  load_param<T, NCH, NT>(a.gamma, b * a.p_bs, a.p_f32, tr, a.D, g, 1.f, a.gamma ? a.offset : 0.f);
  load_param<T, NCH, NT>(a.beta, b * a.p_bs, a.p_f32, tr, a.D, be, 0.f, 0.f);
  const float inv = 1.0f / (float)a.D;
  for (int64_t t0 = (int64_t)blockIdx.x * RPB; t0 < a.T; t0 += (int64_t)gridDim.x * RPB) {
    const int64_t t = t0 + sub;
    if (WPR == 1 && t >= a.T) break;                      // (WPR = 4: one row per block, t < T here; every wave meets the barriers)
    float v[NCH][8];
    load_row<T, NCH, NT>((const E*)a.x + b * a.x_bs + t * a.x_rs, tr, a.D, v);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      for (int j = 0; j < 8; ++j) s += v[i][j];           // elements behind the row's end are zeros
    const float mu = row_sum<WPR>(s, red, turn) * inv;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      for (int j = 0; j < 8; ++j) {
        const float d = v[i][j] - mu;
        q += (tr + i * NT) * 8 + j < a.D ? d * d : 0.f;
      }
    const float r = 1.0f / sqrtf(row_sum<WPR>(q, red, turn) * inv + a.eps);
    const int64_t row = b * a.T + t;
    E* y = (E*)a.y + row * a.D;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float o[8];
      for (int j = 0; j < 8; ++j) o[j] = (v[i][j] - mu) * r * g[i][j] + be[i][j];
      Elem<T>::store8(y, (tr + i * NT) * 8, a.D, o);
    }
    if (tr == 0) {
      a.mean[row] = mu;
      a.rstd[row] = r;
    }
  }
}

// PG: also the parameter gradient: one partial row [2][D] per block, or the gradient itself (a.direct).
template <int T, int WPR, int NCH, bool PG>
__global__ __launch_bounds__(256) void ln_bwd_kernel(LnArgs a) {
  using E = typename Elem<T>::type;
  constexpr int NT = 64 * WPR, RPB = 4 / WPR;
  __shared__ float red[2][4];
  __shared__ float comb[PG && WPR == 1 ? 3 * 64 * NCH * 8 : 1];
  int turn = 0;
  const int tr = threadIdx.x % NT, sub = threadIdx.x / NT;
  const int64_t b = blockIdx.y;
  float g[NCH][8], dg[PG ? NCH : 1][8], db[PG ? NCH : 1][8];
  load_param<T, NCH, NT>(a.gamma, b * a.p_bs, a.p_f32, tr, a.D, g, 1.f, a.gamma ? a.offset : 0.f);
  if constexpr (PG) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      for (int j = 0; j < 8; ++j) dg[i][j] = db[i][j] = 0.f;
  }
  const float inv = 1.0f / (float)a.D;
  for (int64_t t0 = (int64_t)blockIdx.x * RPB; t0 < a.T; t0 += (int64_t)gridDim.x * RPB) {
    const int64_t t = t0 + sub;
    if (WPR == 1 && t >= a.T) break;
    const int64_t row = b * a.T + t;
    float x[NCH][8], d[NCH][8];
    load_row<T, NCH, NT>((const E*)a.x + b * a.x_bs + t * a.x_rs, tr, a.D, x);
    load_row<T, NCH, NT>((const E*)a.dy + b * a.dy_bs + t * a.dy_rs, tr, a.D, d);
    const float mu = a.mean[row], r = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      for (int j = 0; j < 8; ++j) {
        const float xh = (x[i][j] - mu) * r, dy = d[i][j], e = dy * g[i][j];   // dy is zero behind the row's end, so are all sums' terms
        x[i][j] = xh;
        d[i][j] = e;
        s1 += e;
        s2 += e * xh;
        if constexpr (PG) {
          dg[i][j] += dy * xh;
          db[i][j] += dy;
        }
      }
    s1 = row_sum<WPR>(s1, red, turn) * inv;
    s2 = row_sum<WPR>(s2, red, turn) * inv;
    E* dx = (E*)a.y + row * a.D;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float o[8];
      for (int j = 0; j < 8; ++j) o[j] = r * (d[i][j] - s1 - x[i][j] * s2);
      Elem<T>::store8(dx, (tr + i * NT) * 8, a.D, o);
    }
  }
  if constexpr (PG) {
    if constexpr (WPR == 1) {                             // the four waves hold the same columns: add them in wave order
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        auto& v = which ? db : dg;
        __syncthreads();
        if (sub > 0)
          for (int i = 0; i < NCH; ++i)
            for (int j = 0; j < 8; ++j) comb[((sub - 1) * NCH * 8 + i * 8 + j) * 64 + tr] = v[i][j];
        __syncthreads();
        if (sub == 0)
          for (int w = 0; w < 3; ++w)
            for (int i = 0; i < NCH; ++i)
              for (int j = 0; j < 8; ++j) v[i][j] += comb[(w * NCH * 8 + i * 8 + j) * 64 + tr];
      }
      if (sub) return;
    }
    if (a.direct) {
      const int64_t off = b * a.D;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = (tr + i * NT) * 8;
        if (a.p_f32) {
          Elem<2>::store8((float*)a.dgamma + off, c, a.D, dg[i]);
          Elem<2>::store8((float*)a.dbeta + off, c, a.D, db[i]);
        } else {
          Elem<T>::store8((E*)a.dgamma + off, c, a.D, dg[i]);
          Elem<T>::store8((E*)a.dbeta + off, c, a.D, db[i]);
        }
      }
    } else {
      float* part = a.part + ((b * gridDim.x + blockIdx.x) * 2) * (int64_t)a.D;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        Elem<2>::store8(part, (tr + i * NT) * 8, a.D, dg[i]);
        Elem<2>::store8(part + a.D, (tr + i * NT) * 8, a.D, db[i]);
      }
    }
  }
}

// rows too wide for the registers (D > 8192): one block per row, the row is read again for each pass (from L2)
template <int T, bool BWD>
__global__ __launch_bounds__(256) void ln_wide_kernel(LnArgs a) {
  using E = typename Elem<T>::type;
  __shared__ float red[2][4];
  int turn = 0;
  const int64_t b = blockIdx.y;
  const float inv = 1.0f / (float)a.D, off = a.gamma ? a.offset : 0.f;
  auto par = [&](const void* p, int c, float dflt, float add, float (&v)[8]) {
    float w[1][8];
    load_param<T, 1, 256>(p, b * a.p_bs + c, a.p_f32, 0, a.D - c, w, dflt, add);
    for (int j = 0; j < 8; ++j) v[j] = w[0][j];
  };
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const E* x = (const E*)a.x + b * a.x_bs + t * a.x_rs;
    const E* dy = (const E*)a.dy + b * a.dy_bs + t * a.dy_rs;
    const int64_t row = b * a.T + t;
    E* y = (E*)a.y + row * a.D;
    float mu, r, s1 = 0.f, s2 = 0.f, v[8], d[8], g[8], be[8];
    if constexpr (BWD) {
      mu = a.mean[row];
      r = a.rstd[row];
      for (int c = threadIdx.x * 8; c < a.D; c += 2048) {
        Elem<T>::load8(x, c, a.D, v);
        Elem<T>::load8(dy, c, a.D, d);
        par(a.gamma, c, 1.f, off, g);
        for (int j = 0; j < 8; ++j) {
          const float e = d[j] * g[j];
          s1 += e;
          s2 += e * (v[j] - mu) * r;
        }
      }
      s1 = row_sum<4>(s1, red, turn) * inv;
      s2 = row_sum<4>(s2, red, turn) * inv;
    } else {
      float s = 0.f, q = 0.f;
      for (int c = threadIdx.x * 8; c < a.D; c += 2048) {
        Elem<T>::load8(x, c, a.D, v);
        for (int j = 0; j < 8; ++j) s += v[j];
      }
      mu = row_sum<4>(s, red, turn) * inv;
      for (int c = threadIdx.x * 8; c < a.D; c += 2048) {
        Elem<T>::load8(x, c, a.D, v);
        for (int j = 0; j < 8; ++j) q += c + j < a.D ? (v[j] - mu) * (v[j] - mu) : 0.f;
      }
      r = 1.0f / sqrtf(row_sum<4>(q, red, turn) * inv + a.eps);
      if (threadIdx.x == 0) {
        a.mean[row] = mu;
        a.rstd[row] = r;
      }
    }
    for (int c = threadIdx.x * 8; c < a.D; c += 2048) {
      Elem<T>::load8(x, c, a.D, v);
      par(a.gamma, c, 1.f, off, g);
      if constexpr (BWD) {
        Elem<T>::load8(dy, c, a.D, d);
        for (int j = 0; j < 8; ++j) v[j] = r * (d[j] * g[j] - s1 - (v[j] - mu) * r * s2);
      } else {
        par(a.beta, c, 0.f, 0.f, be);
        for (int j = 0; j < 8; ++j) v[j] = (v[j] - mu) * r * g[j] + be[j];
      }
      Elem<T>::store8(y, c, a.D, v);
    }
  }
}
// ... and their parameter gradient: block (column range of 2048, row range, sample), partial rows as above
template <int T>
__global__ __launch_bounds__(256) void ln_wide_param_kernel(LnArgs a) {
  using E = typename Elem<T>::type;
  const int c = (blockIdx.x * 256 + threadIdx.x) * 8;
  const int64_t b = blockIdx.z;
  if (c >= a.D) return;
  float dg[8] = {}, db[8] = {}, v[8], d[8];
  for (int64_t t = blockIdx.y; t < a.T; t += gridDim.y) {
    const int64_t row = b * a.T + t;
    Elem<T>::load8((const E*)a.x + b * a.x_bs + t * a.x_rs, c, a.D, v);
    Elem<T>::load8((const E*)a.dy + b * a.dy_bs + t * a.dy_rs, c, a.D, d);
    const float mu = a.mean[row], r = a.rstd[row];
    for (int j = 0; j < 8; ++j) {
      dg[j] += d[j] * (v[j] - mu) * r;
      db[j] += d[j];
    }
  }
  float* part = a.part + ((b * gridDim.y + blockIdx.y) * 2) * (int64_t)a.D;
  Elem<2>::store8(part, c, a.D, dg);
  Elem<2>::store8(part + a.D, c, a.D, db);
}

// Waves per row and chunks per lane.  Many rows: a wave per row while the row fits 4 chunks a lane (no barrier in the loop);
// few rows: four waves share one, a quarter of the serial work each.
struct Shape { int wpr, nch; };
Shape pick(int64_t rows, int D) {
  const int c = (D + 7) / 8;
  if (c <= 64) return {1, 1};
  if (c <= 256 && rows < 2048) return {4, 1};
  if (c <= 256) return {1, (c + 63) / 64};
  if (c <= 512) return {4, 2};
  if (c <= 1024) return {4, 4};
  return {0, 0};
}
// partial rows per sample: about two blocks a CU in all, and no more than there are row groups
int64_t partials(int64_t B, int64_t T, int D, Shape s) {
  const int64_t rpb = s.wpr == 1 ? 4 : 1, groups = (T + rpb - 1) / rpb;
  if (groups <= 4 && s.wpr) return 1;                     // a handful of rows: one block, no second launch
  int64_t n = 512 / (B < 512 ? B : 512);
  if (!s.wpr) n = 64;
  return n < 1 ? 1 : n < groups ? n : groups;
}

#define LN_DISPATCH(KERNEL, ...)                                              \
  if (s.wpr == 1 && s.nch == 1) KERNEL(1, 1, __VA_ARGS__);                    \
  else if (s.wpr == 1 && s.nch == 2) KERNEL(1, 2, __VA_ARGS__);               \
  else if (s.wpr == 1 && s.nch == 3) KERNEL(1, 3, __VA_ARGS__);               \
  else if (s.wpr == 1) KERNEL(1, 4, __VA_ARGS__);                             \
  else if (s.nch == 1) KERNEL(4, 1, __VA_ARGS__);                             \
  else if (s.nch == 2) KERNEL(4, 2, __VA_ARGS__);                             \
  else KERNEL(4, 4, __VA_ARGS__)

template <int T>
void launch_fwd(const LnArgs& a, int64_t B, hipStream_t st) {
  const Shape s = pick(B * a.T, a.D);
  const int64_t rpb = s.wpr == 1 ? 4 : 1, groups = (a.T + rpb - 1) / rpb, cap = B < 2048 ? 4096 / B : 2;
  const dim3 grid((unsigned)(groups < cap ? groups : cap), (unsigned)B);
  if (!s.wpr) {
    hipLaunchKernelGGL((ln_wide_kernel<T, false>), grid, dim3(256), 0, st, a);
    return;
  }
#define LN_F(W, N, X) hipLaunchKernelGGL((ln_fwd_kernel<T, W, N>), grid, dim3(256), 0, st, a)
  LN_DISPATCH(LN_F, 0);
#undef LN_F
}

template <int T>
void launch_bwd(LnArgs a, int64_t B, hipStream_t st) {
  const Shape s = pick(B * a.T, a.D);
  const bool pg = a.dgamma != nullptr, shared = pg && a.p_bs == 0;
  const int64_t rpb = s.wpr == 1 ? 4 : 1, groups = (a.T + rpb - 1) / rpb, cap = B < 2048 ? 4096 / B : 2;
  const int64_t np = partials(B, a.T, a.D, s), nx = pg && s.wpr ? np : groups < cap ? groups : cap;
  const dim3 grid((unsigned)nx, (unsigned)B);
  a.direct = s.wpr && np == 1 && (B == 1 || !shared);
  if (!s.wpr) {
    hipLaunchKernelGGL((ln_wide_kernel<T, true>), grid, dim3(256), 0, st, a);
    if (pg) hipLaunchKernelGGL((ln_wide_param_kernel<T>), dim3((a.D + 2047) / 2048, (unsigned)np, (unsigned)B), dim3(256), 0, st, a);
  } else if (pg) {
#define LN_B(W, N, PG) hipLaunchKernelGGL((ln_bwd_kernel<T, W, N, PG>), grid, dim3(256), 0, st, a)
    LN_DISPATCH(LN_B, true);
  } else {
    LN_DISPATCH(LN_B, false);
#undef LN_B
  }
  if (pg && !a.direct) {
    const int dt = a.p_f32 ? 2 : T;
    if (shared) launch_colsum_final(a.part, B * np, 1, 2, a.D, a.dgamma, a.dbeta, dt, st);
    else launch_colsum_final(a.part, np, B, 2, a.D, a.dgamma, a.dbeta, dt, st);
  }
}

bool bad_shape(int64_t B, int64_t T, int64_t D, int dtype) {
  return B < 0 || T < 0 || D < 1 || D > (1 << 24) || dtype < 0 || dtype > 2 || B > 65535 || T >= (1ll << 40);
}

}  // namespace

extern "C" int64_t fluxhip_layernorm_grad_ws(int64_t B, int64_t T, int D) {
  if (bad_shape(B, T, D, 0)) return FLUXHIP_EINVAL;
  return B * partials(B, T, D, pick(B * T, D)) * 2 * D * 4;
}

extern "C" int fluxhip_layernorm_stats(const void* x, int64_t x_bs, int64_t x_rs, const void* gamma, const void* beta, int64_t p_bs,
                                       int param_f32, float offset, void* y, float* mean, float* rstd, int64_t B, int64_t T, int D,
                                       float eps, int dtype, void* stream) {
  if (bad_shape(B, T, D, dtype)) return FLUXHIP_EINVAL;
  if (B == 0 || T == 0) return FLUXHIP_OK;
  if (!x || !y || !mean || !rstd || (beta && !gamma)) return FLUXHIP_EINVAL;
  LnArgs a{};
  a.x = x; a.gamma = gamma; a.beta = beta; a.y = y; a.mean = mean; a.rstd = rstd;
  a.x_bs = x_bs; a.x_rs = x_rs; a.T = T; a.p_bs = p_bs; a.D = D; a.p_f32 = param_f32; a.eps = eps; a.offset = offset;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) launch_fwd<0>(a, B, st);
  else if (dtype == 1) launch_fwd<1>(a, B, st);
  else launch_fwd<2>(a, B, st);
  return hipGetLastError() == hipSuccess ? FLUXHIP_OK : FLUXHIP_ELAUNCH;
}

extern "C" int fluxhip_layernorm_grad(const void* dy, int64_t dy_bs, int64_t dy_rs, const void* x, int64_t x_bs, int64_t x_rs,
                                      const float* mean, const float* rstd, const void* gamma, int64_t p_bs, int param_f32, float offset,
                                      void* dx, void* dgamma, void* dbeta, int64_t B, int64_t T, int D, int dtype, void* ws,
                                      int64_t ws_bytes, void* stream) {
  if (bad_shape(B, T, D, dtype)) return FLUXHIP_EINVAL;
  if (B == 0 || T == 0) return FLUXHIP_OK;                 // (the caller owns the zeros of an empty sum)
  if (!dy || !x || !dx || !mean || !rstd || (!dgamma) != (!dbeta)) return FLUXHIP_EINVAL;
  if (dgamma && (!ws || ws_bytes < fluxhip_layernorm_grad_ws(B, T, D))) return FLUXHIP_EINVAL;
  LnArgs a{};
  a.x = x; a.dy = dy; a.gamma = gamma; a.y = dx; a.dgamma = dgamma; a.dbeta = dbeta;
  a.mean = (float*)mean; a.rstd = (float*)rstd; a.part = (float*)ws;
  a.x_bs = x_bs; a.x_rs = x_rs; a.dy_bs = dy_bs; a.dy_rs = dy_rs;
  a.T = T; a.p_bs = p_bs; a.D = D; a.p_f32 = param_f32; a.offset = offset;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) launch_bwd<0>(a, B, st);
  else if (dtype == 1) launch_bwd<1>(a, B, st);
  else launch_bwd<2>(a, B, st);
  return hipGetLastError() == hipSuccess ? FLUXHIP_OK : FLUXHIP_ELAUNCH;
}
