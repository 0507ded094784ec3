// LayerNorm with the statistics its gradient needs, and that gradient - for training adapters through the transformer blocks.
//
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh g + b          g = offset + gamma
//   backward  e = dy g, dx = r (e - mean(e) - xh mean(e xh)), dgamma = sum_rows dy xh, dbeta = sum_rows dy
//
// Both are HBM-bound: a row is read once into registers (8-element chunks, chunk c of a row on the c-th of its threads, modulo
// their number), statistics are float32 and two-pass over the registers.  gamma / beta are [D], or one vector per
// sample ([B][D], adaLN) - then the reduction of their gradient stops at the sample.  Row starts need only element alignment:
// the 16-byte loads of this chip take any address, so an odd width costs its last chunk's element loads and nothing else.
// The parameter gradient is a two-stage sum in a fixed order: every block adds its rows' contributions in registers and
// writes one float32 partial row, colsum_final_kernel (colsum.h) adds those; no atomics, so the result is the same in every run.
// (Rows are added one after the other: float32 gradients of 231 rows end 1.2e-7 from the exact ones, with pairwise sums 0.9e-7.)
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
  int row_blocks, B;                  // ln_bwd_kernel without PG: blocks behind these add up parameter gradients
  int D, p_f32, direct;               // direct: one block sees every row behind a gradient vector and writes it, no partial rows
  float eps, offset;
};

// blocks of eight waves: a row has NT threads (16, or 1, 2, 4, 8 waves), 512 / NT rows lie side by side
constexpr int WAVES = 8;

// sums (one or two at once) over the NT threads that share a row; red: two slots, used in turn (a slot is rewritten only behind
// the next barrier, which every reader of it has passed)
DEVINL float wave_total(float v) {
  v = row16_sum(v);
  const int i = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 0)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 16)) +
         __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 32)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 48));
}
template <int NT>
DEVINL float2 row_sum2(float a, float b, float2 (*red)[WAVES], int& turn) {
  if constexpr (NT == 16) return make_float2(row16_sum(a), row16_sum(b));
  constexpr int WPR = NT / 64;
  a = wave_total(a);
  b = wave_total(b);
  if constexpr (NT <= 64) return make_float2(a, b);
  const int s = turn, w = threadIdx.x >> 6, w0 = w & ~(WPR - 1);
  turn ^= 1;
  if ((threadIdx.x & 63) == 0) red[s][w] = make_float2(a, b);
  __syncthreads();
  float2 r = red[s][w0];
#pragma unroll
  for (int i = 1; i < WPR; ++i) {
    r.x += red[s][w0 + i].x;
    r.y += red[s][w0 + i].y;
  }
  return r;
}

template <int T, int NCH, int NT, bool FULL>
DEVINL void fetch_row(const typename Elem<T>::type* p, int tr, int D, typename Elem<T>::raw8 (&w)[NCH]) {
#pragma unroll
  for (int i = 0; i < NCH; ++i) Elem<T>::template fetch8<FULL>(p, (tr + i * NT) * 8, D, w[i]);
}
template <int T, int NCH>
DEVINL void open_row(const typename Elem<T>::raw8 (&w)[NCH], float (&v)[NCH][8]) {
#pragma unroll
  for (int i = 0; i < NCH; ++i) Elem<T>::open8(w[i], v[i]);
}

// parameters are the tensors' own type or float32
template <int T, int NCH, int NT>
DEVINL void load_param(const void* p, int64_t off, int f32, int tr, int D, float (&v)[NCH][8], float dflt, float add) {
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (!p) {
      for (int j = 0; j < 8; ++j) v[i][j] = dflt;
    } else {
      if (f32) Elem<2>::load8((const float*)p + off, (tr + i * NT) * 8, D, v[i]);
      else Elem<T>::load8((const typename Elem<T>::type*)p + off, (tr + i * NT) * 8, D, v[i]);
      for (int j = 0; j < 8; ++j) v[i][j] += add;
    }
  }
}

// Both kernels walk rows with a stride of the grid and keep the next row's loads in flight while they reduce this one.  A row
// group without a row left (the last round) repeats the sample's last row and drops what it computes: every wave meets every barrier.
template <int T, int NT, int NCH, bool FULL>
__global__ __launch_bounds__(64 * WAVES, NCH == 1 ? 8 : 4) void ln_fwd_kernel(LnArgs a) {
  using E = typename Elem<T>::type;
  constexpr int RPB = 64 * WAVES / NT;
  __shared__ float2 red[2][WAVES];
  int turn = 0;
  const int tr = threadIdx.x % NT, sub = threadIdx.x / NT;
  const int64_t b = blockIdx.y, step = (int64_t)gridDim.x * RPB;
  const E* xb = (const E*)a.x + b * a.x_bs;
  int64_t t0 = (int64_t)blockIdx.x * RPB;
  typename Elem<T>::raw8 w[NCH];
  fetch_row<T, NCH, NT, FULL>(xb + min(t0 + sub, a.T - 1) * a.x_rs, tr, a.D, w);
  float g[NCH][8], be[NCH][8];
  load_param<T, NCH, NT>(a.gamma, b * a.p_bs, a.p_f32, tr, a.D, g, 1.f, a.gamma ? a.offset : 0.f);
  load_param<T, NCH, NT>(a.beta, b * a.p_bs, a.p_f32, tr, a.D, be, 0.f, 0.f);
  const float inv = 1.0f / (float)a.D;
  for (; t0 < a.T; t0 += step) {
    const int64_t t = t0 + sub;
    float v[NCH][8];
    open_row<T, NCH>(w, v);
    if (t0 + step < a.T) fetch_row<T, NCH, NT, FULL>(xb + min(t + step, a.T - 1) * a.x_rs, tr, a.D, w);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      for (int j = 0; j < 8; ++j) s += v[i][j];           // elements behind the row's end are zeros
    const float mu = row_sum2<NT>(s, 0.f, red, turn).x * inv;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      for (int j = 0; j < 8; ++j) {
        const float d = v[i][j] - mu;
        q += (tr + i * NT) * 8 + j < a.D ? d * d : 0.f;
      }
    const float r = 1.0f / sqrtf(row_sum2<NT>(q, 0.f, red, turn).x * inv + a.eps);
    if (t < a.T) {
      const int64_t row = b * a.T + t;
      E* y = (E*)a.y + row * a.D;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        float o[8];
        for (int j = 0; j < 8; ++j) o[j] = (v[i][j] - mu) * r * g[i][j] + be[i][j];
        Elem<T>::template store8<FULL>(y, (tr + i * NT) * 8, a.D, o);
      }
      if (tr == 0) {
        a.mean[row] = mu;
        a.rstd[row] = r;
      }
    }
  }
}

// dgamma (or dbeta) of 64 columns from the inputs, for few rows: eight waves take every eighth row, added in wave order
template <int T>
DEVINL void param_columns(const LnArgs& a, int block, int64_t sample) {
  using E = typename Elem<T>::type;
  __shared__ float lds[WAVES][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nc = (a.D + 63) / 64, which = block / nc, col = (block - which * nc) * 64 + lane;
  const int c = min(col, a.D - 1);
  float s = 0.f;
  const int64_t b0 = a.p_bs ? sample : 0, b1 = a.p_bs ? sample + 1 : a.B;
  for (int64_t b = b0; b < b1; ++b) {
    const E *x = (const E*)a.x + b * a.x_bs + c, *dy = (const E*)a.dy + b * a.dy_bs + c;
    if (which) {
#pragma unroll 8
      for (int64_t t = w; t < a.T; t += WAVES) s += Elem<T>::get(dy + t * a.dy_rs);
    } else {
#pragma unroll 8
      for (int64_t t = w; t < a.T; t += WAVES)
        s += Elem<T>::get(dy + t * a.dy_rs) * ((Elem<T>::get(x + t * a.x_rs) - a.mean[b * a.T + t]) * a.rstd[b * a.T + t]);
    }
  }
  lds[w][lane] = s;
  __syncthreads();
  if (w || col >= a.D) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) s += lds[i][lane];
  void* out = which ? a.dbeta : a.dgamma;
  if (a.p_f32) ((float*)out)[sample * a.D + col] = s;
  else Elem<T>::put((E*)out + sample * a.D + col, s);
}

// PG: also the parameter gradient: one partial row [2][D] per block, or the gradient itself (a.direct).
template <int T, int NT, int NCH, bool FULL, bool PG>
__global__ __launch_bounds__(64 * WAVES, !PG ? (NCH == 1 ? 6 : 4) : NCH == 1 ? 4 : 2) void ln_bwd_kernel(LnArgs a) {
  using E = typename Elem<T>::type;
  constexpr int RPB = 64 * WAVES / NT;
  __shared__ float2 red[2][WAVES];
  __shared__ float comb[PG ? NCH * 8 * NT * RPB : 1];
  if constexpr (!PG) {
    if ((int)blockIdx.x >= a.row_blocks) {
      if (a.p_bs || blockIdx.y == 0) param_columns<T>(a, blockIdx.x - a.row_blocks, blockIdx.y);
      return;
    }
  }
  int turn = 0;
  const int tr = threadIdx.x % NT, sub = threadIdx.x / NT;
  const int64_t b = blockIdx.y, step = (int64_t)(PG ? gridDim.x : a.row_blocks) * RPB;
  const E *xb = (const E*)a.x + b * a.x_bs, *db_ = (const E*)a.dy + b * a.dy_bs;
  int64_t t0 = (int64_t)blockIdx.x * RPB;
  typename Elem<T>::raw8 wx[NCH], wd[NCH];
  float mu, r;
  auto fetch = [&](int64_t t) {
    t = min(t, a.T - 1);
    fetch_row<T, NCH, NT, FULL>(xb + t * a.x_rs, tr, a.D, wx);
    fetch_row<T, NCH, NT, FULL>(db_ + t * a.dy_rs, tr, a.D, wd);
    mu = a.mean[b * a.T + t];
    r = a.rstd[b * a.T + t];
  };
  fetch(t0 + sub);
  float g[NCH][8], dg[PG ? NCH : 1][8], db[PG ? NCH : 1][8];
  load_param<T, NCH, NT>(a.gamma, b * a.p_bs, a.p_f32, tr, a.D, g, 1.f, a.gamma ? a.offset : 0.f);
  if constexpr (PG) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      for (int j = 0; j < 8; ++j) dg[i][j] = db[i][j] = 0.f;
  }
  const float inv = 1.0f / (float)a.D;
  for (; t0 < a.T; t0 += step) {
    const int64_t t = t0 + sub;
    // a repeated row adds nothing to the parameter sums: zeros in its place (its own values times zero would be NaN where the row
    // holds an infinity)
    const bool on = !PG || t < a.T;
    typename Elem<T>::raw8 cx[NCH], cd[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      cx[i] = on ? wx[i] : typename Elem<T>::raw8{};
      cd[i] = on ? wd[i] : typename Elem<T>::raw8{};
    }
    const float m = on ? mu : 0.f, rs = on ? r : 0.f;
    if (t0 + step < a.T) fetch(t + step);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float x[8], d[8];
      Elem<T>::open8(cx[i], x);
      Elem<T>::open8(cd[i], d);
      for (int j = 0; j < 8; ++j) {
        const float xh = (x[j] - m) * rs, dy = d[j], e = dy * g[i][j];   // dy is zero behind the row's end, so are all sums' terms
        s1 += e;
        s2 += e * xh;
        if constexpr (PG) {
          dg[i][j] += dy * xh;
          db[i][j] += dy;
        }
      }
      if constexpr (T < 2) asm volatile("" : "+v"(cx[i]), "+v"(cd[i]));  // unpack again below: half the registers across the reduction
    }
    const float2 s = row_sum2<NT>(s1, s2, red, turn);
    if (t < a.T) {
      E* dx = (E*)a.y + (b * a.T + t) * a.D;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        float x[8], d[8], o[8];
        Elem<T>::open8(cx[i], x);
        Elem<T>::open8(cd[i], d);
        for (int j = 0; j < 8; ++j) o[j] = rs * (d[j] * g[i][j] - s.x * inv - (x[j] - m) * rs * (s.y * inv));
        Elem<T>::template store8<FULL>(dx, (tr + i * NT) * 8, a.D, o);
      }
    }
  }
  if constexpr (PG) {                                     // the row groups hold the same columns: add them in group order
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      auto& v = which ? db : dg;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        for (int j = 0; j < 8; ++j) comb[((sub * NCH + i) * 8 + j) * NT + tr] = v[i][j];
      __syncthreads();
      if (sub == which % RPB) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          float o[8];
          for (int j = 0; j < 8; ++j) {
            o[j] = 0.f;
            for (int k = 0; k < RPB; ++k) o[j] += comb[((k * NCH + i) * 8 + j) * NT + tr];
          }
          const int c = (tr + i * NT) * 8;
          void* out = which ? a.dbeta : a.dgamma;
          if (!a.direct) Elem<2>::store8(a.part + ((b * gridDim.x + blockIdx.x) * 2 + which) * (int64_t)a.D, c, a.D, o);
          else if (a.p_f32) Elem<2>::store8((float*)out + b * a.D, c, a.D, o);
          else Elem<T>::store8((E*)out + b * a.D, c, a.D, o);
        }
      }
    }
  }
}

// rows too wide for the registers (D > 8192): one block per row, the row is read again for each pass (from L2)
template <int T, bool BWD>
__global__ __launch_bounds__(256) void ln_wide_kernel(LnArgs a) {
  using E = typename Elem<T>::type;
  __shared__ float2 red[2][WAVES];
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
      const float2 t2 = row_sum2<256>(s1, s2, red, turn);
      s1 = t2.x * inv;
      s2 = t2.y * inv;
    } else {
      float s = 0.f, q = 0.f;
      for (int c = threadIdx.x * 8; c < a.D; c += 2048) {
        Elem<T>::load8(x, c, a.D, v);
        for (int j = 0; j < 8; ++j) s += v[j];
      }
      mu = row_sum2<256>(s, 0.f, red, turn).x * inv;
      for (int c = threadIdx.x * 8; c < a.D; c += 2048) {
        Elem<T>::load8(x, c, a.D, v);
        for (int j = 0; j < 8; ++j) q += c + j < a.D ? (v[j] - mu) * (v[j] - mu) : 0.f;
      }
      r = 1.0f / sqrtf(row_sum2<256>(q, 0.f, red, turn).x * inv + a.eps);
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

// Threads per row and chunks per thread.  Few rows, float32, a parameter gradient or a width that cuts a chunk: as many threads as
// have one chunk each - short serial work, and registers stay free for the loads in flight.  Else two or three chunks a lane, which
// leaves fewer idle lanes and fewer barriers.  Measured (us a call on changing operands, several chunks / one): 16384 x 1280 f16
// forward 19.4 / 23.4, dx alone 24.6 / 26.9, with parameter gradient 37.0 / 34.2; 4 x 4096 x 2560 bf16 33.7 / 40.2, 42.3 / 51.9,
// 60.5 / 53.9; 16384 x 1280 float32 32.2 / 30.1, 60.9 / 41.4, 53.7 / 46.5.
struct Shape { int nt, nch; };
Shape pick(int64_t rows, int D, bool f32, bool pg) {
  const int c = (D + 7) / 8;
  const bool several = rows >= 2048 && !f32 && !pg && D % 8 == 0;
  if (c <= 16) return {16, 1};
  if (c <= 64) return {64, 1};
  if (several && c <= 192) return {64, (c + 63) / 64};
  if (c <= 128) return {128, 1};
  if (c <= 256) return {256, 1};
  if (several && c <= 384) return {256, 2};
  if (c <= 512) return {512, 1};
  if (c <= 1024) return {512, 2};
  return {0, 0};
}
int64_t row_groups(int64_t T, Shape s) {
  const int64_t rpb = s.nt == 0 ? 1 : 64 * WAVES / s.nt;
  return (T + rpb - 1) / rpb;
}
// blocks per sample: `most` in all, every block the same number of rounds (but the last)
int64_t even_blocks(int64_t B, int64_t groups, int64_t most) {
  const int64_t n = most / (B < most ? B : most), rounds = (groups + n - 1) / n;
  return (groups + rounds - 1) / rounds;
}
// partial rows per sample.  Two blocks a CU in all; at least four rounds a block, since every partial row is read again.
int64_t partials(int64_t B, int64_t T, int D, Shape s) {
  const int64_t groups = row_groups(T, s);
  if (groups <= 4 && s.nt) return 1;                     // a handful of rows: one block, no second launch
  if (!s.nt) return groups < 64 ? groups : 64;
  const int64_t n = even_blocks(B, groups, 512);
  return n > (groups + 3) / 4 ? (groups + 3) / 4 : n;
}

// MANY: two or three chunks a lane are built where pick takes them - 16-bit types, whole chunks, no parameter gradient
#define LN_DISPATCH(KERNEL, MANY, ...)                                        \
  if (s.nt == 16) KERNEL(16, 1, __VA_ARGS__);                                 \
  else if (s.nt == 64 && s.nch == 1) KERNEL(64, 1, __VA_ARGS__);              \
  else if (s.nt == 128) KERNEL(128, 1, __VA_ARGS__);                          \
  else if (s.nt == 256 && s.nch == 1) KERNEL(256, 1, __VA_ARGS__);            \
  else if (s.nt == 512 && s.nch == 1) KERNEL(512, 1, __VA_ARGS__);            \
  else if (s.nt == 512) KERNEL(512, 2, __VA_ARGS__);                          \
  else if constexpr (MANY) {                                                  \
    if (s.nt == 64 && s.nch == 2) KERNEL(64, 2, __VA_ARGS__);                 \
    else if (s.nt == 64) KERNEL(64, 3, __VA_ARGS__);                          \
    else KERNEL(256, 2, __VA_ARGS__);                                         \
  }

template <int T>
void launch_fwd(const LnArgs& a, int64_t B, hipStream_t st) {
  const Shape s = pick(B * a.T, a.D, T == 2, false);
  const dim3 grid((unsigned)even_blocks(B, row_groups(a.T, s), 1024), (unsigned)B);
  if (!s.nt) {
    hipLaunchKernelGGL((ln_wide_kernel<T, false>), grid, dim3(256), 0, st, a);
    return;
  }
#define LN_F(NT, N, FULL) hipLaunchKernelGGL((ln_fwd_kernel<T, NT, N, FULL>), grid, dim3(64 * WAVES), 0, st, a)
  if (a.D % 8 == 0) {
    LN_DISPATCH(LN_F, T < 2, true)
  } else {
    LN_DISPATCH(LN_F, false, false)
  }
#undef LN_F
}

// A parameter vector that few rows feed is added up by extra blocks of the same launch, which read those rows a second time
// (231 x 771 float32: one launch of 9 us instead of 9 + 2.5 and the second launch's 3 us on the host).  With parameters per sample
// this holds while the second reading comes from the caches; one launch / two, bf16: 4 x 77 x 1280 3.8 / 8.0 us, 8 x 256 x 1280
// 10.6 / 10.9, 16 x 64 x 4096 11.1 / 17.5, 16 x 256 x 1024 12.7 / 11.1, 16 x 512 x 2048 31.9 / 25.5, 256 x 77 x 1280 68 / 52.
constexpr int64_t FEW_ROWS = 512, FEW_ELEMENTS = 1 << 22;

template <int T>
void launch_bwd(LnArgs a, int64_t B, hipStream_t st) {
  const bool pg = a.dgamma != nullptr, shared = pg && a.p_bs == 0;
  const bool few = pg && (shared ? B * a.T : a.T) <= FEW_ROWS && B * a.T * a.D <= FEW_ELEMENTS;
  const Shape s = pick(B * a.T, a.D, T == 2, pg);
  const int64_t np = partials(B, a.T, a.D, s);
  a.direct = pg && s.nt && np == 1 && (B == 1 || !shared);
  const bool fold = few && s.nt && !a.direct;
  const int64_t nx = pg && s.nt && !fold ? np : even_blocks(B, row_groups(a.T, s), 1024);
  a.row_blocks = (int)nx;
  a.B = (int)B;
  const dim3 grid((unsigned)(nx + (fold ? (a.D + 63) / 64 * 2 : 0)), (unsigned)B);
#define LN_B(NT, N, FULL, PG) hipLaunchKernelGGL((ln_bwd_kernel<T, NT, N, FULL, PG>), grid, dim3(64 * WAVES), 0, st, a)
  if (!s.nt) {
    hipLaunchKernelGGL((ln_wide_kernel<T, true>), grid, dim3(256), 0, st, a);
    if (pg) hipLaunchKernelGGL((ln_wide_param_kernel<T>), dim3((a.D + 2047) / 2048, (unsigned)np, (unsigned)B), dim3(256), 0, st, a);
  } else if (pg && !fold) {
    if (a.D % 8 == 0) {
      LN_DISPATCH(LN_B, false, true, true)
    } else {
      LN_DISPATCH(LN_B, false, false, true)
    }
  } else if (a.D % 8 == 0) {
    LN_DISPATCH(LN_B, T < 2, true, false)
  } else {
    LN_DISPATCH(LN_B, false, false, false)
  }
#undef LN_B
  if (pg && !fold && !a.direct) {
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
  // few rows: added up without partial rows, whatever the parameters' shape
  if (B * T <= FEW_ROWS && B * T * D <= FEW_ELEMENTS && pick(B * T, D, false, true).nt) return 0;
  return B * partials(B, T, D, pick(B * T, D, false, true)) * 2 * D * 4;
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
  const int64_t need = dgamma ? fluxhip_layernorm_grad_ws(B, T, D) : 0;
  if (need && (!ws || ws_bytes < need)) return FLUXHIP_EINVAL;
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
