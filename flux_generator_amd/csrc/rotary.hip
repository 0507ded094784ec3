// Rotary positions on q and k in one launch, forward and inverse (the gradient).
//
// Pair j of a token at position p turns by the angle a = p[axis(j)] freq[j]:  (x, y) -> s (x cos a - y sin a, x sin a + y cos a);
// the inverse turns by -a with the same amplitude s, which is the transpose, hence the gradient.  Pairs are neighbours (2j, 2j + 1)
// (interleaved) or (j, j + rot / 2) (half); the columns behind rot are copied.  HBM-bound: each element is read and written once.
//
// The angle is formed in 64 bits - at position 10^6 a float32 product is off by 0.06 rad - and reduced to a fraction of a turn
// there; cos / sin of the fraction are float32.  A block takes TB consecutive tokens: one thread per (token, pair) computes the
// pair's cos and sin ONCE into LDS, then all threads walk the tokens' heads in vectors of V elements; a thread keeps its column
// and moves over heads, so a token's q and k heads (and the values between them in a fused projection) need no index division.
#include "../../include/fluxhip.h"
#include "common.h"
#include "elem.h"

namespace {

struct RopeTensor {
  const void* x;
  void* y;
  int64_t xb, xt, xh, yb, yt, yh;      // element strides of batch, token, head
};
struct RopeArgs {
  RopeTensor q, k;
  const void* pos;
  const double* freq;
  int64_t pb, pt, ntok;                // element strides of the positions; B * T
  int pos64, n_axes, ax1, ax2, ax3;    // first pair of axis 1, 2, 3
  int T, H, K, hd, rot, tb, slots, lanes;
  float scale;
};

template <int T, int V>
DEVINL void vload(const typename Elem<T>::type* p, float (&v)[V]) {
  typename Elem<T>::type w[V];
  __builtin_memcpy(w, p, sizeof(w));
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = Elem<T>::get(&w[j]);
}
template <int T, int V>
DEVINL void vstore(typename Elem<T>::type* p, const float (&v)[V]) {
  typename Elem<T>::type w[V];
#pragma unroll
  for (int j = 0; j < V; ++j) Elem<T>::put(&w[j], v[j]);
  __builtin_memcpy(p, w, sizeof(w));
}

// V: elements per vector (interleaved: V / 2 pairs; half: V pairs, two vectors), dividing the rotated columns
template <int T, int V, bool INTER, bool INV>
__global__ __launch_bounds__(256) void rotary_kernel(RopeArgs a) {
  using E = typename Elem<T>::type;
  extern __shared__ float2 cs[];       // [tb][rot / 2]
  const int np = a.rot >> 1;
  const int64_t tok0 = (int64_t)blockIdx.x * a.tb;
  const int ntb = (int)(a.ntok - tok0 < a.tb ? a.ntok - tok0 : a.tb);
  const int64_t b0 = tok0 / a.T;
  const int t0 = (int)(tok0 - b0 * a.T);
  for (int i = threadIdx.x; i < ntb * np; i += 256) {
    const int tk = i / np, j = i - tk * np;
    int64_t b = b0;
    int t = t0 + tk;
    while (t >= a.T) { t -= a.T; ++b; }
    const int ax = (j >= a.ax1) + (j >= a.ax2) + (j >= a.ax3);
    const int64_t at = b * a.pb + t * a.pt + ax;
    const double p = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
    const double turns = p * a.freq[j] * 0.15915494309189533576888;
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(c * a.scale, INV ? -s * a.scale : s * a.scale);
  }
  __syncthreads();
  const int heads = a.H + a.K, per = 256 / a.lanes;       // `lanes` threads cover a head's slots, `per` heads side by side
  const int lane = threadIdx.x % a.lanes;
  if ((int)threadIdx.x >= per * a.lanes) return;
  const int rot_slots = INTER ? a.rot / V : np / V;
  for (int slot = lane; slot < a.slots; slot += a.lanes) {
    int64_t b = b0;
    int tk = 0, t = t0, h = threadIdx.x / a.lanes + blockIdx.y * per;
    const int step = per * gridDim.y;
    while (true) {
      while (h >= heads) {
        h -= heads;
        ++tk;
        if (++t == a.T) { t = 0; ++b; }
      }
      if (tk >= ntb) break;
      const bool isk = h >= a.H;
      const RopeTensor& r = isk ? a.k : a.q;
      const int64_t hh = isk ? h - a.H : h;
      const E* x = (const E*)r.x + b * r.xb + t * r.xt + hh * r.xh;
      E* y = (E*)r.y + b * r.yb + t * r.yt + hh * r.yh;
      const float2* w = cs + tk * np;
      if (slot >= rot_slots) {                            // behind the rotated part
        const int c = a.rot + (slot - rot_slots) * V;
        if (c + V <= a.hd) {
          float v[V];
          vload<T, V>(x + c, v);
          vstore<T, V>(y + c, v);
        } else {
          for (int e = c; e < a.hd; ++e) y[e] = x[e];
        }
      } else if constexpr (INTER) {
        float v[V], o[V];
        vload<T, V>(x + slot * V, v);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
          const float2 u = w[slot * (V / 2) + j];
          o[2 * j] = v[2 * j] * u.x - v[2 * j + 1] * u.y;
          o[2 * j + 1] = v[2 * j] * u.y + v[2 * j + 1] * u.x;
        }
        vstore<T, V>(y + slot * V, o);
      } else {
        float p[V], q[V], o1[V], o2[V];
        vload<T, V>(x + slot * V, p);
        vload<T, V>(x + np + slot * V, q);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float2 u = w[slot * V + j];
          o1[j] = p[j] * u.x - q[j] * u.y;
          o2[j] = p[j] * u.y + q[j] * u.x;
        }
        vstore<T, V>(y + slot * V, o1);
        vstore<T, V>(y + np + slot * V, o2);
      }
      h += step;
    }
  }
}

template <int T, int V>
void launch_v(const RopeArgs& a, int interleaved, int inverse, dim3 grid, size_t lds, hipStream_t st) {
  if (interleaved) {
    if constexpr (V >= 2) {
      if (inverse) hipLaunchKernelGGL((rotary_kernel<T, V, true, true>), grid, dim3(256), lds, st, a);
      else hipLaunchKernelGGL((rotary_kernel<T, V, true, false>), grid, dim3(256), lds, st, a);
    }
  } else {
    if (inverse) hipLaunchKernelGGL((rotary_kernel<T, V, false, true>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((rotary_kernel<T, V, false, false>), grid, dim3(256), lds, st, a);
  }
}

}  // namespace

extern "C" int fluxhip_rotary(const fluxhip_rotary_desc* d, void* stream) {
  if (!d || d->B < 0 || d->T < 0 || d->H < 0 || d->K < 0 || d->hd < 1 || d->hd > 4096 || d->rot < 2 || d->rot > d->hd || (d->rot & 1) ||
      d->n_axes < 1 || d->n_axes > 4 || d->dtype < 0 || d->dtype > 2)
    return FLUXHIP_EINVAL;
  int pairs = 0, ax[4] = {0, 1 << 30, 1 << 30, 1 << 30};
  for (int i = 0; i < d->n_axes; ++i) {
    if (d->axis_pairs[i] < 0) return FLUXHIP_EINVAL;
    if (i) ax[i] = pairs;
    pairs += d->axis_pairs[i];
    if (pairs > d->rot / 2) return FLUXHIP_EINVAL;
  }
  if (pairs != d->rot / 2) return FLUXHIP_EINVAL;
  const int64_t ntok = d->B * d->T;
  if (ntok == 0 || d->H + d->K == 0) return FLUXHIP_OK;
  if (d->T > (1ll << 31) - 1 || !d->positions || !d->freqs || (d->H && (!d->q || !d->q_out)) || (d->K && (!d->k || !d->k_out))) return FLUXHIP_EINVAL;
  RopeArgs a{};
  a.q = {d->q, d->q_out, d->q_strides[0], d->q_strides[1], d->q_strides[2], d->qo_strides[0], d->qo_strides[1], d->qo_strides[2]};
  a.k = {d->k, d->k_out, d->k_strides[0], d->k_strides[1], d->k_strides[2], d->ko_strides[0], d->ko_strides[1], d->ko_strides[2]};
  a.pos = d->positions; a.freq = (const double*)d->freqs;
  a.pb = d->pos_strides[0]; a.pt = d->pos_strides[1]; a.pos64 = d->pos64; a.n_axes = d->n_axes;
  a.ax1 = ax[1]; a.ax2 = ax[2]; a.ax3 = ax[3];
  a.ntok = ntok; a.T = (int)d->T; a.H = d->H; a.K = d->K; a.hd = d->hd; a.rot = d->rot; a.scale = d->scale;
  // vectors: 16 bytes where the rotated columns (halves) divide into them; the loads themselves take any address
  const int part = d->interleaved ? d->rot : d->rot / 2, tail = d->hd - d->rot, most = d->dtype == 2 ? 4 : 8;
  int V = most;
  while (part % V) V >>= 1;                               // (interleaved: rot is even, so V >= 2)
  a.slots = part / V + (tail + V - 1) / V;
  a.lanes = a.slots < 256 ? a.slots : 256;
  const int per = 256 / a.lanes, heads = d->H + d->K, np = d->rot / 2;
  // tokens per block: one sincos per thread (256 / pairs tokens), fewer while the launch would leave CUs idle; with few tokens
  // the heads are spread over blocks instead
  int tb = 256 / np > 1 ? 256 / np : 1;
  if (tb > 16) tb = 16;
  while (tb > 1 && ntok / tb < 1024) tb >>= 1;
  a.tb = tb;
  const int64_t nb = (ntok + tb - 1) / tb;
  if (nb > (1ll << 31) - 1) return FLUXHIP_EINVAL;
  int gy = 1;
  if (tb == 1)
    while (nb * gy < 512 && gy * per < heads && gy < 64) gy <<= 1;
  const dim3 grid((unsigned)nb, (unsigned)gy);
  const size_t lds = (size_t)tb * np * sizeof(float2);
  hipStream_t st = (hipStream_t)stream;
#define ROPE(T, V) launch_v<T, V>(a, d->interleaved, d->inverse, grid, lds, st)
  if (d->dtype == 0) { if (V == 8) ROPE(0, 8); else if (V == 4) ROPE(0, 4); else if (V == 2) ROPE(0, 2); else ROPE(0, 1); }
  else if (d->dtype == 1) { if (V == 8) ROPE(1, 8); else if (V == 4) ROPE(1, 4); else if (V == 2) ROPE(1, 2); else ROPE(1, 1); }
  else { if (V == 4) ROPE(2, 4); else if (V == 2) ROPE(2, 2); else ROPE(2, 1); }
#undef ROPE
  return hipGetLastError() == hipSuccess ? FLUXHIP_OK : FLUXHIP_ELAUNCH;
}
