// Rotary positions on q and k in one launch, forward and inverse (the gradient).
//
// Pair j of a token at position p turns by the angle a = p[axis(j)] freq[j]:  (x, y) -> s (x cos a - y sin a, x sin a + y cos a);
// the inverse turns by -a with the same amplitude s, which is the transpose, hence the gradient.  Pairs are neighbours (2j, 2j + 1)
// (interleaved) or (j, j + rot / 2) (half); the columns behind rot are copied.  HBM-bound: each element is read and written once.
//
// The angle is formed in 64 bits - at position 10^6 a float32 product is off by 0.06 rad - and reduced to a fraction of a turn
// there; cos / sin of the fraction are float32 (its rounding is at most 2 pi 2^-26 rad: a float32 result ends 4.7e-8 from the exact
// one, with 64-bit sines 3.5e-8; 16-bit results do not see it).  A block takes TB consecutive tokens: one thread per (token, pair)
// computes the pair's cos and sin ONCE into LDS, then all threads walk the tokens' q and k heads in vectors of V elements; a thread
// keeps its columns and moves over (token, head) items.
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
  int pos64, ax1, ax2, ax3;            // first pair of axis 1, 2, 3
  int T, H, K, hd, rot, tb, slots, lanes;
  uint32_t magic;                      // ceil(2^32 / heads): i / heads = umulhi(i, magic) for i heads < 2^32
  float scale;
};

// V elements as they lie in memory
template <int T, int V>
struct Vec {
  typename Elem<T>::type w[V];
  DEVINL void load(const typename Elem<T>::type* p) { __builtin_memcpy(w, p, sizeof(w)); }
  DEVINL void store(typename Elem<T>::type* p) const { __builtin_memcpy(p, w, sizeof(w)); }
  DEVINL float get(int j) const { return Elem<T>::get(&w[j]); }
  DEVINL void put(int j, float v) { Elem<T>::put(&w[j], v); }
  // the last n < V elements, in pieces of 4, 2 and 1 (constant offsets: the vector stays in registers)
  template <int N> DEVINL void piece(typename Elem<T>::type* p, int j) const { __builtin_memcpy(p + j, w + j, N * sizeof(w[0])); }
  DEVINL void store_last(typename Elem<T>::type* p, int n) const {
    if constexpr (V == 8) {
      if (n & 4) {
        piece<4>(p, 4);
        if (n & 2) { piece<2>(p, 2); if (n & 1) piece<1>(p, 1); }
        else if (n & 1) piece<1>(p, 3);
        return;
      }
    }
    if (n & 2) { piece<2>(p, V - 2); if (n & 1) piece<1>(p, V - 3); }
    else if (n & 1) piece<1>(p, V - 1);
  }
};

// V: elements per vector (interleaved: V / 2 pairs; half: V pairs, two vectors), 16 bytes.  Where the rotated columns do not divide,
// the last vector is moved back to end with them and stores only what the one before it does not (in place, a column still has one
// writer); rows only need element alignment.  A thread takes UNROLL (token, head) items at a time, all loads before the first use;
// the first batch's loads go out before the block works on its angles.  4608 tokens x 48 heads x 128 bf16: 25.3 us for 113 MB
// (4.5 TB/s); 4 x 4352 tokens 90.9 us (4.7 TB/s); one load at a time: 29.9 and 127 us.
template <int T, int V, bool INTER, bool INV>
__global__ __launch_bounds__(256) void rotary_kernel(RopeArgs a) {
  using E = typename Elem<T>::type;
  constexpr int UNROLL = INTER ? 4 : 2;
  extern __shared__ float2 cs[];       // [tb][rot / 2]
  const int np = a.rot >> 1;
  const int64_t tok0 = (int64_t)blockIdx.x * a.tb, b0 = tok0 / a.T;
  const int ntb = (int)(a.ntok - tok0 < a.tb ? a.ntok - tok0 : a.tb), t0 = (int)(tok0 - b0 * a.T);

  const int heads = a.H + a.K, per = 256 / a.lanes;       // `lanes` threads cover a head's slots, `per` heads side by side
  const int row = threadIdx.x / a.lanes, lane = threadIdx.x - row * a.lanes;
  const int part = INTER ? a.rot : np, rot_slots = (part + V - 1) / V, step = per * gridDim.y, items = row < per ? ntb * heads : 0;
  const int first = row + blockIdx.y * per;

  const E* x[UNROLL];
  E* y[UNROLL];
  int tk[UNROLL];
  Vec<T, V> p[UNROLL], q[INTER ? 1 : UNROLL];
  auto fetch = [&](int it, int slot) {                    // items it, it + step, ..: an item behind the end repeats the last one
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = min(it + u * step, items - 1);
      tk[u] = (int)__umulhi((uint32_t)i, a.magic);        // i / heads
      if (heads == 1) tk[u] = i;
      const int h = i - tk[u] * heads;
      uint32_t t = t0 + tk[u], bq = t / (uint32_t)a.T;
      t -= bq * a.T;
      const int64_t b = b0 + bq;
      const bool isk = h >= a.H;
      const RopeTensor& r = isk ? a.k : a.q;
      const int64_t hh = isk ? h - a.H : h;
      x[u] = (const E*)r.x + b * r.xb + t * r.xt + hh * r.xh;
      y[u] = (E*)r.y + b * r.yb + t * r.yt + hh * r.yh;
      if (slot < rot_slots && part >= V) {
        const int c = min(slot * V, part - V);
        p[u].load(x[u] + c);
        if constexpr (!INTER) q[u].load(x[u] + np + c);
      }
    }
  };
  if (first < items && lane < a.slots) fetch(first, lane);

  for (int i = threadIdx.x; i < ntb * np; i += 256) {
    const int k = i / np, j = i - k * np;
    uint32_t t = t0 + k;
    const uint32_t bq = t / (uint32_t)a.T;
    t -= bq * a.T;
    const int ax = (j >= a.ax1) + (j >= a.ax2) + (j >= a.ax3);
    const int64_t at = (b0 + bq) * a.pb + t * a.pt + ax;
    const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
    const double turns = pos * a.freq[j] * 0.15915494309189533576888;
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(c * a.scale, INV ? -s * a.scale : s * a.scale);
  }
  __syncthreads();

  for (int slot = lane; slot < a.slots; slot += a.lanes) {
    for (int it = first; it < items; it += step * UNROLL) {
      if (it != first || slot != lane) fetch(it, slot);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (it + u * step >= items) break;
        const float2* w = cs + tk[u] * np;
        if (slot >= rot_slots) {                          // behind the rotated part
          const int c = a.rot + (slot - rot_slots) * V;
          if (c + V <= a.hd) {
            Vec<T, V> v;
            v.load(x[u] + c);
            v.store(y[u] + c);
          } else {
            for (int e = c; e < a.hd; ++e) y[u][e] = x[u][e];
          }
        } else if (part < V) {                            // a few columns only: by element
          for (int e = 0; e < part; e += INTER ? 2 : 1) {
            const float2 c = w[INTER ? e >> 1 : e];
            const int f = INTER ? e + 1 : np + e;
            const float m = Elem<T>::get(x[u] + e), n = Elem<T>::get(x[u] + f);
            Elem<T>::put(y[u] + e, m * c.x - n * c.y);
            Elem<T>::put(y[u] + f, m * c.y + n * c.x);
          }
        } else {
          const int c0 = min(slot * V, part - V), cnt = part - slot * V;   // cnt < V: of the last, moved vector
          Vec<T, V> o1, o2;
          if constexpr (INTER) {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
              const float2 c = w[(c0 >> 1) + j];
              const float m = p[u].get(2 * j), n = p[u].get(2 * j + 1);
              o1.put(2 * j, m * c.x - n * c.y);
              o1.put(2 * j + 1, m * c.y + n * c.x);
            }
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float2 c = w[c0 + j];
              const float m = p[u].get(j), n = q[u].get(j);
              o1.put(j, m * c.x - n * c.y);
              o2.put(j, m * c.y + n * c.x);
            }
          }
          if (cnt >= V) {
            o1.store(y[u] + c0);
            if constexpr (!INTER) o2.store(y[u] + np + c0);
          } else {
            o1.store_last(y[u] + c0, cnt);
            if constexpr (!INTER) o2.store_last(y[u] + np + c0, cnt);
          }
        }
      }
    }
  }
}

template <int T>
void launch(const RopeArgs& a, int interleaved, int inverse, dim3 grid, size_t lds, hipStream_t st) {
  constexpr int V = T == 2 ? 4 : 8;
  if (interleaved) {
    if (inverse) hipLaunchKernelGGL((rotary_kernel<T, V, true, true>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((rotary_kernel<T, V, true, false>), grid, dim3(256), lds, st, a);
  } else {
    if (inverse) hipLaunchKernelGGL((rotary_kernel<T, V, false, true>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((rotary_kernel<T, V, false, false>), grid, dim3(256), lds, st, a);
  }
}

// ---- what an output may share with the inputs (host)
struct View {                          // a tensor's bytes: first address, and the dimensions that move, the widest stride first
  int64_t at = 0, stride[4], n[4];
  int dims = 0, e = 0;
  bool repeats = false;                // several elements at one address
  View(const void* p, const int64_t* strides, int64_t B, int64_t T, int64_t H, int64_t hd, int size) : at((int64_t)p), e(size) {
    const int64_t s[4] = {strides[0] * size, strides[1] * size, strides[2] * size, size}, c[4] = {B, T, H, hd};
    for (int i = 0; i < 4; ++i) {
      if (c[i] <= 1) continue;
      if (s[i] == 0) { repeats = true; continue; }
      if (s[i] < 0) at += s[i] * (c[i] - 1);
      int j = dims++;
      for (; j > 0 && stride[j - 1] < llabs(s[i]); --j) stride[j] = stride[j - 1], n[j] = n[j - 1];
      stride[j] = llabs(s[i]);
      n[j] = c[i];
    }
    __int128 inside = e;
    for (int i = dims; i-- > 0;) {     // each stride has to pass over all that lies inside it
      repeats |= stride[i] < inside;
      inside += (__int128)stride[i] * (n[i] - 1);
    }
  }
  bool operator==(const View& o) const {
    bool same = at == o.at && dims == o.dims;
    for (int i = 0; same && i < dims; ++i) same = stride[i] == o.stride[i] && n[i] == o.n[i];
    return same;
  }
  // bytes from the first to behind the last, of the dimensions from the d-th with strides below `below`
  __int128 length(int d, __int128 below) const {
    __int128 l = e;
    for (int i = d; i < dims; ++i) l += stride[i] < below ? (__int128)stride[i] * (n[i] - 1) : 0;
    return l;
  }
  bool multiple(int d, int64_t period) const {
    bool ok = true;
    for (int i = d; i < dims; ++i) ok &= stride[i] < period || stride[i] % period == 0;
    return ok;
  }
};
// Whether two views provably share no byte: one ends in front of the other, or they lie in different columns of a common period (the
// heads of a fused projection), sample by sample where their widest strides agree and no sample reaches into the next.
bool apart(const View& a, const View& b) {
  const __int128 all = (__int128)1 << 100;
  const int64_t gap = b.at - a.at;
  for (int d = 0;; ++d) {
    const __int128 la = a.length(d, all), lb = b.length(d, all);
    if (gap >= la || -gap >= lb) return true;
    for (const View* v : {&a, &b})
      for (int i = d; i < v->dims; ++i) {
        const int64_t period = v->stride[i], m = (gap % period + period) % period;
        if (a.multiple(d, period) && b.multiple(d, period) && m >= a.length(d, period) && m + b.length(d, period) <= period) return true;
      }
    if (d >= a.dims || d >= b.dims || a.stride[d] != b.stride[d]) return false;
    const __int128 ia = a.length(d + 1, all), ib = gap + b.length(d + 1, all);
    if ((ia > ib ? ia : ib) - (gap < 0 ? gap : 0) > a.stride[d]) return false;
  }
}

}  // namespace

extern "C" int fluxhip_rotary_overlap(const fluxhip_rotary_desc* d) {
  if (!d) return FLUXHIP_EINVAL;
  const int e = d->dtype == 2 ? 4 : 2;
  const View q(d->q, d->q_strides, d->B, d->T, d->H, d->hd, e), qo(d->q_out, d->qo_strides, d->B, d->T, d->H, d->hd, e);
  const View k(d->k, d->k_strides, d->B, d->T, d->K, d->hd, e), ko(d->k_out, d->ko_strides, d->B, d->T, d->K, d->hd, e);
  if (d->B * d->T == 0) return 0;
  if ((d->H && qo.repeats) || (d->K && ko.repeats)) return 3;
  if (d->H && !(qo == q) && !apart(qo, q)) return 1;
  if (d->K && !(ko == k) && !apart(ko, k)) return 2;
  return d->H && d->K && !(apart(qo, ko) && apart(qo, k) && apart(q, ko)) ? 4 : 0;
}

extern "C" int fluxhip_rotary(const fluxhip_rotary_desc* d, void* stream) {
  if (!d || d->B < 0 || d->B > (1ll << 32) || d->T < 0 || d->T > (1 << 30) || d->H < 0 || d->K < 0 || d->hd < 1 || d->hd > 4096 ||
      d->rot < 2 || d->rot > d->hd || (d->rot & 1) || d->n_axes < 1 || d->n_axes > 4 || d->dtype < 0 || d->dtype > 2)
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
  if (d->H > 4096 || d->K > 4096 || !d->positions || !d->freqs ||
      (d->H && (!d->q || !d->q_out)) || (d->K && (!d->k || !d->k_out)) || fluxhip_rotary_overlap(d)) return FLUXHIP_EINVAL;
  RopeArgs a{};
  a.q = {d->q, d->q_out, d->q_strides[0], d->q_strides[1], d->q_strides[2], d->qo_strides[0], d->qo_strides[1], d->qo_strides[2]};
  a.k = {d->k, d->k_out, d->k_strides[0], d->k_strides[1], d->k_strides[2], d->ko_strides[0], d->ko_strides[1], d->ko_strides[2]};
  a.pos = d->positions; a.freq = (const double*)d->freqs;
  a.pb = d->pos_strides[0]; a.pt = d->pos_strides[1]; a.pos64 = d->pos64;
  a.ax1 = ax[1]; a.ax2 = ax[2]; a.ax3 = ax[3];
  a.ntok = ntok; a.T = (int)d->T; a.H = d->H; a.K = d->K; a.hd = d->hd; a.rot = d->rot; a.scale = d->scale;
  const int part = d->interleaved ? d->rot : d->rot / 2, tail = d->hd - d->rot, V = d->dtype == 2 ? 4 : 8;
  a.slots = (part + V - 1) / V + (tail + V - 1) / V;
  a.lanes = a.slots < 256 ? a.slots : 256;
  const int per = 256 / a.lanes, heads = d->H + d->K, np = d->rot / 2;
  a.magic = (uint32_t)(((1ull << 32) + heads - 1) / heads);
  // tokens per block: one sincos per thread (256 / pairs tokens), fewer while the launch would leave CUs idle; with few tokens
  // the heads are spread over blocks instead
  int tb = 256 / np > 1 ? 256 / np : 1;
  if (tb > 16) tb = 16;
  while (tb > 1 && ntok / tb < 1024) tb >>= 1;
  a.tb = tb;
  const int64_t nb = (ntok + tb - 1) / tb;
  if (nb >= (1ll << 24)) return FLUXHIP_EINVAL;           // (a grid holds 2^32 threads)
  int gy = 1;
  if (tb == 1)
    while (nb * gy < 512 && gy * per < heads && gy < 64) gy <<= 1;
  const dim3 grid((unsigned)nb, (unsigned)gy);
  const size_t lds = (size_t)tb * np * sizeof(float2);
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == 0) launch<0>(a, d->interleaved, d->inverse, grid, lds, st);
  else if (d->dtype == 1) launch<1>(a, d->interleaved, d->inverse, grid, lds, st);
  else launch<2>(a, d->interleaved, d->inverse, grid, lds, st);
  return hipGetLastError() == hipSuccess ? FLUXHIP_OK : FLUXHIP_ELAUNCH;
}
