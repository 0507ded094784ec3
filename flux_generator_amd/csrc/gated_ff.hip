// Gated feed-forward block, forward and backward, for training adapters (and whole blocks) and for serving.
//
//   value = x Wv^T + bv, gate = x Wg^T + bg, hidden = value act(gate), y = hidden Wo^T + bo
//   dh = dy Wo, dvalue = dh act(gate), dgate = dh value act'(gate)
//   dx = dvalue Wv + dgate Wg, dWv = dvalue^T x, dWg = dgate^T x, dWo = dy^T hidden, db = column sums
//
// Five matrix products of 2 M D F flops each way and more (6 M D F forward, 12 M D F backward): MFMA-bound for many tokens, bound
// by the bytes of the weights for few.  One kernel template serves them: out[m][n] = sum_k Q(m, k) P(n, k), where either operand
// lies with k contiguous ("row": activations and nn.Linear weights in the forward pass) or with k strided ("col": the weights of
// the input gradient, both operands of the weight gradients).  Nothing is transposed in memory: a "col" tile is staged as it lies
// and its fragments are read with the transposing LDS read of this chip (ds_read_b64_tr_b16).
//
// P is the MFMA's first operand, so a lane's four accumulators are four neighbouring n of one m; one permlane16 swap per register
// pair makes that eight (a 16-byte store).
#include "../../include/fluxhip.h"
#include "common.h"
#include "elem.h"
#include "colsum.h"

namespace {

constexpr int BK = 64;
constexpr uint32_t OOB = 0xFFFFFFF0u;                      // a buffer offset that fails every range check: the load writes zeros
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) char lds_char;

enum { EPI_STORE = 0, EPI_UP = 1, EPI_DH = 2 };

struct FfArgs {
  const char *P[2], *Q[2];
  char* out[2];
  int64_t ldp, ldq;           // element strides of the operands' rows
  int64_t ldo;                // ... of the output's rows
  int M, N, K;                // output rows and columns, contraction length of a segment
  int nseg, nbatch, splits;   // segments s add P[s] Q[s]; batches b write out[b] = P[0] Q[b]
  int tiles_m, tiles_n, act;
  const char *bias[2], *value, *gate;
  char *vout, *gout;          // EPI_UP: saved value / gate (or null); EPI_DH: dvalue / dgate
  float* part;                // EPI_STORE with splits > 1: partial products; EPI_DH: column sums [2 tiles_m][2][N] (or null)
};

// gfx950 fragment swizzles.  row tile: 64 k = 8 chunks of 16 bytes a row, chunk ^= (row >> 1) & 7.  col tile: one k a row, its
// 32-byte granules (16 columns) ^= f(k): the rows one transposing read touches fall on different banks either way.
DEVINL int col_f(int k) { return (k & 3) | ((k >> 1) & 4); }

// 16 bytes a lane from the buffer straight into LDS at dst + 16 lane (dst wave-uniform; m0 carries it).  Inline asm because the
// compiler, which cannot tell the two stages apart, would wait for all of these before every transposing LDS read; it has no
// output register, and the main loop's own vmcnt waits cover it.
DEVINL void dma16(u32x4 rs, uint32_t voff, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(voff), "s"(rs) : "memory");
}

template <bool COL, int BI>     // BI: indices of the tile, 64 (half a "row" tile), 128 or 256
struct Stager {
  static constexpr int NP = 4;                             // 1 KiB pieces per wave
  int64_t ld;
  int i0, ni, K;
  uint32_t voff[NP];
  int chunk[2];                                            // row tile: this lane's k chunk in even / odd pieces
  u32x4 rs;
  int kk;

  DEVINL void init(int lane, int piece0, int64_t ld_, int i0_, int ni_, int K_) {
    ld = ld_; i0 = i0_; ni = ni_; K = K_;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int piece = piece0 + j;
      if constexpr (!COL) {
        const int row = piece * 8 + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
        voff[j] = (uint32_t)(row * ld * 2 + c * 16);
        chunk[j & 1] = c;                                  // piece0 is even
      } else {
        constexpr int KR = 512 / BI;                       // k rows per piece
        const int k = piece * KR + lane / (BI / 8), s = lane % (BI / 8);
        const int c = (((s >> 1) ^ col_f(k)) << 1) | (s & 1);
        voff[j] = i0 + c * 8 < ni ? (uint32_t)(k * ld * 2 + c * 16) : OOB;
      }
    }
  }
  // the resource for k0 .. k0 + 63; indices and k behind the ends become zeros (piece() then stages this wave's j-th KiB)
  DEVINL void step(const char* base, int k0, bool on) {
    const char* b;
    int64_t num;
    if constexpr (!COL) {
      const int rows = min(ni - i0, BI);
      b = base + ((int64_t)i0 * ld + k0) * 2;
      num = rows > 0 && k0 < K ? ((int64_t)(rows - 1) * ld + (K - k0)) * 2 : 0;
    } else {
      const int rows = min(K - k0, BK);
      b = base + ((int64_t)k0 * ld + i0) * 2;
      num = rows > 0 ? ((int64_t)(rows - 1) * ld + min(ni - i0, BI)) * 2 : 0;
    }
    if (!on) num = 0;
    rs = u32x4{(uint32_t)(uintptr_t)b, (uint32_t)((uintptr_t)b >> 32) & 0xffffu, (uint32_t)num, 0x00020000u};
    kk = k0;
  }
  DEVINL void piece(int j, uint32_t dst) const {
    uint32_t v = voff[j];
    if constexpr (!COL) v = kk + chunk[j & 1] * 8 < K ? v : OOB;
    dma16(rs, v, dst + j * 1024);
  }
};

// fragment (16 indices from i, 32 k from 32 ks): lane l holds index i + (l & 15), k = 32 ks + 8 (l >> 4) + 0..7
template <bool COL, int BI>
struct Reader {
  int a0, a1;                                              // lane byte offsets
  DEVINL void init(int lane) {
    const int r = lane & 15, g = lane >> 4;
    if constexpr (!COL) {
      const int f = (r >> 1) & 7;
      a0 = r * 128 + ((g ^ f) << 4);
      a1 = r * 128 + (((g | 4) ^ f) << 4);
    } else {
      const int k = 8 * g + (r >> 2);                      // + 4 for the second half: col_f ignores that bit
      a0 = k * (BI * 2) + (col_f(k) << 5) + ((r & 3) << 3);
      a1 = 0;
    }
  }
  DEVINL bf16x8 read(const char* tile, int i, int ks) const {
    if constexpr (!COL) {
      return *(const bf16x8*)(tile + (ks ? a1 : a0) + i * 128);
    } else {
      const char* t = tile + (a0 ^ ((i >> 4 & 7) << 5)) + (i >> 7) * 256 + ks * 32 * (BI * 2);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)t);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(t + 4 * (BI * 2)));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

template <bool H>
DEVINL f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
  if constexpr (H) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(__attribute__((ext_vector_type(8))) __bf16, a),
                                                     __builtin_bit_cast(__attribute__((ext_vector_type(8))) __bf16, b), c, 0, 0, 0);
}

DEVINL float act_f(float x, int act) {
  return act == FLUXHIP_EPI_GELU_TANH ? gelu_tanh_f(x) : act == FLUXHIP_EPI_SILU ? silu_f(x) : gelu_erf_f(x);
}
// act(x) and act'(x).  silu: p (1 + x (1 - p)), p = sigmoid x.  tanh form: p + x p (1 - p) u', p = sigmoid(2 u).
// erf form: Phi(x) + x phi(x), Phi from the same rational erfc as gelu_erf_f with its exponential shared.
DEVINL void act_grad(float x, int act, float& f, float& df) {
  if (act == FLUXHIP_EPI_SILU) {
    const float p = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
    f = x * p;
    df = p * (1.0f + x * (1.0f - p));
  } else if (act == FLUXHIP_EPI_GELU_TANH) {
    constexpr float c0 = -2.0f * 0.7978845608028654f * 1.4426950408889634f, c1 = c0 * 0.044715f;
    const float x2 = x * x;
    const float p = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * __builtin_fmaf(x2, c1, c0)));
    f = x * p;
    df = p + f * (1.0f - p) * (1.5957691216057308f * __builtin_fmaf(x2, 0.134145f, 1.0f));
  } else {
    const float z = fabsf(x) * 0.7071067811865476f;
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, z, 1.0f));
    float q = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
    q = __builtin_fmaf(t, q, 1.421413741f);
    q = __builtin_fmaf(t, q, -0.284496736f);
    q = __builtin_fmaf(t, q, 0.254829592f);
    const float e = __builtin_amdgcn_exp2f(-1.4426950408889634f * (z * z)), h = 0.5f * (t * q) * e;
    const float phi = x >= 0.f ? 1.0f - h : h;
    f = x * phi;
    df = phi + x * e * 0.3989422804014327f;
  }
}

DEVINL void swap16(float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}

// NF n and MF m fragments per wave, WN x WM waves; block tile BT = 16 NF WN = 16 MF WM squared, 1 KiB x 4 pieces of either
// operand per wave and stage.  MF = 8: 256 square, eight waves (two a SIMD); MF = 4: 128 square, four waves, two blocks a CU.
template <int MF, bool PC, bool QC, int EPI, bool H>
__global__ __launch_bounds__(MF == 8 ? 512 : 256, 2) void ff_gemm_kernel(FfArgs a) {
  constexpr int NF = 4, BT = 32 * MF, WN = BT / 64, OPB = BT * BK * 2, STAGE = 2 * OPB;   // bytes of an operand tile, of a stage
  __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WN, wn = wave % WN;

  // block -> (split, batch, tile): consecutive ids of one XCD (id mod 8) walk bands of four row tiles, so its 32 CUs share
  // operand tiles in that XCD's L2
  int id = blockIdx.x;
  {
    const int n = gridDim.x, per = n >> 3, rem = n & 7, x = id & 7;
    id = x * per + min(x, rem) + (id >> 3);
  }
  const int tiles = a.tiles_m * a.tiles_n;
  int t = id % tiles;
  const int z = id / tiles, batch = z % a.nbatch, split = z / a.nbatch;
  const int band = t / (4 * a.tiles_n), bm = min(4, a.tiles_m - band * 4);
  t -= band * 4 * a.tiles_n;
  const int m0 = (band * 4 + t % bm) * BT;
  const int tn = t / bm, n0 = tn * (EPI == EPI_UP ? BT / 2 : BT);

  const int sps = (a.K + BK - 1) / BK, total = sps * a.nseg;
  const int s_lo = (int)((int64_t)total * split / a.splits), s_hi = (int)((int64_t)total * (split + 1) / a.splits), ns = s_hi - s_lo;

  // EPI_UP: P is two half tiles, value rows then gate rows, staged by the first and the second half of the waves
  Stager<PC, EPI == EPI_UP ? BT / 2 : BT> sp;
  Stager<QC, BT> sq;
  const char *pbase[2] = {a.P[0], a.P[1]}, *qbase[2] = {a.nbatch > 1 ? a.Q[batch] : a.Q[0], a.Q[1]};
  if (EPI == EPI_UP && wave >= WN) pbase[0] = a.P[1];      // (WN is half the number of waves)
  sp.init(lane, (EPI == EPI_UP ? wave % WN : wave) * 4, a.ldp, n0, a.N, a.K);
  sq.init(lane, wave * 4, a.ldq, m0, a.M, a.K);
  Reader<PC, BT> rp;
  Reader<QC, BT> rq;
  rp.init(lane);
  rq.init(lane);

  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + wave * 4096;
  auto open = [&](int s) {                                 // resources of step s
    const bool on = s < ns;                                // behind the last step: empty resources, the pieces write zeros
    const int st = s_lo + s, seg = a.nseg > 1 && st >= sps ? 1 : 0, k0 = (st - seg * sps) * BK;
    sp.step(pbase[EPI == EPI_UP ? 0 : seg], k0, on);
    sq.step(qbase[seg], k0, on);
  };
  auto piece = [&](int j, int buf) {                       // j-th of the wave's 8 pieces of a stage
    const uint32_t d = lds0 + buf * STAGE;
    if (j < 4) sp.piece(j, d);
    else sq.piece(j - 4, d + OPB);
  };

  f32x4 acc[NF][MF];                                       // [n fragment][m fragment]
  static_for<0, NF>([&](auto i) { static_for<0, MF>([&](auto j) { acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f}; }); });
  bf16x8 fp[2][NF], fq[MF];
  auto read_p = [&](int i, int buf, int ks) {              // fragments of k half ks of a stage
    const int row = EPI == EPI_UP ? (i >= NF / 2 ? BT / 2 : 0) + wn * (NF * 8) + (i % (NF / 2)) * 16 : wn * (NF * 16) + i * 16;
    fp[ks][i] = rp.read(smem + buf * STAGE, row, ks);
  };
  auto read_q = [&](int j, int buf, int ks) { fq[j] = rq.read(smem + buf * STAGE + OPB, wm * (MF * 16) + j * 16, ks); };
  auto mul = [&](auto j, int ks) {
    static_for<0, NF>([&](auto i) { acc[i][j] = mma<H>(fp[ks][i], fq[j], acc[i][j]); });
  };

  // Main loop: two LDS stages of 64 k, a step = two halves of 32 k, a half = MF groups of NF products.  Behind group j the Q
  // fragment it used is free and is read for the next half (P fragments alternate between two sets), so every LDS read has
  // about MF groups to land.  Once per step, behind the first group of the second half (it covers the last reads' latency),
  // the waves meet: all have the stage in registers and all pieces of the next stage are in LDS; the stage is then refilled
  // with step s + 2, whose loads have a whole step to land.
  if (ns > 0) {
    open(0);
    static_for<0, 8>([&](auto j) { piece(j, 0); });
    open(1);
    static_for<0, 8>([&](auto j) { piece(j, 1); });
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    static_for<0, NF>([&](auto i) { read_p(i, 0, 0); });
    static_for<0, MF>([&](auto j) { read_q(j, 0, 0); });
    for (int s = 0; s < ns; ++s) {
      const int buf = s & 1;
      static_for<0, MF>([&](auto j) {
        mul(j, 0);
        read_q(j, buf, 1);
        if constexpr (j < NF) read_p(j, buf, 1);
        __builtin_amdgcn_sched_barrier(0);
      });
      open(s + 2);
      static_for<0, MF>([&](auto j) {
        mul(j, 1);
        if constexpr (j == 0) {
          __builtin_amdgcn_sched_barrier(0);
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        static_for<j * 8 / MF, (j + 1) * 8 / MF>([&](auto e) { piece(e, buf); });
        read_q(j, buf ^ 1, 0);                             // (behind the last step: a stale stage, in bounds and not used)
        if constexpr (j < NF) read_p(j, buf ^ 1, 0);
        __builtin_amdgcn_sched_barrier(0);
      });
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // no piece outlives the loop
  }

  // ---- epilogue: lane holds m = .. + (lane & 15); after the swap 8 neighbouring n
  const int c = lane & 15, q = lane >> 4, noff = (q & 1) * 16 + (q >> 1) * 8;
  const int nb = n0 + (EPI == EPI_UP ? wn * (NF * 8) : wn * (NF * 16)) + noff, mb = m0 + wm * (MF * 16) + c;
  typedef uint16_t E;
  typedef Elem<H ? 1 : 0> El;
  if constexpr (EPI == EPI_UP) {
    static_for<0, NF / 4>([&](auto ih) {
      constexpr int i = 2 * ih;
      const int n = nb + i * 16;
      const bool in = n < a.N;
      float bv[8] = {}, bg[8] = {};
      if (in && a.bias[0]) {
        El::load8((const E*)a.bias[0] + n, 0, 8, bv);
        El::load8((const E*)a.bias[1] + n, 0, 8, bg);
      }
      static_for<0, MF>([&](auto j) {
        const int m = mb + j * 16;
        float v[8], g[8], h[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = acc[i][j][e]; v[4 + e] = acc[i + 1][j][e];
          g[e] = acc[i + NF / 2][j][e]; g[4 + e] = acc[i + 1 + NF / 2][j][e];
          swap16(v[e], v[4 + e]);
          swap16(g[e], g[4 + e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] += bv[e];
          g[e] += bg[e];
          h[e] = v[e] * act_f(g[e], a.act);
        }
        if (in && m < a.M) {
          const int64_t o = (int64_t)m * a.N;
          El::store8((E*)a.out[0] + o + n, 0, 8, h);
          if (a.vout) {
            El::store8((E*)a.vout + o + n, 0, 8, v);
            El::store8((E*)a.gout + o + n, 0, 8, g);
          }
        }
      });
    });
  } else if constexpr (EPI == EPI_DH) {
    static_for<0, NF / 2>([&](auto ih) {
      constexpr int i = 2 * ih;
      const int n = nb + i * 16;
      const bool in = n < a.N;
      float sv[8] = {}, sg[8] = {};
      static_for<0, MF>([&](auto j) {
        const int m = mb + j * 16;
        float d[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d[e] = acc[i][j][e]; d[4 + e] = acc[i + 1][j][e];
          swap16(d[e], d[4 + e]);
        }
        if (in && m < a.M) {
          const int64_t o = (int64_t)m * a.N;
          float v[8], g[8];
          El::load8((const E*)a.value + o + n, 0, 8, v);
          El::load8((const E*)a.gate + o + n, 0, 8, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float f, df;
            act_grad(g[e], a.act, f, df);
            g[e] = d[e] * v[e] * df;
            v[e] = d[e] * f;
            sv[e] += v[e];
            sg[e] += g[e];
          }
          El::store8((E*)a.vout + o + n, 0, 8, v);
          El::store8((E*)a.gout + o + n, 0, 8, g);
        }
      });
      if (a.part) {                                        // column sums over the wave's rows: 16 lanes, fixed order
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sv[e] = row16_sum(sv[e]);
          sg[e] = row16_sum(sg[e]);
        }
        if (c == 0 && in) {
          float* p = a.part + (int64_t)((m0 / BT) * 2 + wm) * 2 * a.N;
          Elem<2>::store8(p + n, 0, 8, sv);
          Elem<2>::store8(p + a.N + n, 0, 8, sg);
        }
      }
    });
  } else {
    static_for<0, NF / 2>([&](auto ih) {
      constexpr int i = 2 * ih;
      const int n = nb + i * 16;
      const bool in = n < a.N;
      float b[8] = {};
      if (in && a.bias[0] && a.splits == 1) El::load8((const E*)a.bias[0] + n, 0, 8, b);
      static_for<0, MF>([&](auto j) {
        const int m = mb + j * 16;
        float d[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d[e] = acc[i][j][e]; d[4 + e] = acc[i + 1][j][e];
          swap16(d[e], d[4 + e]);
        }
        if (in && m < a.M) {
          if (a.splits > 1) {
            Elem<2>::store8(a.part + (((int64_t)split * a.nbatch + batch) * a.M + m) * a.N + n, 0, 8, d);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] += b[e];
            El::store8((E*)a.out[batch] + (int64_t)m * a.ldo + n, 0, 8, d);
          }
        }
      });
    });
  }
}

// adds the split-K partial products in split order (+ bias), eight neighbouring columns a thread
template <bool H>
__global__ __launch_bounds__(256) void ff_reduce_kernel(FfArgs a) {
  typedef Elem<H ? 1 : 0> El;
  const int64_t n8 = a.N / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x, batch = blockIdx.y;
  if (i >= n8 * a.M) return;
  const int64_t m = i / n8;
  const int n = (int)(i - m * n8) * 8;
  float s[8] = {}, v[8];
  if (a.bias[0]) El::load8((const uint16_t*)a.bias[0] + n, 0, 8, s);
  for (int z = 0; z < a.splits; ++z) {
    Elem<2>::load8(a.part + (((int64_t)z * a.nbatch + batch) * a.M + m) * a.N + n, 0, 8, v);
    for (int e = 0; e < 8; ++e) s[e] += v[e];
  }
  El::store8((uint16_t*)a.out[batch] + m * a.ldo + n, 0, 8, s);
}

// column sums of [M][N] (first stage; colsum.h adds the partial rows): block = 2048 columns x a range of rows
template <bool H>
__global__ __launch_bounds__(256) void ff_colsum_kernel(const uint16_t* x, int64_t ld, int M, int N, float* part) {
  const int c = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (c >= N) return;
  float s[8] = {}, v[8];
#pragma unroll 4
  for (int m = blockIdx.y; m < M; m += gridDim.y) {
    Elem<H ? 1 : 0>::load8(x + m * ld, c, N, v);
    for (int e = 0; e < 8; ++e) s[e] += v[e];
  }
  Elem<2>::store8(part + (int64_t)blockIdx.y * N, c, N, s);
}

struct Plan { int mf, splits; };
// Tile and split of an [M][N] product of `steps` k-steps (nb batches).  256-square tiles (one block a CU) where they fill the
// chip, else 128-square ones (two a CU); a product of few tiles is split along k, its partials added by ff_reduce_kernel.
Plan pick(int64_t M, int64_t N, int nb, int64_t steps, bool can_split) {
  auto tiles = [&](int64_t b) { return ((M + b - 1) / b) * ((N + b - 1) / b) * nb; };
  const int64_t t256 = tiles(256), t128 = tiles(128);
  if (t256 >= 200) return {8, 1};
  int splits = 1;
  if (can_split)
    while (t128 * splits < 384 && steps / (splits * 2) >= 4 && splits < 16) splits *= 2;
  return {4, splits};
}
int64_t part_bytes(int64_t M, int64_t N, int nb, Plan p) { return p.splits > 1 ? M * N * nb * p.splits * 4 : 0; }
constexpr int COLSUM_ROWS = 256;

template <int MF, bool PC, bool QC, int EPI, bool H>
void launch_mf(FfArgs& a, hipStream_t st) {
  constexpr int BT = 32 * MF, BN = EPI == EPI_UP ? BT / 2 : BT;
  a.tiles_m = (a.M + BT - 1) / BT;
  a.tiles_n = (a.N + BN - 1) / BN;
  hipLaunchKernelGGL((ff_gemm_kernel<MF, PC, QC, EPI, H>), dim3((unsigned)(a.tiles_m * a.tiles_n * a.nbatch * a.splits)), dim3(MF == 8 ? 512 : 256), 0,
                     st, a);
}
template <bool PC, bool QC, int EPI, bool H>
void launch(FfArgs& a, Plan p, hipStream_t st) {
  a.splits = p.splits;
  if (p.mf == 8) launch_mf<8, PC, QC, EPI, H>(a, st);
  else launch_mf<4, PC, QC, EPI, H>(a, st);
  if (EPI == EPI_STORE && a.splits > 1)
    hipLaunchKernelGGL((ff_reduce_kernel<H>), dim3((unsigned)(((int64_t)a.M * (a.N / 8) + 255) / 256), a.nbatch), dim3(256), 0, st, a);
}

int64_t steps_of(int64_t k) { return (k + BK - 1) / BK; }
Plan plan_up(int64_t M, int D, int F) { return pick(M, 2 * (int64_t)F, 1, steps_of(D), false); }
Plan plan_down(int64_t M, int D, int F) { return pick(M, D, 1, steps_of(F), true); }
Plan plan_dh(int64_t M, int D, int F) { return pick(M, F, 1, steps_of(D), false); }
Plan plan_dx(int64_t M, int D, int F) { return pick(M, D, 1, 2 * steps_of(F), true); }
Plan plan_dwo(int64_t M, int D, int F) { return pick(D, F, 1, steps_of(M), true); }
Plan plan_dwv(int64_t M, int D, int F) { return pick(F, D, 2, steps_of(M), true); }

bool bad(int64_t M, int D, int F, int act, int dtype) {
  return M < 0 || M > (1 << 30) || D < 8 || F < 8 || D % 8 || F % 8 || D > (1 << 20) || F > (1 << 20) || dtype < 0 || dtype > 1 ||
         (act != FLUXHIP_EPI_GELU_TANH && act != FLUXHIP_EPI_GELU_ERF && act != FLUXHIP_EPI_SILU);
}
bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }

template <bool H>
void forward(const fluxhip_gated_ff_desc* d, hipStream_t st) {
  FfArgs a{};
  a.P[0] = (const char*)d->w_value; a.P[1] = (const char*)d->w_gate; a.Q[0] = a.Q[1] = (const char*)d->x;
  a.out[0] = (char*)d->hidden; a.vout = (char*)d->value; a.gout = (char*)d->gate;
  a.bias[0] = (const char*)d->b_value; a.bias[1] = (const char*)d->b_gate;
  a.ldp = d->D; a.ldq = d->ldx; a.M = (int)d->M; a.N = d->F; a.K = d->D; a.nseg = a.nbatch = 1; a.act = d->act;
  launch<false, false, EPI_UP, H>(a, plan_up(d->M, d->D, d->F), st);
  FfArgs b{};
  b.P[0] = b.P[1] = (const char*)d->w_out; b.Q[0] = b.Q[1] = (const char*)d->hidden; b.out[0] = (char*)d->y;
  b.bias[0] = (const char*)d->b_out;
  b.ldp = b.ldq = d->F; b.ldo = d->D; b.M = (int)d->M; b.N = d->D; b.K = d->F; b.nseg = b.nbatch = 1; b.part = (float*)d->ws;
  launch<false, false, EPI_STORE, H>(b, plan_down(d->M, d->D, d->F), st);
}

template <bool H>
void backward(const fluxhip_gated_ff_grad_desc* d, hipStream_t st) {
  const int64_t M = d->M;
  const int D = d->D, F = d->F;
  {
    FfArgs a{};
    a.P[0] = a.P[1] = (const char*)d->w_out; a.Q[0] = a.Q[1] = (const char*)d->dy;
    a.value = (const char*)d->value; a.gate = (const char*)d->gate; a.vout = (char*)d->dvalue; a.gout = (char*)d->dgate;
    a.ldp = F; a.ldq = d->lddy; a.M = (int)M; a.N = F; a.K = D; a.nseg = a.nbatch = 1; a.act = d->act;
    a.part = d->db_value ? (float*)d->ws : nullptr;
    launch<true, false, EPI_DH, H>(a, plan_dh(M, D, F), st);
    if (d->db_value) {
      launch_colsum_final(a.part, 2 * a.tiles_m, 1, 2, F, d->db_value, d->db_gate, H ? 1 : 0, st);
      const int rows = (int)(M < COLSUM_ROWS ? M : COLSUM_ROWS);
      hipLaunchKernelGGL((ff_colsum_kernel<H>), dim3((D + 2047) / 2048, rows), dim3(256), 0, st, (const uint16_t*)d->dy, d->lddy, (int)M, D,
                         (float*)d->ws);
      launch_colsum_final((const float*)d->ws, rows, 1, 1, D, d->db_out, nullptr, H ? 1 : 0, st);
    }
  }
  if (d->dx) {
    FfArgs a{};
    a.P[0] = (const char*)d->w_value; a.P[1] = (const char*)d->w_gate; a.Q[0] = (const char*)d->dvalue; a.Q[1] = (const char*)d->dgate;
    a.out[0] = (char*)d->dx; a.ldp = D; a.ldq = F; a.ldo = D; a.M = (int)M; a.N = D; a.K = F; a.nseg = 2; a.nbatch = 1; a.part = (float*)d->ws;
    launch<true, false, EPI_STORE, H>(a, plan_dx(M, D, F), st);
  }
  if (d->dw_value) {
    FfArgs a{};
    a.P[0] = a.P[1] = (const char*)d->x; a.Q[0] = (const char*)d->dvalue; a.Q[1] = (const char*)d->dgate;
    a.out[0] = (char*)d->dw_value; a.out[1] = (char*)d->dw_gate;
    a.ldp = d->ldx; a.ldq = F; a.ldo = D; a.M = F; a.N = D; a.K = (int)M; a.nseg = 1; a.nbatch = 2; a.part = (float*)d->ws;
    launch<true, true, EPI_STORE, H>(a, plan_dwv(M, D, F), st);
  }
  if (d->dw_out) {
    FfArgs a{};
    a.P[0] = a.P[1] = (const char*)d->hidden; a.Q[0] = a.Q[1] = (const char*)d->dy; a.out[0] = (char*)d->dw_out;
    a.ldp = F; a.ldq = d->lddy; a.ldo = F; a.M = D; a.N = F; a.K = (int)M; a.nseg = a.nbatch = 1; a.part = (float*)d->ws;
    launch<true, true, EPI_STORE, H>(a, plan_dwo(M, D, F), st);
  }
}

int64_t most(int64_t a, int64_t b) { return a > b ? a : b; }

}  // namespace

extern "C" int64_t fluxhip_gated_ff_ws(int64_t M, int D, int F) {
  if (bad(M, D, F, FLUXHIP_EPI_SILU, 0)) return FLUXHIP_EINVAL;
  return part_bytes(M, D, 1, plan_down(M, D, F));
}
extern "C" int64_t fluxhip_gated_ff_grad_ws(int64_t M, int D, int F) {
  if (bad(M, D, F, FLUXHIP_EPI_SILU, 0)) return FLUXHIP_EINVAL;
  int64_t b = most(((M + 127) / 128) * 2 * 2 * (int64_t)F * 4, (int64_t)COLSUM_ROWS * D * 4);
  b = most(b, part_bytes(M, D, 1, plan_dx(M, D, F)));
  b = most(b, part_bytes(F, D, 2, plan_dwv(M, D, F)));
  return most(b, part_bytes(D, F, 1, plan_dwo(M, D, F)));
}

extern "C" int fluxhip_gated_ff(const fluxhip_gated_ff_desc* d, void* stream) {
  if (!d || bad(d->M, d->D, d->F, d->act, d->dtype)) return FLUXHIP_EINVAL;
  if (d->M == 0) return FLUXHIP_OK;
  const int64_t need = fluxhip_gated_ff_ws(d->M, d->D, d->F);
  if (!d->x || !d->w_value || !d->w_gate || !d->w_out || !d->hidden || !d->y || !d->value != !d->gate || !d->b_value != !d->b_gate ||
      d->ldx < d->D || d->ldx % 8 || d->ldx > (1 << 21) || (need && (!d->ws || d->ws_bytes < need)))
    return FLUXHIP_EINVAL;
  for (const void* p : {d->x, d->w_value, d->w_gate, d->w_out, (const void*)d->hidden, (const void*)d->y, (const void*)d->ws})
    if (misaligned(p)) return FLUXHIP_EINVAL;
  if (d->dtype == 1) forward<true>(d, (hipStream_t)stream);
  else forward<false>(d, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? FLUXHIP_OK : FLUXHIP_ELAUNCH;
}

extern "C" int fluxhip_gated_ff_grad(const fluxhip_gated_ff_grad_desc* d, void* stream) {
  if (!d || bad(d->M, d->D, d->F, d->act, d->dtype)) return FLUXHIP_EINVAL;
  if (d->M == 0) return FLUXHIP_OK;                        // (the caller owns the zeros of an empty sum)
  const int64_t need = fluxhip_gated_ff_grad_ws(d->M, d->D, d->F);
  if (!d->dy || !d->value || !d->gate || !d->w_out || !d->dvalue || !d->dgate || !d->dw_value != !d->dw_gate || !d->db_value != !d->db_gate ||
      !d->db_value != !d->db_out || (d->dx && (!d->w_value || !d->w_gate)) || (d->dw_value && !d->x) || (d->dw_out && !d->hidden) ||
      d->lddy < d->D || d->lddy % 8 || d->lddy > (1 << 21) || (d->dw_value && (d->ldx < d->D || d->ldx % 8 || d->ldx > (1 << 21))) ||
      !d->ws || d->ws_bytes < need)
    return FLUXHIP_EINVAL;
  for (const void* p : {d->dy, d->x, d->value, d->gate, d->hidden, d->w_value, d->w_gate, d->w_out, (const void*)d->dvalue, (const void*)d->dgate,
                        (const void*)d->ws})
    if (misaligned(p)) return FLUXHIP_EINVAL;
  if (d->dtype == 1) backward<true>(d, (hipStream_t)stream);
  else backward<false>(d, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? FLUXHIP_OK : FLUXHIP_ELAUNCH;
}
