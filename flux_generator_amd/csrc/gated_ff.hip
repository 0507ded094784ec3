// Gated feed-forward block, forward and backward, for training adapters (and whole blocks) and for serving.
//
//   value = x Wv^T + bv, gate = x Wg^T + bg, hidden = value act(gate), y = hidden Wo^T + bo
//   dh = dy Wo, dvalue = dh act(gate), dgate = dh value act'(gate)
//   dx = dvalue Wv + dgate Wg, dWv = dvalue^T x, dWg = dgate^T x, dWo = dy^T hidden, db = column sums
//
// Three matrix products of 2 M D F flops forward, six backward (three with frozen weights): MFMA-bound for many tokens, bound by the
// bytes of the weights for few.  One kernel template serves them: out[m][n] = sum_k Q(m, k) P(n, k), where either operand
// lies with k contiguous ("row": activations and nn.Linear weights in the forward pass) or with k strided ("col": the weights of
// the input gradient, both operands of the weight gradients).  Nothing is transposed in memory: a "col" tile is staged as it lies
// and its fragments are read with the transposing LDS read of this chip (ds_read_b64_tr_b16).
//
// Roundings: products and column sums accumulate in float32.  hidden, dvalue and dgate are rounded to the tensors' type before the
// next product, whose MFMA takes 16-bit operands (a second MFMA for a low half would double that product); hidden is formed from the
// unrounded value and gate.  What lies behind such an operand ends 1.4 roundings from the exact result instead of one (bf16 2.3e-3
// against 1.7e-3).
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

enum { EPI_STORE = 0, EPI_UP = 1, EPI_DH = 2 };

struct FfProd {                 // out[m][n] = sum over segments of Q[seg] P[seg]
  const char *P[2], *Q[2];
  char* out;
  int64_t ldp, ldq;             // element strides of the rows of P, Q (out: N)
  int M, N, tiles_m, tiles_n;
};
// One launch: up to three products of one contraction length, their tiles in one list.  The first `full` tiles are whole work
// items, every tile behind them is `splits` items along k whose partial tiles ff_finish_kernel adds.
struct FfArgs {
  FfProd pr[3];
  int nprod, K, nseg, act;      // K: contraction length of a segment
  int full, splits, items;
  float* part;                  // partial tiles of the split items
  const char *bias[2], *value, *gate;
  char *vout, *gout;            // EPI_UP: saved value / gate (or null); EPI_DH: dvalue / dgate
  float* colsum;                // EPI_DH: partial column sums [rows][2][N] (or null)
};

// gfx950 fragment swizzles.  row tile: 64 k = 8 chunks of 16 bytes a row, chunk ^= (row >> 1) & 7.  col tile: one k a row, its
// 32-byte granules (16 columns) ^= f(k): the rows one transposing read touches fall on different banks either way.
DEVINL int col_f(int k) { return (k & 3) | ((k >> 1) & 4); }

// 16 bytes a lane from the buffer straight into LDS at dst + 16 lane (dst wave-uniform; m0 carries it).  Inline asm because the
// compiler, which cannot tell the two stages apart, would wait for all of these before every transposing LDS read; it has no
// output register, and the main loop's own vmcnt waits cover it.  (s_nop: no resource register may be younger than five wait states
// if a vector instruction wrote it, which the compiler does not look after inside inline asm.)
DEVINL void dma16(u32x4 rs, uint32_t voff, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(voff), "s"(rs) : "memory", "m0");
}

template <bool COL, int BI, int NP>     // BI: indices of the tile (col: 128 or 256), NP: 1 KiB pieces per wave
struct Stager {
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
        chunk[j & 1] = c;                                  // (the swizzle alternates with the piece)
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

template <int ACT>
DEVINL float act_f(float x) {
  return ACT == FLUXHIP_EPI_GELU_TANH ? gelu_tanh_f(x) : ACT == FLUXHIP_EPI_SILU ? silu_f(x) : gelu_erf_f(x);
}
// act(x) and act'(x).  silu: p (1 + x (1 - p)), p = sigmoid x.  tanh form: p + x p (1 - p) u', p = sigmoid(2 u).
// erf form: Phi(x) + x phi(x), Phi from the same rational erfc as gelu_erf_f with its exponential shared.
template <int ACT>
DEVINL void act_grad(float x, float& f, float& df) {
  if constexpr (ACT == FLUXHIP_EPI_SILU) {
    const float p = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
    f = x * p;
    df = p * (1.0f + x * (1.0f - p));
  } else if constexpr (ACT == FLUXHIP_EPI_GELU_TANH) {
    constexpr float c0 = -2.0f * 0.7978845608028654f * 1.4426950408889634f, c1 = c0 * 0.044715f;
    const float x2 = fminf(x * x, 1e30f);                  // (an infinite square would meet 1 - p = 0 below)
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
// eight at once: one branch on the activation for all of them, not one an element (first product of 10170 x 2040 from 120, all
// three outputs: 70 -> 61 us with its second)
template <class F>
DEVINL void each_act(int act, F f) {
  if (act == FLUXHIP_EPI_SILU) f(std::integral_constant<int, FLUXHIP_EPI_SILU>{});
  else if (act == FLUXHIP_EPI_GELU_TANH) f(std::integral_constant<int, FLUXHIP_EPI_GELU_TANH>{});
  else f(std::integral_constant<int, FLUXHIP_EPI_GELU_ERF>{});
}

DEVINL void swap16(float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}

// A wave's tile is NF n by MF m fragments of 16 (128, 96 or 64 columns - long pieces of output rows - by 64 rows), the block's
// WN x WM waves; block tile BM x BP, of which every wave stages PP and QP pieces of 1 KiB a step.  NF = 8 and 6: 256 rows by 256 or
// 192 columns, eight waves (two a SIMD), one block a CU; NF = 4: 128 square, four waves, two blocks a CU.
template <int NF, int EPI>
struct Geo {
  static constexpr int MF = 4, BP = 32 * NF, BM = NF == 4 ? 128 : 256, WN = 2, WM = BM / 64, NW = WN * WM, BN = EPI == EPI_UP ? BP / 2 : BP;
  static constexpr int PP = BP / 8 / NW, QP = BM / 8 / NW, OPB = BP * BK * 2, STAGE = OPB + BM * BK * 2;
};

// 16 rows by 64 columns of 16-bit elements: as the fragments lie (a, b: row = lane & 15, 64 bytes of it each) <-> as they are moved
// (a: rows 0..7, b: rows 8..15, a whole 128-byte line of each).  Lanes 8..15 of every 16 trade their a for the b of lanes 0..7.
DEVINL void trade8(u32x4& a, u32x4& b) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int x = (int)a[e], y = (int)b[e];
    a[e] = (uint32_t)__builtin_amdgcn_update_dpp(x, y, 0x128, 0xf, 0xc, false);      // row_ror:8
    b[e] = (uint32_t)__builtin_amdgcn_update_dpp(y, x, 0x128, 0xf, 0x3, false);
  }
}

struct Item { int p, m0, n0, s_lo, ns, slot; };            // slot: of the partial tile, -1 for a whole one
template <int NF, int EPI>
DEVINL Item item_of(const FfArgs& a, int it) {
  typedef Geo<NF, EPI> G;
  Item r;
  const int sps = (a.K + BK - 1) / BK, total = sps * a.nseg;
  int t = it, split = 0;
  r.slot = -1;
  r.s_lo = 0;
  r.ns = total;
  if (it >= a.full) {
    const int u = it - a.full, q = u / a.splits;
    t = a.full + q;
    if (a.splits > 1) {
      split = u - q * a.splits;
      r.slot = u;
      r.s_lo = (uint32_t)(total * split) / (uint32_t)a.splits;       // (total <= 2^25, splits <= 16)
      r.ns = (uint32_t)(total * (split + 1)) / (uint32_t)a.splits - r.s_lo;
    }
  }
  r.p = 0;
  while (r.p + 1 < a.nprod && t >= a.pr[r.p].tiles_m * a.pr[r.p].tiles_n) t -= a.pr[r.p].tiles_m * a.pr[r.p].tiles_n, ++r.p;
  // bands of four row tiles: neighbouring items share operand tiles
  const int tm = a.pr[r.p].tiles_m, tn = a.pr[r.p].tiles_n, band = t / (4 * tn), bm = min(4, tm - band * 4);
  t -= band * 4 * tn;
  r.m0 = (band * 4 + t % bm) * G::BM;
  r.n0 = t / bm * G::BN;
  return r;
}

// writes J m fragments of a wave's tile, from the j0-th.  Rows outside, their columns inside: one row's pieces (of one or several
// tensors) are written together, which keeps the pages in reach of the CU's TLB (dvalue / dgate of 16384 x 5120 from 1280: 372 -> 325 us
// against the other order), and pairs of fragments are traded into whole 128-byte lines (from 128: 200 -> 163 us; a plain copy in
// that tiling: 157 -> 140).
template <int NF, int EPI, bool H, int J>
DEVINL void epilogue(const FfArgs& a, const FfProd& pr, f32x4 (&acc)[NF][J], int m0, int n0, int wm, int wn, int j0) {
  typedef Geo<NF, EPI> G;
  constexpr int HALVES = EPI == EPI_UP ? NF / 4 : NF / 2;  // pairs of fragments = 32 columns (EPI_UP with NF = 6: and a single one)
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int nb = n0 + wn * (EPI == EPI_UP ? NF * 8 : NF * 16) + (q & 1) * 16 + (q >> 1) * 8;    // the lane's 8 columns behind the swap
  const int mb = m0 + wm * (G::MF * 16) + j0 * 16 + c;
  // Traded pairs move through buffer resources whose range check ends the rows; a lane behind the last column takes an offset
  // beyond them all (256 rows of at most 2^21 bytes).  c0: the pair's first column from the wave's.
  const uint32_t row_bytes = (uint32_t)pr.N * 2;
  const int nx = nb + (c >> 3) * 32;                       // traded: the lane's 8 columns; its rows: c & 7, and 8 behind that
  const uint32_t lane_at = (uint32_t)(wm * (G::MF * 16) + j0 * 16 + (c & 7)) * row_bytes + (uint32_t)(nx - n0) * 2;
  auto rows_of = [&](const void* t) {
    return __builtin_amdgcn_make_buffer_rsrc((char*)t + ((int64_t)m0 * pr.N + n0) * 2, 0, (int)(min(pr.M - m0, G::BM) * row_bytes), 0x00020000);
  };
  auto at = [&](int c0, int j) { return (nx + c0 < pr.N ? lane_at + c0 * 2 : 1u << 31) + (uint32_t)(j * 16) * row_bytes; };
  typedef uint16_t E;
  typedef Elem<H ? 1 : 0> El;
  auto take = [&](auto i, auto j, float (&d)[8]) {         // fragments i, i + 1 -> 8 neighbouring n
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      d[e] = acc[i][j][e];
      d[4 + e] = acc[i + 1][j][e];
      swap16(d[e], d[4 + e]);
    }
  };
  auto move8 = [&](__amdgpu_buffer_rsrc_t t, const u32x4 (&r)[2], int c0, int j) {        // stores a traded pair
    const uint32_t o = at(c0, j);
    __builtin_amdgcn_raw_buffer_store_b128(r[0], t, o, 0, 0);
    __builtin_amdgcn_raw_buffer_store_b128(r[1], t, o + 8 * row_bytes, 0, 0);
  };
  if constexpr (EPI == EPI_UP) {
    auto finish = [&](int n, float (&v)[8], float (&g)[8], float (&h)[8]) {
      if (a.bias[0] && n < pr.N) {
        El::load8((const E*)a.bias[0] + n, 0, 8, h);
        for (int e = 0; e < 8; ++e) v[e] += h[e];
        El::load8((const E*)a.bias[1] + n, 0, 8, h);
        for (int e = 0; e < 8; ++e) g[e] += h[e];
      }
      each_act(a.act, [&](auto act) {
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = v[e] * act_f<act>(g[e]);
      });
    };
    auto put = [&](int m, int n, float (&v)[8], float (&g)[8]) {
      float h[8];
      finish(n, v, g, h);
      if (n < pr.N && m < pr.M) {
        const int64_t o = (int64_t)m * pr.N + n;
        El::store8((E*)pr.out + o, 0, 8, h);
        if (a.vout) {
          El::store8((E*)a.vout + o, 0, 8, v);
          El::store8((E*)a.gout + o, 0, 8, g);
        }
      }
    };
    static_for<0, J>([&](auto j) {
      float v[8], g[8];
      if constexpr (HALVES == 2) {
        u32x4 rh[2], rv[2], rg[2];
        static_for<0, 2>([&](auto ih) {
          float h[8];
          take(std::integral_constant<int, 2 * ih>{}, j, v);
          take(std::integral_constant<int, 2 * ih + NF / 2>{}, j, g);
          finish(nb + ih * 32, v, g, h);
          rh[ih] = El::close8(h);
          rv[ih] = El::close8(v);
          rg[ih] = El::close8(g);
        });
        trade8(rh[0], rh[1]);
        move8(rows_of(pr.out), rh, 0, j);
        if (a.vout) {
          trade8(rv[0], rv[1]);
          move8(rows_of(a.vout), rv, 0, j);
          trade8(rg[0], rg[1]);
          move8(rows_of(a.gout), rg, 0, j);
        }
      } else {
        take(std::integral_constant<int, 0>{}, j, v);
        take(std::integral_constant<int, NF / 2>{}, j, g);
        put(mb + j * 16, nb, v, g);
      }
    });
    if constexpr (NF / 2 % 2) {                            // the odd fragment pairs with itself 16 rows on: 8 columns of either row
      static_assert(J % 2 == 0, "two row fragments at a time");
      constexpr int i = NF / 2 - 1;
      static_for<0, J / 2>([&](auto jh) {
        constexpr int j = 2 * jh;
        float v[8], g[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = acc[i][j][e]; v[4 + e] = acc[i][j + 1][e];
          g[e] = acc[i + NF / 2][j][e]; g[4 + e] = acc[i + NF / 2][j + 1][e];
          swap16(v[e], v[4 + e]);
          swap16(g[e], g[4 + e]);
        }
        put(mb + (j + (q & 1)) * 16, nb - (q & 1) * 16 + i * 16, v, g);
      });
    }
  } else if constexpr (EPI == EPI_DH) {
    // The saved value and gate of the next 16 rows are in flight while these are worked on (large tiles: from the middle of the
    // work, where registers are free - on repeated operands and without bias sums 16384 x 5120 from 1280 took 298 us, from its
    // start 314 with 94 spilled registers; small ones 163 / 168 from 128.  On changing operands 312, with bias sums 325.)  The
    // large kernel stands at 256 registers and still spills 11 (bf16) or 17 (f16) of them.  64 columns a pass, whose sums fit the
    // registers.
    constexpr int PASS = 2;
    static_assert(HALVES % PASS == 0, "whole lines");
    const auto value = rows_of(a.value), gate = rows_of(a.gate), vout = rows_of(a.vout), gout = rows_of(a.gout);
    static_for<0, HALVES / PASS>([&](auto pass) {
      u32x4 rv[2][2], rg[2][2];
      const int np = nb + pass * (PASS * 32);
      auto fetch = [&](auto j) {
        const uint32_t o = at(pass * (PASS * 32), j);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          rv[j & 1][k] = __builtin_amdgcn_raw_buffer_load_b128(value, o + k * 8 * row_bytes, 0, 0);
          rg[j & 1][k] = __builtin_amdgcn_raw_buffer_load_b128(gate, o + k * 8 * row_bytes, 0, 0);
        }
      };
      fetch(std::integral_constant<int, 0>{});
      float sv[PASS][8] = {}, sg[PASS][8] = {};
      static_for<0, J>([&](auto j) {
        const int m = mb + j * 16;
        u32x4 (&qv)[2] = rv[j & 1], (&qg)[2] = rg[j & 1];
        if constexpr (NF == 4 && j + 1 < J) fetch(std::integral_constant<int, j + 1>{});
        trade8(qv[0], qv[1]);
        trade8(qg[0], qg[1]);
        static_for<0, PASS>([&](auto ih) {
          const bool ok = np + ih * 32 < pr.N && m < pr.M;
          float d[8], v[8], g[8];
          take(std::integral_constant<int, 2 * (pass * PASS + ih)>{}, j, d);
          El::open8(qv[ih], v);
          El::open8(qg[ih], g);
          each_act(a.act, [&](auto act) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float f, df;
              act_grad<act>(g[e], f, df);
              g[e] = d[e] * v[e] * df;
              v[e] = d[e] * f;
            }
          });
          qv[ih] = El::close8(v);
          qg[ih] = El::close8(g);
          if (a.colsum) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              sv[ih][e] += ok ? v[e] : 0.f;
              sg[ih][e] += ok ? g[e] : 0.f;
            }
          }
        });
        if constexpr (NF > 4 && j + 1 < J) fetch(std::integral_constant<int, j + 1>{});
        trade8(qv[0], qv[1]);
        trade8(qg[0], qg[1]);
        move8(vout, qv, pass * (PASS * 32), j);
        move8(gout, qg, pass * (PASS * 32), j);
        // column sums over the wave's rows: 16 lanes in a fixed order; per 16 rows where the launch has split tiles
        if (a.colsum && (j == J - 1 || a.splits > 1)) {
          static_for<0, PASS>([&](auto ih) {
            const int n = np + ih * 32;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              sv[ih][e] = row16_sum(sv[ih][e]);
              sg[ih][e] = row16_sum(sg[ih][e]);
            }
            if (c == 0 && n < pr.N) {
              const int64_t row = (int64_t)(m0 / G::BM) * G::WM + wm;
              float* p = a.colsum + (a.splits > 1 ? row * G::MF + j0 + j : row) * 2 * pr.N + n;
              Elem<2>::store8(p, 0, 8, sv[ih]);
              Elem<2>::store8(p + pr.N, 0, 8, sg[ih]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sv[ih][e] = sg[ih][e] = 0.f;
          });
        }
      });
    });
  } else {
    const auto out = rows_of(pr.out);
    u32x4 w[2];
    static_for<0, J>([&](auto j) {
      static_for<0, HALVES>([&](auto ih) {
        const int n = nb + ih * 32;
        float d[8], b[8];
        take(std::integral_constant<int, 2 * ih>{}, j, d);
        if (a.bias[0] && n < pr.N) {
          El::load8((const E*)a.bias[0] + n, 0, 8, b);
          for (int e = 0; e < 8; ++e) d[e] += b[e];
        }
        w[ih & 1] = El::close8(d);
        if constexpr (ih & 1) {
          trade8(w[0], w[1]);
          move8(out, w, (ih - 1) * 32, j);
        } else if constexpr (ih + 1 == HALVES) {           // (NF = 6: an odd one)
          if (n < pr.N && mb + j * 16 < pr.M) __builtin_memcpy((E*)pr.out + (int64_t)(mb + j * 16) * pr.N + n, &w[0], 16);
        }
      });
    });
  }
}

template <int NF, bool PC, bool QC, int EPI, bool H>
__global__ __launch_bounds__(NF == 4 ? 256 : 512, 2) void ff_gemm_kernel(FfArgs a) {
  typedef Geo<NF, EPI> G;
  constexpr int MF = G::MF, OPB = G::OPB, STAGE = G::STAGE, PT = G::PP + G::QP;
  static_assert(!PC || NF != 6, "a col tile's swizzle wants 128 or 256 columns");
  __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / G::WN, wn = wave % G::WN;

  // block -> first item: the blocks of one XCD (id mod 8) take neighbouring items, so its CUs share operand tiles in their L2;
  // then every gridDim-th
  int it0 = blockIdx.x;
  {
    const int n = gridDim.x, per = n >> 3, rem = n & 7, x = it0 & 7;
    it0 = x * per + min(x, rem) + (it0 >> 3);
  }

  // ---- what is being fetched: a stream of steps that runs two ahead of the products, across items
  // EPI_UP: P is two half tiles, value rows then gate rows, staged by the first and the second half of the waves
  constexpr int HW = G::NW / 2;
  Stager<PC, G::BN, G::PP> sp;
  Stager<QC, G::BM, G::QP> sq;
  int f_it = it0, f_s = 0, f_ns = 0, f_lo = 0;
  const char *pb[2], *qb[2];
  const int sps = (a.K + BK - 1) / BK;
  auto f_item = [&]() {
    const Item r = item_of<NF, EPI>(a, f_it);
    const FfProd& pr = a.pr[r.p];
    f_s = 0;
    f_ns = r.ns;
    f_lo = r.s_lo;
    pb[0] = EPI == EPI_UP && wave >= HW ? pr.P[1] : pr.P[0];
    pb[1] = pr.P[1];
    qb[0] = pr.Q[0];
    qb[1] = pr.Q[1];
    sp.init(lane, (EPI == EPI_UP ? wave % HW : wave) * G::PP, pr.ldp, r.n0, pr.N, a.K);
    sq.init(lane, wave * G::QP, pr.ldq, r.m0, pr.M, a.K);
  };
  f_item();
  auto open = [&]() {                                      // resources of the stream's next step
    if (f_s == f_ns && f_it < a.items) {
      f_it += gridDim.x;
      if (f_it < a.items) f_item();
    }
    const bool on = f_it < a.items;                        // behind the last step: empty resources, the pieces write zeros
    const int st = f_lo + f_s, seg = a.nseg > 1 && st >= sps ? 1 : 0, k0 = (st - seg * sps) * BK;
    sp.step(seg ? pb[1] : pb[0], k0, on);
    sq.step(seg ? qb[1] : qb[0], k0, on);
    f_s += on ? 1 : 0;
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  auto piece = [&](int j, int buf) {                       // j-th of the wave's pieces of a stage
    const uint32_t d = lds0 + buf * STAGE;
    if (j < G::PP) sp.piece(j, d + wave * (G::PP * 1024));
    else sq.piece(j - G::PP, d + OPB + wave * (G::QP * 1024));
  };

  // ---- products
  Reader<PC, G::BP> rp;
  Reader<QC, G::BM> rq;
  rp.init(lane);
  rq.init(lane);
  f32x4 acc[NF][MF];                                       // [n fragment][m fragment]
  bf16x8 fp[NF], fq[2][MF];
  auto read_p = [&](int i, int buf, int ks) {              // fragments of k half ks of a stage
    const int row = EPI == EPI_UP ? (i >= NF / 2 ? G::BP / 2 : 0) + wn * (NF * 8) + (i % (NF / 2)) * 16 : wn * (NF * 16) + i * 16;
    fp[i] = rp.read(smem + buf * STAGE, row, ks);
  };
  auto read_q = [&](int j, int buf, int ks) { fq[ks][j] = rq.read(smem + buf * STAGE + OPB, wm * (MF * 16) + j * 16, ks); };
  auto mul = [&](auto i, int ks) {
    static_for<0, MF>([&](auto j) { acc[i][j] = mma<H>(fp[i], fq[ks][j], acc[i][j]); });
  };

  // Main loop: two LDS stages of 64 k, a step = two halves of 32 k, a half = NF groups of MF products.  Behind group i the P
  // fragment it used is free and is read for the next half (Q fragments alternate between two sets), so every LDS read has
  // about NF groups to land.  Once per step, behind the first group of the second half (it covers the last reads' latency),
  // the waves meet: all have the stage in registers and all pieces of the next stage are in LDS; the stage is then refilled
  // with the step after the next, whose loads have a whole step to land.  The stream does not stop at an item's end: the next
  // item's first stages land while this one's tile is written.
  open();
  static_for<0, PT>([&](auto j) { piece(j, 0); });
  open();
  static_for<0, PT>([&](auto j) { piece(j, 1); });
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PT) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  int buf = 0;
  for (int it = it0; it < a.items; it += gridDim.x) {
    const Item r = item_of<NF, EPI>(a, it);
    static_for<0, MF>([&](auto j) { read_q(j, buf, 0); });   // (read again behind an epilogue: it needs the registers)
    static_for<0, NF>([&](auto i) { read_p(i, buf, 0); });
    static_for<0, NF>([&](auto i) { static_for<0, MF>([&](auto j) { acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f}; }); });
    for (int s = 0; s < r.ns; ++s) {
      static_for<0, NF>([&](auto i) {
        mul(i, 0);
        read_p(i, buf, 1);
        if constexpr (i < MF) read_q(i, buf, 1);
        __builtin_amdgcn_sched_barrier(0);
      });
      open();
      static_for<0, NF>([&](auto i) {
        mul(i, 1);
        if constexpr (i == 0) {
          __builtin_amdgcn_sched_barrier(0);
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        static_for<i * PT / NF, (i + 1) * PT / NF>([&](auto e) { piece(e, buf); });
        read_p(i, buf ^ 1, 0);                             // (behind the very last step: zeros, not used)
        if constexpr (i < MF) read_q(i, buf ^ 1, 0);
        __builtin_amdgcn_sched_barrier(0);
      });
      buf ^= 1;
    }
    if (r.slot >= 0) {                                     // a partial tile, fragments as they lie in the registers
      f32x4* p = (f32x4*)a.part + (((int64_t)r.slot * G::NW + wave) * (NF * MF)) * 64 + lane;
      static_for<0, MF>([&](auto j) {                      // (rows behind the end are not looked at)
        if (r.m0 + (wm * MF + j) * 16 < a.pr[r.p].M) static_for<0, NF>([&](auto i) { p[(i * MF + j) * 64] = acc[i][j]; });
      });
    } else {
      epilogue<NF, EPI, H, MF>(a, a.pr[r.p], acc, r.m0, r.n0, wm, wn, 0);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // no piece outlives the kernel
}

// adds a split tile's partials in split order and writes it; a block takes one m fragment of each wave's tile.  Few blocks where few
// rows are: bound by latency, so four splits' loads are in flight (forward of 36 tokens, 1064 -> 240, on repeated operands: 16.5 us, with
// two 21.2; on changing ones 18.8, 6.4 of them here)
template <int NF, int EPI, bool H>
__global__ __launch_bounds__(NF == 4 ? 256 : 512) void ff_finish_kernel(FfArgs a) {
  typedef Geo<NF, EPI> G;
  constexpr int MF = G::MF;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int tile = blockIdx.x / MF, j0 = blockIdx.x % MF;
  const Item r = item_of<NF, EPI>(a, a.full + tile * a.splits);
  // (rows behind the end: only their zero column sums)
  if (r.m0 + ((wave / G::WN) * MF + j0) * 16 >= a.pr[r.p].M && !(EPI == EPI_DH && a.colsum)) return;
  f32x4 acc[NF][1];
  static_for<0, NF>([&](auto i) { acc[i][0] = f32x4{0.f, 0.f, 0.f, 0.f}; });
  const f32x4* p = (const f32x4*)a.part + (((int64_t)tile * a.splits * G::NW + wave) * (NF * MF) + j0) * 64 + lane;
#pragma unroll 4
  for (int z = 0; z < a.splits; ++z) {
    static_for<0, NF>([&](auto i) { acc[i][0] += p[i * MF * 64]; });
    p += (int64_t)G::NW * (NF * MF) * 64;
  }
  epilogue<NF, EPI, H, 1>(a, a.pr[r.p], acc, r.m0, r.n0, wave / G::WN, wave % G::WN, j0);
}

// ---- one or two tokens (serving): bound by reading the weights once.  A wave owns one output column - its value and gate row, or
// its row of the out weight - and reads the rows whole, 1 KiB at a time and eight loads ahead, against the tokens' vectors from
// L1; products are float32 FMAs.  4096 -> 10240 at one token: 26.0 us for 168 MB (6.4 TB/s), back 15.4 us.  (Three tokens and
// more: the tiles above with their split along k are faster: 63 us forward at four tokens, 90 this way.)
constexpr int GEMV = 2;
template <bool DUAL, int MT, bool H>
__global__ __launch_bounds__(256) void ff_gemv_kernel(FfArgs a) {
  typedef uint16_t E;
  typedef Elem<H ? 1 : 0> El;
  constexpr int R = DUAL ? 2 : 1, U = 8 / R;
  const FfProd& pr = a.pr[0];
  const int n = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, nch = a.K / 8;
  if (n >= pr.N) return;
  const E *p[R], *q[MT];
#pragma unroll
  for (int i = 0; i < R; ++i) p[i] = (const E*)pr.P[i] + (int64_t)n * pr.ldp;
#pragma unroll
  for (int m = 0; m < MT; ++m) q[m] = (const E*)pr.Q[0] + (int64_t)m * pr.ldq;
  float acc[R][MT] = {};
  for (int c0 = lane; c0 < nch; c0 += 64 * U) {
    u32x4 rp[U][R], rq[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = min(c0 + u * 64, nch - 1) * 8;         // a chunk behind the end repeats the last one and becomes zeros
#pragma unroll
      for (int i = 0; i < R; ++i) rp[u][i] = __builtin_nontemporal_load((const u32x4*)(p[i] + c));
#pragma unroll
      for (int m = 0; m < MT; ++m) rq[u][m] = *(const u32x4*)(q[m] + c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u == 0) __builtin_amdgcn_sched_barrier(0);       // (all loads before the first use)
      const bool on = c0 + u * 64 < nch;
#pragma unroll
      for (int i = 0; i < R; ++i) rp[u][i] = on ? rp[u][i] : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        rq[u][m] = on ? rq[u][m] : u32x4{0, 0, 0, 0};
        float v[8], x[8];
        El::open8(rq[u][m], x);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          El::open8(rp[u][i], v);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[i][m] = __builtin_fmaf(v[e], x[e], acc[i][m]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    float v = wave_sum(acc[0][m]), g = wave_sum(acc[R - 1][m]);
    if (lane) continue;
    if (a.bias[0]) v += e2f<H>(((const E*)a.bias[0])[n]);
    const int64_t o = (int64_t)m * pr.N + n;
    if constexpr (DUAL) {
      if (a.bias[0]) g += e2f<H>(((const E*)a.bias[1])[n]);
      if (a.vout) {
        ((E*)a.vout)[o] = f2e<H>(v);
        ((E*)a.gout)[o] = f2e<H>(g);
      }
      each_act(a.act, [&](auto act) { v *= act_f<act>(g); });
    }
    ((E*)pr.out)[o] = f2e<H>(v);
  }
}

template <bool DUAL, bool H>
void launch_gemv(const FfArgs& a, hipStream_t st) {
  const dim3 grid((a.pr[0].N + 3) / 4);
  if (a.pr[0].M == 1) hipLaunchKernelGGL((ff_gemv_kernel<DUAL, 1, H>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((ff_gemv_kernel<DUAL, 2, H>), grid, dim3(256), 0, st, a);
}

// column sums of [M][N] (first stage; colsum.h adds the partial rows): a wave takes 512 columns of every gridDim.y-th row
template <bool H>
__global__ __launch_bounds__(64) void ff_colsum_kernel(const uint16_t* x, int64_t ld, int M, int N, float* part) {
  typedef Elem<H ? 1 : 0> El;
  const int c = (blockIdx.x * 64 + threadIdx.x) * 8;
  if (c >= N) return;
  float s[8] = {}, v[8];
#pragma unroll 16
  for (int m = blockIdx.y; m < M; m += gridDim.y) {
    El::load8(x + m * ld + c, 0, 8, v);
    for (int e = 0; e < 8; ++e) s[e] += v[e];
  }
  Elem<2>::store8(part + (int64_t)blockIdx.y * N + c, 0, 8, s);
}

// How a launch is cut: the estimated time of every way, the least wins.  256-square tiles run one block a CU at 1.5 us a step (64 k)
// of all CUs, 128-square ones two a CU at 1.13 us (16384 x 5120 x 1280 and 512 x 20480 x 4096, bf16).  What the epilogue moves
// comes on top at 4.9 TB/s - all of it for the large tiles, whose CU has nothing else to run, a bit more than half for the small
// ones (dvalue / dgate of 16384 x 5120 on repeated operands, large / small: from 128 178 / 163 us, from 1280 298 / 341).  Whole
// rounds of tiles run as they are; the tiles of the last, broken round are split along k over the idle CUs where that pays for
// writing and reading their float32 partials (0.117 us a 256-square split tile at 4.5 TB/s over the chip, and 8 us for the second
// launch).
// 256 x 192 tiles (row operands only; 1.2 us) where they fill the CUs better: EPI_UP of 512 x 10240 from 4096 is 214 of them in
// 96 to 109 us (the estimate says 81: it prices loops whose weights lie in the caches, these come from HBM), or 160 squares in 118;
// its product back, split, 57 to 60 and 9.5 adding up, with squares 51 and 15.
struct Plan { int nf, full, splits, items; };
struct Dims { int64_t M, N; };                             // output of a product; EPI_UP: N = F
int64_t tile_rows(int nf) { return nf == 4 ? 128 : 256; }
Plan pick(const Dims* d, int n, int64_t steps, int epi, bool rows_only = false) {
  Plan best{};
  double least = 1e30;
  for (int nf = 8; nf >= 4; nf -= 2) {
    if (nf == 6 && !rows_only) continue;
    const int64_t bm = tile_rows(nf), bn = epi == EPI_UP ? 16 * nf : 32 * nf, slots = nf == 4 ? 512 : 256;
    const double step = nf == 8 ? 1.5 : nf == 6 ? 1.2 : 1.13, part = 0.117 / 65536 * bm * 32 * nf;
    int64_t tiles = 0;
    double out = 0, rows = 0, padded = 0;
    for (int i = 0; i < n; ++i) {
      const int64_t tm = (d[i].M + bm - 1) / bm;
      tiles += tm * ((d[i].N + bn - 1) / bn);
      out += (double)d[i].M * d[i].N;
      rows += (double)d[i].M;
      padded += (double)(tm * bm);
    }
    const double moved = out * (epi == EPI_DH ? 8 : epi == EPI_UP ? 4 : 2) / 4.9e6 * (nf == 4 ? 0.57 : 1.0);
    const int64_t full = tiles / slots * slots, tail = tiles - full, most = nf == 6 && epi == EPI_UP ? 1 : 16;
    for (int64_t s = 1; s <= most && s <= steps; ++s) {
      const double us = moved + step * steps * ((double)(full / slots) + (double)((tail * s + slots - 1) / slots) / s) +
                        (s > 1 ? 8 + tail * s * part * (rows / padded) : 0);
      if (us < least) {
        least = us;
        best = {nf, (int)full, (int)s, (int)(full + tail * s)};
      }
      if (!tail) break;
    }
  }
  return best;
}
int64_t part_bytes(const Plan& p) { return p.splits > 1 ? (int64_t)(p.items - p.full) * tile_rows(p.nf) * (32 * p.nf) * 4 : 0; }

template <int NF, bool PC, bool QC, int EPI, bool H>
void launch_nf(FfArgs& a, const Plan& p, hipStream_t st) {
  typedef Geo<NF, EPI> G;
  constexpr int slots = NF == 4 ? 512 : 256;
  for (int i = 0; i < a.nprod; ++i) {
    a.pr[i].tiles_m = (a.pr[i].M + G::BM - 1) / G::BM;
    a.pr[i].tiles_n = (a.pr[i].N + G::BN - 1) / G::BN;
  }
  hipLaunchKernelGGL((ff_gemm_kernel<NF, PC, QC, EPI, H>), dim3(p.items < slots ? p.items : slots), dim3(G::NW * 64), 0, st, a);
  if constexpr (!(NF == 6 && EPI == EPI_UP))
    if (p.splits > 1)
      hipLaunchKernelGGL((ff_finish_kernel<NF, EPI, H>), dim3((p.items - p.full) / p.splits * G::MF), dim3(G::NW * 64), 0, st, a);
}
template <bool PC, bool QC, int EPI, bool H>
void launch(FfArgs& a, const Plan& p, hipStream_t st) {
  a.full = p.full;
  a.splits = p.splits;
  a.items = p.items;
  if (p.nf == 8) launch_nf<8, PC, QC, EPI, H>(a, p, st);
  else if (p.nf == 4) launch_nf<4, PC, QC, EPI, H>(a, p, st);
  else if constexpr (!PC && !QC) launch_nf<6, PC, QC, EPI, H>(a, p, st);
}

int64_t steps_of(int64_t k) { return (k + BK - 1) / BK; }
Plan plan_up(int64_t M, int D, int F) { const Dims d{M, F}; return pick(&d, 1, steps_of(D), EPI_UP, true); }
Plan plan_down(int64_t M, int D, int F) { const Dims d{M, D}; return pick(&d, 1, steps_of(F), EPI_STORE, true); }
Plan plan_dh(int64_t M, int D, int F) { const Dims d{M, F}; return pick(&d, 1, steps_of(D), EPI_DH); }
Plan plan_dx(int64_t M, int D, int F) { const Dims d{M, D}; return pick(&d, 1, 2 * steps_of(F), EPI_STORE); }
Plan plan_dw(int64_t M, int D, int F) { const Dims d[3] = {{F, D}, {F, D}, {D, F}}; return pick(d, 3, steps_of(M), EPI_STORE); }
Plan plan_dw2(int64_t M, int D, int F) { const Dims d[2] = {{F, D}, {F, D}}; return pick(d, 2, steps_of(M), EPI_STORE); }
Plan plan_dw1(int64_t M, int D, int F) { const Dims d{D, F}; return pick(&d, 1, steps_of(M), EPI_STORE); }
int64_t colsum_rows(int64_t M, const Plan& p) {
  return (M + tile_rows(p.nf) - 1) / tile_rows(p.nf) * (tile_rows(p.nf) / 64) * (p.splits > 1 ? 4 : 1);
}
constexpr int COLSUM_ROWS = 1024;                          // (16384 x 1280, both stages alone: 15.1 us, with 512 17.4)

bool bad(int64_t M, int D, int F, int act, int dtype) {
  return M < 0 || M > (1 << 30) || D < 8 || F < 8 || D % 8 || F % 8 || D > (1 << 20) || F > (1 << 20) || dtype < 0 || dtype > 1 ||
         (M / 128 + 1) * ((D > F ? D : F) / 64 + 1) > (1 << 30) ||       // (tiles are counted in 32 bits)
         (act != FLUXHIP_EPI_GELU_TANH && act != FLUXHIP_EPI_GELU_ERF && act != FLUXHIP_EPI_SILU);
}
bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }

FfProd prod(const void* P, const void* Q, void* out, int64_t ldp, int64_t ldq, int64_t M, int64_t N) {
  FfProd r{};
  r.P[0] = r.P[1] = (const char*)P;
  r.Q[0] = r.Q[1] = (const char*)Q;
  r.out = (char*)out;
  r.ldp = ldp; r.ldq = ldq; r.M = (int)M; r.N = (int)N;
  return r;
}

template <bool H>
void forward(const fluxhip_gated_ff_desc* d, hipStream_t st) {
  const int64_t M = d->M;
  const int D = d->D, F = d->F;
  FfArgs a{};
  a.pr[0] = prod(d->w_value, d->x, d->hidden, D, d->ldx, M, F);
  a.pr[0].P[1] = (const char*)d->w_gate;
  a.nprod = a.nseg = 1; a.K = D; a.act = d->act; a.part = (float*)d->ws;
  a.vout = (char*)d->value; a.gout = (char*)d->gate;
  a.bias[0] = (const char*)d->b_value; a.bias[1] = (const char*)d->b_gate;
  if (M <= GEMV) launch_gemv<true, H>(a, st);
  else launch<false, false, EPI_UP, H>(a, plan_up(M, D, F), st);
  FfArgs b{};
  b.pr[0] = prod(d->w_out, d->hidden, d->y, F, F, M, D);
  b.nprod = b.nseg = 1; b.K = F; b.part = (float*)d->ws; b.bias[0] = (const char*)d->b_out;
  if (M <= GEMV) launch_gemv<false, H>(b, st);
  else launch<false, false, EPI_STORE, H>(b, plan_down(M, D, F), st);
}

template <bool H>
void backward(const fluxhip_gated_ff_grad_desc* d, hipStream_t st) {
  const int64_t M = d->M;
  const int D = d->D, F = d->F;
  {
    const Plan p = plan_dh(M, D, F);
    FfArgs a{};
    a.pr[0] = prod(d->w_out, d->dy, nullptr, F, d->lddy, M, F);
    a.nprod = a.nseg = 1; a.K = D; a.act = d->act;
    a.value = (const char*)d->value; a.gate = (const char*)d->gate; a.vout = (char*)d->dvalue; a.gout = (char*)d->dgate;
    a.part = (float*)((char*)d->ws + (d->db_value ? colsum_rows(M, p) * 2 * F * 4 : 0));
    a.colsum = d->db_value ? (float*)d->ws : nullptr;
    launch<true, false, EPI_DH, H>(a, p, st);
    if (d->db_value) {                                     // dy's columns: few rows are added up by the same launch as they are
      Extra e{d->dy, d->db_out, d->lddy, M, D, 0};
      if (M > 2 * COLSUM_ROWS) {
        float* part = (float*)d->ws + colsum_rows(M, p) * 2 * F;
        hipLaunchKernelGGL((ff_colsum_kernel<H>), dim3((D + 511) / 512, COLSUM_ROWS), dim3(64), 0, st, (const uint16_t*)d->dy, d->lddy, (int)M, D,
                           part);
        e = Extra{part, d->db_out, D, COLSUM_ROWS, D, 1};
      }
      launch_colsum_final(a.colsum, colsum_rows(M, p), 1, 2, F, d->db_value, d->db_gate, H ? 1 : 0, st, e);
    }
  }
  if (d->dx) {
    FfArgs a{};
    a.pr[0] = prod(d->w_value, d->dvalue, d->dx, D, F, M, D);
    a.pr[0].P[1] = (const char*)d->w_gate;
    a.pr[0].Q[1] = (const char*)d->dgate;
    a.nprod = 1; a.nseg = 2; a.K = F; a.part = (float*)d->ws;
    launch<true, false, EPI_STORE, H>(a, plan_dx(M, D, F), st);
  }
  if (d->dw_value || d->dw_out) {                          // all weight gradients in one launch
    FfArgs a{};
    if (d->dw_value) {
      a.pr[a.nprod++] = prod(d->x, d->dvalue, d->dw_value, d->ldx, F, F, D);
      a.pr[a.nprod++] = prod(d->x, d->dgate, d->dw_gate, d->ldx, F, F, D);
    }
    if (d->dw_out) a.pr[a.nprod++] = prod(d->hidden, d->dy, d->dw_out, F, d->lddy, D, F);
    a.nseg = 1; a.K = (int)M; a.part = (float*)d->ws;
    launch<true, true, EPI_STORE, H>(a, a.nprod == 3 ? plan_dw(M, D, F) : a.nprod == 2 ? plan_dw2(M, D, F) : plan_dw1(M, D, F), st);
  }
}

int64_t most(int64_t a, int64_t b) { return a > b ? a : b; }

}  // namespace

extern "C" int64_t fluxhip_gated_ff_ws(int64_t M, int D, int F) {
  if (bad(M, D, F, FLUXHIP_EPI_SILU, 0)) return FLUXHIP_EINVAL;
  return M <= GEMV ? 0 : most(part_bytes(plan_up(M, D, F)), part_bytes(plan_down(M, D, F)));
}
extern "C" int64_t fluxhip_gated_ff_grad_ws(int64_t M, int D, int F) {
  if (bad(M, D, F, FLUXHIP_EPI_SILU, 0)) return FLUXHIP_EINVAL;
  const Plan dh = plan_dh(M, D, F);
  int64_t b = colsum_rows(M, dh) * 2 * F * 4 + most(part_bytes(dh), (int64_t)COLSUM_ROWS * D * 4);
  b = most(b, part_bytes(plan_dx(M, D, F)));
  b = most(b, most(part_bytes(plan_dw(M, D, F)), part_bytes(plan_dw2(M, D, F))));
  return most(b, part_bytes(plan_dw1(M, D, F)));
}

extern "C" int fluxhip_gated_ff(const fluxhip_gated_ff_desc* d, void* stream) {
  if (!d || bad(d->M, d->D, d->F, d->act, d->dtype)) return FLUXHIP_EINVAL;
  if (d->M == 0) return FLUXHIP_OK;
  const int64_t need = fluxhip_gated_ff_ws(d->M, d->D, d->F);
  if (!d->x || !d->w_value || !d->w_gate || !d->w_out || !d->hidden || !d->y || !d->value != !d->gate || !d->b_value != !d->b_gate ||
      d->ldx < d->D || d->ldx % 8 || d->ldx > (1 << 21) || (need && (!d->ws || d->ws_bytes < need)))
    return FLUXHIP_EINVAL;
  for (const void* p : {d->x, d->w_value, d->w_gate, d->w_out, (const void*)d->value, (const void*)d->gate, (const void*)d->hidden,
                        (const void*)d->y, (const void*)d->ws})
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
                        (const void*)d->dx, (const void*)d->dw_value, (const void*)d->dw_gate, (const void*)d->dw_out, (const void*)d->ws})
    if (misaligned(p)) return FLUXHIP_EINVAL;
  if (d->dtype == 1) backward<true>(d, (hipStream_t)stream);
  else backward<false>(d, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? FLUXHIP_OK : FLUXHIP_ELAUNCH;
}
