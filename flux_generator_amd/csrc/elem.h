// Element types of the operators that take bfloat16, float16 or float32 tensors (dtype codes of include/fluxhip.h): 8-element
// chunks to and from float32 registers.  Rows need element alignment only; a chunk that a row's end cuts is moved by element.
#pragma once
#include "common.h"

template <int T> struct Elem;

template <bool H>
struct Elem16 {
  typedef uint16_t type;
  static DEVINL float get(const type* p) { return e2f<H>(*p); }
  static DEVINL void put(type* p, float v) { *p = f2e<H>(v); }
  static DEVINL void load8(const type* p, int c, int n, float (&v)[8]) {
    if (c + 8 <= n) {
      uint32_t w[4];
      __builtin_memcpy(w, p + c, 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = e_lo<H>(w[j]);
        v[2 * j + 1] = e_hi<H>(w[j]);
      }
    } else {
      raw8 w;
      fetch8(p, c, n, w);
      open8(w, v);
    }
  }
  typedef u32x4 raw8;                  // a chunk as it lies in memory (loads in flight, converted when used)
  template <bool FULL = false>          // FULL: n is a multiple of 8, no chunk is cut
  static DEVINL void fetch8(const type* p, int c, int n, raw8& w) {
    if (FULL ? c < n : c + 8 <= n) {
      __builtin_memcpy(&w, p + c, 16);
    } else if (!FULL && c < n) {
      uint16_t h[8];                     // the row's last, cut chunk: eight loads at once, the ones behind the end repeat its last element
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = p[min(c + j, n - 1)];
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = c + j < n ? h[j] : (uint16_t)0;
      __builtin_memcpy(&w, h, 16);
    } else {
      w = raw8{0, 0, 0, 0};
    }
  }
  static DEVINL void open8(const raw8& w, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = e_lo<H>(w[j]);
      v[2 * j + 1] = e_hi<H>(w[j]);
    }
  }
  static DEVINL raw8 close8(const float (&v)[8]) {
    return raw8{e_pack<H>(v[0], v[1]), e_pack<H>(v[2], v[3]), e_pack<H>(v[4], v[5]), e_pack<H>(v[6], v[7])};
  }
  template <bool FULL = false>
  static DEVINL void store8(type* p, int c, int n, const float (&v)[8]) {
    if (FULL ? c < n : c + 8 <= n) {
      const raw8 w = close8(v);
      __builtin_memcpy(p + c, &w, 16);
    } else if (!FULL && c < n) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < n) p[c + j] = f2e<H>(v[j]);
    }
  }
};
template <> struct Elem<0> : Elem16<false> {};
template <> struct Elem<1> : Elem16<true> {};
template <>
struct Elem<2> {
  typedef float type;
  static DEVINL float get(const type* p) { return *p; }
  static DEVINL void put(type* p, float v) { *p = v; }
  template <bool FULL = false>
  static DEVINL void load8(const float* p, int c, int n, float (&v)[8]) {
    if (FULL ? c < n : c + 8 <= n) {
      __builtin_memcpy(&v[0], p + c, 16);
      __builtin_memcpy(&v[4], p + c + 4, 16);
    } else if (!FULL && c < n) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = p[min(c + j, n - 1)];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < n ? v[j] : 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
  }
  struct raw8 { float v[8]; };
  template <bool FULL = false>
  static DEVINL void fetch8(const float* p, int c, int n, raw8& w) { load8<FULL>(p, c, n, w.v); }
  static DEVINL void open8(const raw8& w, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = w.v[j];
  }
  template <bool FULL = false>
  static DEVINL void store8(float* p, int c, int n, const float (&v)[8]) {
    if (FULL ? c < n : c + 8 <= n) {
      __builtin_memcpy(p + c, &v[0], 16);
      __builtin_memcpy(p + c + 4, &v[4], 16);
    } else if (!FULL && c < n) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < n) p[c + j] = v[j];
    }
  }
};
