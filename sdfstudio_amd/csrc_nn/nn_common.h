// sdfnn — shared device / host helpers of the gated feed-forward block's kernels (gfx950 only).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/sdfnn.h"

#define NN_D __device__ __forceinline__
#define NN_HD __host__ __device__ __forceinline__

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// ---- element types of the C ABI (SDFNN_F32 / _BF16 / _F16)
template <int DT> struct Elem;
template <> struct Elem<SDFNN_F32> { typedef float type; };
template <> struct Elem<SDFNN_BF16> { typedef __bf16 type; };
template <> struct Elem<SDFNN_F16> { typedef _Float16 type; };
template <int DT> using elem_t = typename Elem<DT>::type;
NN_HD constexpr int elem_size(const int dt) { return dt == SDFNN_F32 ? 4 : 2; }

// Eight consecutive elements as one (fp32: two) 16-byte access.  The address needs the element's own alignment only: gfx950 runs with
// unaligned access on, so rows of an odd width keep their wide loads and only the last, partial group of a row goes element by element.
template <int N, int ALIGN>
struct __attribute__((packed, aligned(ALIGN))) Bytes { uint32_t w[N]; };

template <int DT> using Raw8 = Bytes<elem_size(DT) * 2, elem_size(DT)>;  // eight elements as they lie in memory

template <int DT>
NN_D void widen8(const Raw8<DT>& raw, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (DT == SDFNN_F32) v[i] = __builtin_bit_cast(float, (uint32_t)raw.w[i]);
    else if constexpr (DT == SDFNN_BF16) v[i] = __builtin_bit_cast(float, i & 1 ? raw.w[i / 2] & 0xffff0000u : raw.w[i / 2] << 16);
    else v[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(raw.w[i / 2] >> (16 * (i & 1))));
  }
}
template <int DT>
NN_D Raw8<DT> raw8(const elem_t<DT>* p) { return *reinterpret_cast<const Raw8<DT>*>(p); }
// the same with `n` valid elements and zeros behind them
template <int DT>
NN_D Raw8<DT> raw8_n(const elem_t<DT>* p, const int n) {
  if (n >= 8) return raw8<DT>(p);
  Raw8<DT> raw;
  if constexpr (DT == SDFNN_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw.w[i] = i < n ? ((const uint32_t*)p)[i] : 0u;
  } else {
    const uint16_t* q = (const uint16_t*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      raw.w[i] = 2 * i < n ? q[2 * i] : 0u;
      if (2 * i + 1 < n) raw.w[i] |= (uint32_t)q[2 * i + 1] << 16;
    }
  }
  return raw;
}
template <int DT>
NN_D void load8(const elem_t<DT>* p, float (&v)[8]) { widen8<DT>(raw8<DT>(p), v); }
template <int DT>
NN_D void load8_n(const elem_t<DT>* p, const int n, float (&v)[8]) { widen8<DT>(raw8_n<DT>(p, n), v); }
// two values rounded to a 16-bit type, as one word
template <class E>
NN_D uint32_t pack2(const float a, const float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef E e2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), e2));
}
template <int DT>
NN_D void store8(elem_t<DT>* p, const float (&v)[8]) {
  Raw8<DT> raw;
  if constexpr (DT == SDFNN_F32) {
    __builtin_memcpy(&raw, v, 32);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) raw.w[i] = pack2<elem_t<DT>>(v[2 * i], v[2 * i + 1]);
  }
  *reinterpret_cast<Raw8<DT>*>(p) = raw;
}
template <int DT>
NN_D void store8_n(elem_t<DT>* p, const int n, const float (&v)[8]) {
  if (n >= 8) return store8<DT>(p, v);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = (elem_t<DT>)v[i];
}

// x = p0 + p1 + p2, each a bf16, of eight values: three rows of 16 bytes, `plane` bytes apart.  The largest finite values would round to infinity as
// bf16: p0 is held at the largest bf16, the rest goes to p1.  Of a value that is not finite p2 at least is NaN.
NN_D void store_parts(char* p, const int64_t plane, const float (&v)[8]) {
  uint32_t h[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    constexpr float top = 0x1.fep127f;
    float a = v[2 * i], b = v[2 * i + 1];
    h[0][i] = pack2<__bf16>(__builtin_amdgcn_fmed3f(a, -top, top), __builtin_amdgcn_fmed3f(b, -top, top));
#pragma unroll
    for (int k = 1; k < 3; ++k) {
      a -= __builtin_bit_cast(float, h[k - 1][i] << 16), b -= __builtin_bit_cast(float, h[k - 1][i] & 0xffff0000u);
      h[k][i] = pack2<__bf16>(a, b);
    }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) *(uint4*)(p + k * plane) = *(const uint4*)h[k];
}

// ---- activations of the gated block and their derivatives.  FAST (16-bit results): the hardware's exponential and reciprocal, one ulp of
// fp32 each, the exponent rounded to fp32 before it.  fp32 results: the part of x log2(e) that this rounding loses goes back in to first
// order, and one Newton step follows the reciprocal; x <= 0 there, cut at -128, where the exponential has long been 0 (it ends with the normal numbers,
// below -87.3), so that nothing is left to multiply a large z with.
template <bool FAST>
NN_D float nn_exp(float x) {
  if constexpr (FAST) return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f);
  x = __builtin_amdgcn_fmed3f(x, -128.0f, 0.0f);
  const float t = x * 1.44269504088896340736f;
  const float lost = fmaf(x, 1.44269504088896340736f, -t) + x * 1.92596299112661746887e-8f;
  const float e = __builtin_amdgcn_exp2f(t);
  return fmaf(e, lost * 0.69314718055994530942f, e);
}
template <bool FAST>
NN_D float nn_recip(const float x) {  // 1 <= x < 2^127
  const float r = __builtin_amdgcn_rcpf(x);
  if constexpr (FAST) return r;
  return fmaf(fmaf(-x, r, 1.0f), r, r);
}
// Phi(z), the normal distribution function.  For x = |z|:
//   16-bit results: Phi(-x) = 2^(P(x) - x^2 / (2 ln 2)), P of degree 10 fitted to log2(erfcx(x / sqrt 2) / 2) on [0, 13.2], behind which Phi lies
//   below the normal numbers: off by 6e-7 at most and by 1.3e-4 (2^-13) of its value, one exponential and no reciprocal.  The epilogues that call it are
//   bound by such instructions.
//   fp32 results: Phi(-x) = exp(-x^2 / 2) t P(t) / 2 with t = 1 / (1 + 0.4 x / sqrt 2), P of degree 8 fitted for the smallest relative error over
//   x >= 0 (1.3e-7).
template <bool FAST>
NN_D float nn_phi(const float z) {
  const float x = fabsf(z);
  float p, c;
  if constexpr (FAST) {
    const float y = __builtin_amdgcn_fmed3f(x, 0.0f, 13.2f);
    p = -1.88042928e-10f;
    p = fmaf(p, y, 9.56122825e-09f);
    p = fmaf(p, y, -1.5210604e-07f);
    p = fmaf(p, y, -4.91635603e-07f);
    p = fmaf(p, y, 5.22080772e-05f);
    p = fmaf(p, y, -0.000877389451f);
    p = fmaf(p, y, 0.0083174957f);
    p = fmaf(p, y, -0.0536075197f);
    p = fmaf(p, y, 0.262596905f);
    p = fmaf(p, y, -1.15117240f);
    p = fmaf(p, y, -0.999998510f);
    c = __builtin_amdgcn_exp2f(fmaf(z * z, -0.72134752044448170368f, p));
  } else {
    const float t = nn_recip<FAST>(fmaf(0.28284271247461900976f, x, 1.0f));
    p = 0.0502621084f;
    p = fmaf(p, t, -0.182901412f);
    p = fmaf(p, t, 0.169085339f);
    p = fmaf(p, t, -0.00560746621f);
    p = fmaf(p, t, 0.141431406f);
    p = fmaf(p, t, 0.168541983f);
    p = fmaf(p, t, 0.207842693f);
    p = fmaf(p, t, 0.225669593f);
    p = fmaf(p, t, 0.225675866f);
    c = 0.5f * nn_exp<FAST>(-0.5f * z * z) * t * p;
  }
  return z < 0.0f ? c : 1.0f - c;
}
// a = act(z), d = act'(z)
template <bool FAST, int ACT>
NN_D void act_both(const float z, float& a, float& d) {
  if constexpr (ACT == SDFNN_SILU && FAST) {
    const float s = nn_recip<FAST>(1.0f + nn_exp<FAST>(-z));
    a = z * s;
    d = s * (1.0f + z * (1.0f - s));
  } else if constexpr (ACT == SDFNN_SILU) {  // the sigmoid of |z| and of -|z| from exp(-|z|), which does not overflow
    const float e = nn_exp<FAST>(-fabsf(z)), r = nn_recip<FAST>(1.0f + e), q = e * r;
    const float s = z < 0.0f ? q : r;
    a = z * s;
    d = s * (1.0f + z * (z < 0.0f ? r : q));
  } else if constexpr (ACT == SDFNN_GELU) {
    const float phi = nn_phi<FAST>(z);
    a = z * phi;
    d = fmaf(z * 0.39894228040143267794f, nn_exp<FAST>(-0.5f * z * z), phi);
  } else {
    a = z < 0.0f ? 0.0f : z;  // (a NaN stays one)
    d = z > 0.0f ? 1.0f : 0.0f;
  }
}
// of eight values: one branch on the activation for all of them
template <bool FAST, int ACT>
NN_D void act8_of(float (&z)[8], float (&d)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) act_both<FAST, ACT>(z[i], z[i], d[i]);
}
template <bool FAST>
NN_D void act8(const int act, float (&z)[8], float (&d)[8]) {
  if (act == SDFNN_SILU) act8_of<FAST, SDFNN_SILU>(z, d);
  else if (act == SDFNN_GELU) act8_of<FAST, SDFNN_GELU>(z, d);
  else act8_of<FAST, SDFNN_RELU>(z, d);
}
template <bool FAST, int ACT>
NN_D void act8_of(float (&z)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float d;
    act_both<FAST, ACT>(z[i], z[i], d);  // (what the derivative alone needs is dropped by the compiler)
  }
}
template <bool FAST>
NN_D void act8(const int act, float (&z)[8]) {
  if (act == SDFNN_SILU) act8_of<FAST, SDFNN_SILU>(z);
  else if (act == SDFNN_GELU) act8_of<FAST, SDFNN_GELU>(z);
  else act8_of<FAST, SDFNN_RELU>(z);
}

// ---- host side
void sdfnn_set_error(const char* fmt, ...);
#define NN_REQUIRE(cond, ...)        \
  do {                               \
    if (!(cond)) {                   \
      sdfnn_set_error(__VA_ARGS__);  \
      return -1;                     \
    }                                \
  } while (0)
#define NN_LAUNCHED(what)                                                       \
  do {                                                                          \
    const hipError_t e_ = hipGetLastError();                                    \
    if (e_ != hipSuccess) {                                                     \
      sdfnn_set_error("%s: launch failed: %s", what, hipGetErrorString(e_));    \
      return -2;                                                                \
    }                                                                           \
  } while (0)
NN_HD constexpr int64_t round_up(const int64_t n, const int64_t m) { return (n + m - 1) / m * m; }
NN_HD constexpr int64_t ceil_div(const int64_t n, const int64_t m) { return (n + m - 1) / m; }
