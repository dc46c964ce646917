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

template <int DT>
NN_D void load8(const elem_t<DT>* p, float (&v)[8]) {
  typedef elem_t<DT> T;
  constexpr int NW = 8 * sizeof(T) / 4;
  const Bytes<NW, sizeof(T)> raw = *reinterpret_cast<const Bytes<NW, sizeof(T)>*>(p);
  T t[8];
  __builtin_memcpy(t, &raw, sizeof(t));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
}
template <int DT>
NN_D void store8(elem_t<DT>* p, const float (&v)[8]) {
  typedef elem_t<DT> T;
  constexpr int NW = 8 * sizeof(T) / 4;
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
  Bytes<NW, sizeof(T)> raw;
  __builtin_memcpy(&raw, t, sizeof(t));
  *reinterpret_cast<Bytes<NW, sizeof(T)>*>(p) = raw;
}
// the same with `n` valid elements (zeros behind them on a load)
template <int DT>
NN_D void load8_n(const elem_t<DT>* p, const int n, float (&v)[8]) {
  if (n >= 8) return load8<DT>(p, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
}
template <int DT>
NN_D void store8_n(elem_t<DT>* p, const int n, const float (&v)[8]) {
  if (n >= 8) return store8<DT>(p, v);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = (elem_t<DT>)v[i];
}

// ---- activations of the gated block and their derivatives.  FAST (16-bit results): the hardware's exponential and reciprocal, one ulp of
// fp32 each; fp32 results use the library's expf / erff.
template <bool FAST>
NN_D float nn_exp(const float x) {
  if constexpr (FAST) return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f);
  else return expf(x);
}
template <bool FAST>
NN_D float nn_recip(const float x) {
  if constexpr (FAST) return __builtin_amdgcn_rcpf(x);
  else return 1.0f / x;
}
// a = act(z), d = act'(z)
template <bool FAST>
NN_D void act_both(const int act, const float z, float& a, float& d) {
  if (act == SDFNN_SILU) {
    const float s = nn_recip<FAST>(1.0f + nn_exp<FAST>(-z));
    a = z * s;
    d = s * (1.0f + z * (1.0f - s));
  } else if (act == SDFNN_GELU) {
    const float phi = 0.5f * erfcf(-0.70710678118654752440f * z);
    a = z * phi;
    d = phi + z * 0.39894228040143267794f * nn_exp<FAST>(-0.5f * z * z);
  } else {
    a = z < 0.0f ? 0.0f : z;  // (a NaN stays one)
    d = z > 0.0f ? 1.0f : 0.0f;
  }
}
template <bool FAST>
NN_D float act_only(const int act, const float z) {
  if (act == SDFNN_SILU) return z * nn_recip<FAST>(1.0f + nn_exp<FAST>(-z));
  if (act == SDFNN_GELU) return z * (0.5f * erfcf(-0.70710678118654752440f * z));
  return z < 0.0f ? 0.0f : z;
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
