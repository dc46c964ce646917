// sdfnn — operands that the product kernels cannot read where they lie: fp32 matrices (split into three bf16 parts), rows that are not 16-byte
// aligned, and matrices whose k runs down the columns (transposed).  HBM-bound copies; k is padded with zeros to whole steps.
#pragma once
#include "nn_common.h"

// x = p0 + p1 + p2, each a bf16.  The largest finite values round to infinity as bf16: they are cut instead.  A value that is not finite is
// its first part alone.
NN_D void split3(const float x, uint16_t& p0, uint16_t& p1, uint16_t& p2) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, x);
  uint16_t h = __builtin_bit_cast(uint16_t, (__bf16)x);
  const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
  if ((h & 0x7fffu) == 0x7f80u && finite) h = (uint16_t)(bits >> 16);
  const float r = finite ? x - __builtin_bit_cast(float, (uint32_t)h << 16) : 0.0f;
  p0 = h;
  p1 = __builtin_bit_cast(uint16_t, (__bf16)r);
  p2 = __builtin_bit_cast(uint16_t, (__bf16)(r - __builtin_bit_cast(float, (uint32_t)p1 << 16)));
}

struct PackArgs {
  const void* src;
  int64_t ld;         // elements between rows of src
  int64_t rows, cols;
  char* dst;
  int64_t dst_ld;     // elements between rows of dst
  int64_t plane;      // bytes between the parts
  int64_t pad;        // columns of dst that are written (>= cols, resp. >= rows when transposed), a multiple of 64
};

// rows as they are: one thread 8 elements.  ES: bytes of an element (4: fp32 into parts)
template <int ES>
__global__ __launch_bounds__(256) void pack_rows_kernel(const PackArgs a) {
  const int64_t groups = a.pad / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= groups * a.rows) return;
  const int64_t row = i / groups, c = (i - row * groups) * 8;
  const int64_t left = a.cols - c;
  if constexpr (ES == 4) {
    float v[8];
    load8_n<SDFNN_F32>((const float*)a.src + row * a.ld + c, (int)(left < 0 ? 0 : left < 8 ? left : 8), v);
    alignas(16) uint16_t p[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) split3(v[e], p[0][e], p[1][e], p[2][e]);
#pragma unroll
    for (int k = 0; k < 3; ++k) *(uint4*)(a.dst + k * a.plane + (row * a.dst_ld + c) * 2) = *(const uint4*)p[k];
  } else {
    const char* s = (const char*)a.src + (row * a.ld + c) * ES;
    char b[8 * ES];
    if (left >= 8) {
      const Bytes<2 * ES, ES> raw = *reinterpret_cast<const Bytes<2 * ES, ES>*>(s);
      __builtin_memcpy(b, &raw, 8 * ES);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e < left) __builtin_memcpy(b + e * ES, s + e * ES, ES);
        else __builtin_memset(b + e * ES, 0, ES);
      }
    }
    Bytes<2 * ES, 8> raw;
    __builtin_memcpy(&raw, b, 8 * ES);
    *reinterpret_cast<Bytes<2 * ES, 8>*>(a.dst + (row * a.dst_ld + c) * ES) = raw;
  }
}

// transposed: dst[c][r] = src[r][c].  64 x 64 tiles through LDS (odd row length: both directions hit all banks), 16-byte reads and writes
template <bool F32>
__global__ __launch_bounds__(256) void pack_transposed_kernel(const PackArgs a) {
  typedef typename std::conditional<F32, float, uint16_t>::type T;
  __shared__ T tile[64][F32 ? 65 : 66];
  const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (t >> 3) + 32 * i, c = (t & 7) * 8;
    T v[8];
    const int64_t left = r0 + r < a.rows ? a.cols - (c0 + c) : 0;
    const T* s = (const T*)a.src + (r0 + r) * a.ld + c0 + c;
    if (left >= 8) {
      typedef Bytes<2 * sizeof(T), sizeof(T)> V;
      const V raw = *reinterpret_cast<const V*>(s);
      __builtin_memcpy(v, &raw, sizeof(v));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < left ? s[e] : (T)0;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) tile[r][c + e] = v[e];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = (t >> 3) + 32 * i, r = (t & 7) * 8;
    if (c0 + c >= a.cols || r0 + r >= a.pad) continue;
    char* d = a.dst + ((c0 + c) * a.dst_ld + r0 + r) * 2;
    if constexpr (F32) {
      alignas(16) uint16_t p[3][8];
#pragma unroll
      for (int e = 0; e < 8; ++e) split3(tile[r + e][c], p[0][e], p[1][e], p[2][e]);
#pragma unroll
      for (int k = 0; k < 3; ++k) *(uint4*)(d + k * a.plane) = *(const uint4*)p[k];
    } else {
      alignas(16) uint16_t p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = tile[r + e][c];
      *(uint4*)d = *(const uint4*)p;
    }
  }
}
