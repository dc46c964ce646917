// sdfnn — operands that the product kernels cannot read where they lie: fp32 matrices (split into three bf16 parts) and rows that are not
// 16-byte aligned.  HBM-bound copies; rows are padded with zeros to whole steps.
#pragma once
#include "nn_common.h"

struct PackArgs {
  const void* src;
  int64_t ld;         // elements between rows of src
  int64_t rows, cols;
  char* dst;
  int64_t dst_ld;     // elements between rows of dst
  int64_t plane;      // bytes between the parts
  int64_t pad;        // columns of dst that are written (>= cols), a multiple of 64
};

// What a call needs copied, in one launch: matrix k has the workgroups [first[k], first[k + 1])
constexpr int kPacks = 5;
struct PackBatch {
  PackArgs a[kPacks];
  unsigned first[kPacks + 1];
  int count;
};

// one thread 8 elements.  ES: bytes of an element (4: fp32 into parts)
template <int ES>
__global__ __launch_bounds__(256) void pack_rows_kernel(const PackBatch b) {
  int k = 0;
#pragma unroll
  for (int j = 1; j < kPacks; ++j)
    if (j < b.count && blockIdx.x >= b.first[j]) k = j;
  const PackArgs& a = b.a[k];
  const int64_t groups = a.pad / 8, total = groups * a.rows, threads = (int64_t)(b.first[k + 1] - b.first[k]) * 256;
  for (int64_t i = (int64_t)(blockIdx.x - b.first[k]) * 256 + threadIdx.x; i < total; i += threads) {  // (more than one turn: beyond 2^32 elements)
    const int64_t row = i / groups, c = (i - row * groups) * 8;
    const int64_t left = a.cols - c;
    if constexpr (ES == 4) {
      float v[8];
      load8_n<SDFNN_F32>((const float*)a.src + row * a.ld + c, (int)(left < 0 ? 0 : left < 8 ? left : 8), v);
      store_parts(a.dst + (row * a.dst_ld + c) * 2, a.plane, v);
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
}
