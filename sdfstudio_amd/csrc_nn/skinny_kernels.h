// sdfnn — products of few rows (one token, a handful of rays): y[m, n] = sum_k x[m, k] w[n, k] for m <= 32 (fp32: 64).
//
// Bound by reading the weights once.  They go from HBM straight into the operand registers of the matrix instruction (nothing is read twice,
// so LDS would only add a trip): a wavefront owns 16 rows of w (DUAL: 16 of each projection), a lane 16 bytes of one row at a time; the
// eight wavefronts of a workgroup take turns of 8 KiB along k and join their sums in LDS.  x comes from L2.  fp32 runs on
// v_mfma_f32_16x16x4_f32 as it is - at so few rows its rate suffices - and needs no splitting pass over the weights.  Rows need their element's
// alignment only.  One row, 4096 -> 2 x 16384 -> 4096 bf16: 49 us (5.4 TB/s) and 32 us (4.1 TB/s, of which ~5 us are start and end).
#pragma once
#include "gemm_core.h"

template <int KIND> struct Small;  // KIND 0 bf16, 1 fp16, 2 int8, 3 fp32: one 16-byte fragment a lane, 64 bytes of k an instruction
template <> struct Small<0> {
  typedef f32x4 acc; typedef float el; static constexpr int ES = 2;
  static NN_D acc run(const i32x4 a, const i32x4 b, const acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Small<1> {
  typedef f32x4 acc; typedef float el; static constexpr int ES = 2;
  static NN_D acc run(const i32x4 a, const i32x4 b, const acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <> struct Small<2> {
  typedef i32x4 acc; typedef int el; static constexpr int ES = 1;
  static NN_D acc run(const i32x4 a, const i32x4 b, const acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};
template <> struct Small<3> {
  typedef f32x4 acc; typedef float el; static constexpr int ES = 4;
  static NN_D acc run(const i32x4 a, const i32x4 b, acc c) {
    const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
    // element e of every lane is one k of the lane's four: any assignment of k to lanes serves as long as both operands share it
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(af[e], bf[e], c, 0, 0, 0);
    return c;
  }
};

template <int ES>
NN_D i32x4 load16(const char* p, const int64_t left) {  // 16 bytes, `left` of them valid (zeros behind)
  if (left >= 16) {
    const Bytes<4, ES> raw = *reinterpret_cast<const Bytes<4, ES>*>(p);
    return __builtin_bit_cast(i32x4, raw);
  }
  i32x4 v = {0, 0, 0, 0};
  if (left > 0) {
    char b[16];
#pragma unroll
    for (int e = 0; e < 16 / ES; ++e) {
      if (e * ES < left) __builtin_memcpy(b + e * ES, p + e * ES, ES);
      else __builtin_memset(b + e * ES, 0, ES);
    }
    __builtin_memcpy(&v, b, 16);
  }
  return v;
}

constexpr int kSkinnyWaves = 8;

template <int KIND, int MT, bool DUAL, class EPI>
__global__ __launch_bounds__(kSkinnyWaves * 64) void skinny_kernel(const GemmArgs<EPI> g) {
  typedef Small<KIND> S_;
  const int64_t kb = g.b[0].width;
  constexpr int NP = DUAL ? 2 : 1, U = (DUAL ? 4 : 8) / MT;  // 8 KiB of weights a wavefront and turn (half of it where x takes the registers)
  __shared__ typename S_::el part[kSkinnyWaves][NP * MT][4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int n0 = blockIdx.x * 16;
  // lanes beyond the last row read the last one; their sums are not stored
  const int n = n0 + col < g.N ? n0 + col : g.N - 1;
  const char* w[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) w[p] = g.b[p].p + (int64_t)n * g.b[p].ld + grp * 16;
  const char* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = i * 16 + col < g.M ? i * 16 + col : g.M - 1;
    x[i] = g.a.p + m * g.a.ld + grp * 16;
  }
  typename S_::acc acc[NP][MT];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[p][i][r] = 0;
  // two sets of fragments: the loads of the next turn are under way while this one's are multiplied
  i32x4 wv[2][U][NP], xv[2][U][MT];
  auto load = [&](const int64_t k, auto set) __attribute__((always_inline)) {
    constexpr int S = decltype(set)::value;
    if (k + U * 64 <= kb) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int p = 0; p < NP; ++p) wv[S][u][p] = load16<S_::ES>(w[p] + k + u * 64, 16);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < MT; ++i) xv[S][u][i] = load16<S_::ES>(x[i] + k + u * 64, 16);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t left = kb - (k + u * 64 + grp * 16);
#pragma unroll
        for (int p = 0; p < NP; ++p) wv[S][u][p] = load16<S_::ES>(w[p] + k + u * 64, left);
#pragma unroll
        for (int i = 0; i < MT; ++i) xv[S][u][i] = load16<S_::ES>(x[i] + k + u * 64, left);
      }
    }
  };
  auto multiply = [&](auto set) __attribute__((always_inline)) {
    constexpr int S = decltype(set)::value;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[p][i] = S_::run(wv[S][u][p], xv[S][u][i], acc[p][i]);
  };
  const std::integral_constant<int, 0> s0{};
  const std::integral_constant<int, 1> s1{};
  constexpr int64_t turn = kSkinnyWaves * U * 64;
  int64_t k = wave * (U * 64);
  if (k < kb) load(k, s0);
  for (; k < kb; k += 2 * turn) {
    if (k + turn < kb) load(k + turn, s1);
    multiply(s0);
    if (k + turn >= kb) break;
    if (k + 2 * turn < kb) load(k + 2 * turn, s0);
    multiply(s1);
  }
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[wave][p * MT + i][r][lane] = acc[p][i][r];
  __syncthreads();
  // a lane (grp, col) of a wavefront holds rows n = 4 grp + r of column m = col; a thread joins the eight sums of 8 consecutive n
  if (threadIdx.x < MT * 32) {  // (MT <= 4: 128 of 512 threads)
    const int i = threadIdx.x >> 5, half = (threadIdx.x >> 4) & 1, c = threadIdx.x & 15;
    const int64_t m = i * 16 + c;
    typename S_::el v[NP][8];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        typename S_::el s = 0;
#pragma unroll
        for (int k = 0; k < kSkinnyWaves; ++k) s += part[k][p * MT + i][e & 3][(half * 2 + (e >> 2)) * 16 + c];
        v[p][e] = n0 + half * 8 + e < g.N ? s : (typename S_::el)0;  // the padding columns of a workspace are zeros
      }
    if (m < g.M) {
      const int c = n0 + half * 8;
      if constexpr (DUAL) g.epi.pair(0, m, c, v[0], v[1], g.epi.cols(c), g.epi.fetch(m, g.M, c));
      else g.epi.one(0, m, c, v[0], g.epi.cols(c), g.epi.fetch(m, g.M, c));
    }
  }
}
