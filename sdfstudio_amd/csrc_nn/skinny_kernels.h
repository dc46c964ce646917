// sdfnn — products of few rows (one token, a handful of rays): y[m, n] = sum_k x[m, k] w[n, k] for m <= 32 (fp32: 64).
//
// Bound by reading the weights once.  They go from HBM straight into the operand registers of the matrix instruction (nothing is read twice,
// so LDS would only add a trip): a wavefront owns 16 rows of w (DUAL: 16 of each projection), a lane 16 bytes of one row at a time; the
// eight wavefronts of a workgroup take turns of 8 KiB along k and join their sums in LDS.  x comes from L2.  PAIR: a row of x is the sum of two rows of
// the operand, m and m + M / 2 (a value in two 16-bit numbers): both are multiplied, the join adds them.  fp32 runs on
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

template <int KIND, int MT, bool DUAL, bool PAIR, class EPI>
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
    const int64_t m = i * 16 + c, M = PAIR ? g.M / 2 : g.M;
    if (m >= M) return;
    const int j = PAIR ? (int)(m + M) >> 4 : 0, d = PAIR ? (int)(m + M) & 15 : 0;  // (m + M < 16 MT)
    typename S_::el v[NP][8];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        typename S_::el s = 0;
#pragma unroll
        for (int k = 0; k < kSkinnyWaves; ++k) s += part[k][p * MT + i][e & 3][(half * 2 + (e >> 2)) * 16 + c];
        if constexpr (PAIR) {
#pragma unroll
          for (int k = 0; k < kSkinnyWaves; ++k) s += part[k][p * MT + j][e & 3][(half * 2 + (e >> 2)) * 16 + d];
        }
        v[p][e] = n0 + half * 8 + e < g.N ? s : (typename S_::el)0;  // the padding columns of a workspace are zeros
      }
    const int n8 = n0 + half * 8;
    if constexpr (DUAL) g.epi.pair(0, m, n8, v[0], v[1], g.epi.cols(n8), g.epi.fetch(m, M, n8));
    else g.epi.one(0, m, n8, v[0], g.epi.cols(n8), g.epi.fetch(m, M, n8));
  }
}

// ---- the backward pass of few fp32 rows, on the same instruction: the tiles would have to split all weights into parts first.
// y[m, n] = sum_k x[m, k] w[k, n], the weights' k down the rows.  A workgroup owns 64 columns (256 bytes of a row), its four wavefronts take turns
// of 16 rows: a lane loads 16 bytes of four of them, and its four elements are operands of four instructions (columns 4 c + e of instruction e), so that
// a lane ends up with 16 consecutive columns of one m.  b[1] follows b[0] along k from row `turn` (a multiple of 16) on; g.nk, g.per: in units of 16
// rows; where columns are few k is split over blockIdx.y.  16 x 4096 x 16384: the gradient of a 43 us (6.3 TB/s, a part
// from the last-level cache), dx 103 us (5.2 TB/s); 64 rows, where the instructions take as long as the loads, 114 and 221 us.
constexpr int kDownWaves = 4;

template <int MT, class EPI>
__global__ __launch_bounds__(kDownWaves * 64) void skinny_down_kernel(const GemmArgs<EPI> g) {
  __shared__ float part[kDownWaves][MT][16][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int n0 = blockIdx.x * 64, n = n0 + col * 4;
  const int64_t left_n = ((int64_t)g.N - n) * 4;
  const char* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {  // lanes beyond the last row read the last one; their sums are not stored
    const int64_t m = i * 16 + col < g.M ? i * 16 + col : g.M - 1;
    x[i] = g.a.p + m * g.a.ld;
  }
  f32x4 acc[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  f32x4 wv[2][4], xv[2][MT];
  auto load = [&](const int s, auto set) __attribute__((always_inline)) {
    constexpr int S = decltype(set)::value;
    const int64_t k0 = (int64_t)s * 16;
    const bool after = k0 >= g.turn;
    const char* p = after ? g.b[1].p : g.b[0].p;
    const int64_t ld = after ? g.b[1].ld : g.b[0].ld, rows = after ? g.b[1].rows : g.b[0].rows, at = k0 - (after ? g.turn : 0);
    const int64_t k = k0 + grp * 4, row = at + grp * 4;
    if (at + 16 <= rows && n0 + 64 <= g.N && (k0 + 16) * 4 <= g.a.width) {
#pragma unroll
      for (int j = 0; j < 4; ++j) wv[S][j] = __builtin_bit_cast(f32x4, load16<4>(p + (row + j) * ld + (int64_t)n * 4, 16));
#pragma unroll
      for (int i = 0; i < MT; ++i) xv[S][i] = __builtin_bit_cast(f32x4, load16<4>(x[i] + k * 4, 16));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        wv[S][j] = __builtin_bit_cast(f32x4, load16<4>(p + (row + j) * ld + (int64_t)n * 4, row + j < rows ? left_n : 0));
#pragma unroll
      for (int i = 0; i < MT; ++i) xv[S][i] = __builtin_bit_cast(f32x4, load16<4>(x[i] + k * 4, g.a.width - k * 4));
    }
  };
  auto multiply = [&](auto set) __attribute__((always_inline)) {
    constexpr int S = decltype(set)::value;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[S][j][e], xv[S][i][j], acc[i][e], 0, 0, 0);
  };
  const std::integral_constant<int, 0> s0{};
  const std::integral_constant<int, 1> s1{};
  const int first = blockIdx.y * g.per, last = first + g.per < g.nk ? first + g.per : g.nk;
  int s = first + wave;
  if (s < last) load(s, s0);
  for (; s < last; s += 2 * kDownWaves) {
    if (s + kDownWaves < last) load(s + kDownWaves, s1);
    multiply(s0);
    if (s + kDownWaves >= last) break;
    if (s + 2 * kDownWaves < last) load(s + 2 * kDownWaves, s0);
    multiply(s1);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave][i][4 * r + e][lane] = acc[i][e][r];
  __syncthreads();
  for (int id = threadIdx.x; id < MT * 128; id += kDownWaves * 64) {
    const int i = id >> 7, half = (id >> 6) & 1, from = id & 63;
    const int64_t m = i * 16 + (from & 15);
    const int c = n0 + (from >> 4) * 16 + half * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = 0.0f;
#pragma unroll
      for (int k = 0; k < kDownWaves; ++k) v[e] += part[k][i][half * 8 + e][from];
    }
    if (m < g.M) g.epi.one((int)blockIdx.y, m, c, v, g.epi.cols(c), g.epi.fetch(m, g.M, c));
  }
}

// w[r, c] = sum_m p[m, r] x[m, c] of few rows m: bound by writing w.  64 x 64 results a wavefront, four wavefronts side by side along c; both operands are
// read 16 bytes a lane (rows 4 i + a, columns 4 i + e of instruction (a, e)), so that a lane ends up with runs of four columns.  The operands are small
// and come from L2.  16 x 4096 x 16384: 805 MB of gradients in 220 us (3.7 TB/s).
struct OuterArgs {
  Operand p, x;  // rows m; width: bytes of a row that exist
  int64_t M;
  StoreEpi<SDFNN_F32> to;
};
__global__ __launch_bounds__(256) void outer_kernel(const OuterArgs g) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int64_t r0 = (int64_t)blockIdx.y * 64, c0 = ((int64_t)blockIdx.x * 4 + wave) * 64;
  const int64_t left_p = g.p.width - (r0 + col * 4) * 4, left_x = g.x.width - (c0 + col * 4) * 4;
  const char *p = g.p.p + (r0 + col * 4) * 4, *x = g.x.p + (c0 + col * 4) * 4;
  f32x4 acc[4][4];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[a][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t k = 0; k < g.M; k += 4) {
    const int64_t m = k + grp;
    const bool there = m < g.M;
    const f32x4 pv = __builtin_bit_cast(f32x4, load16<4>(p + m * g.p.ld, there ? left_p : 0));
    const f32x4 xv = __builtin_bit_cast(f32x4, load16<4>(x + m * g.x.ld, there ? left_x : 0));
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[a][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(pv[a], xv[e], acc[a][e], 0, 0, 0);
  }
  const int64_t c = c0 + col * 4;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const float v[4] = {acc[a][0][r], acc[a][1][r], acc[a][2][r], acc[a][3][r]};
      g.to.four(r0 + grp * 16 + r * 4 + a, c, v);
    }
}
