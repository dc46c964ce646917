// sdfnn — matrix products C[m, n] = sum_k A[m, k] B[n, k] on the matrix cores, both operands with their k adjacent in memory.
//
// One kernel serves 16-bit floats (v_mfma_f32_32x32x16), 8-bit integers (v_mfma_i32_32x32x32) and fp32 as three bf16 parts a value: to it a
// row is a string of bytes, a step is 128 of them (64 16-bit or 128 8-bit elements of k), and an operand fragment is 16 bytes a lane
// whatever they hold.
//   * Tiles go from HBM / L2 to LDS without passing registers (buffer_load_dwordx4 ... lds), double buffered: one barrier a step; the loads
//     of step s + 1 are issued when step s begins.  A row past the end of a matrix, and the bytes past k in the last step, lie outside the
//     buffer's range, where the load returns zeros: ragged sizes cost no branch in the loop.
//   * LDS rows are 128 bytes = half of the banks, so a fragment read (32 rows at one k) would hit the same 16 bytes of every row: the
//     16-byte pieces of row r are stored in the order piece ^ (r & 7) instead (the permutation is applied to the GLOBAL address of the
//     load, LDS itself is written in order), which spreads the reads over all banks.
//   * The weights' rows (n) are operand A of the instruction and the tokens' rows (m) operand B: a lane then owns ONE m and runs of 4
//     consecutive n, and one v_permlane32_swap a register pair makes runs of 8, i.e. 16-byte stores.
//   * fp32: x = p0 + p1 + p2 with p0 = bf16(x), p1 = bf16(x - p0), p2 = bf16(x - p0 - p1) holds all 24 bits; of the nine products of two
//     such sums the six largest are formed (the rest is below 2^-24 of |a b|), the small ones first: six passes over k that differ
//     in the pair of parts they read.
//   * Workgroups are numbered so that the ones that run at the same time on one XCD (ids equal mod 8) form a square-ish patch of tiles and
//     share their operands in that XCD's L2.
//   * Few tiles: k is split over workgroups; raw sums go to the workspace and a second kernel adds them in order and applies the epilogue.
#pragma once
#include "nn_common.h"

struct Operand {
  const char* p;
  int64_t ld;     // bytes between rows
  int64_t plane;  // bytes between the parts of an fp32 matrix
};

template <class EPI>
struct GemmArgs {
  Operand a, b[2];  // b[1]: the second projection of a gated product
  int64_t M;
  int N;            // rows of one projection
  int kb;           // bytes of k in a row (a multiple of 16)
  int nk;           // steps of one pass: ceil(kb / 128)
  int per;          // steps (over all passes) of one split
  int gm, gn, splits;
  EPI epi;
};

// ---- instruction by operand type.  KIND 0: bf16, 1: fp16, 2: int8
template <int KIND> struct Mfma;
template <> struct Mfma<0> {
  typedef f32x16 acc; typedef float el;
  static NN_D acc run(const i32x4 a, const i32x4 b, const acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mfma<1> {
  typedef f32x16 acc; typedef float el;
  static NN_D acc run(const i32x4 a, const i32x4 b, const acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mfma<2> {
  typedef i32x16 acc; typedef int el;
  static NN_D acc run(const i32x4 a, const i32x4 b, const acc c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
};

typedef __attribute__((address_space(3))) char lds_char;

// the buffer over the rows of an operand from `row` on: its range ends with the last row's last byte
NN_D __amdgpu_buffer_rsrc_t rows_buffer(const char* base, const int64_t row, const int64_t rows, const int64_t ld, const int kb) {
  const int64_t left = rows - row;
  int64_t bytes = left > 0 ? (left - 1) * ld + kb : 0;
  bytes = bytes > 0x7ffffff0 ? 0x7ffffff0 : bytes;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + (left > 0 ? row * ld : 0)), 0, (int)bytes, 0x00020000);
}

// the parts multiplied by pass t of an fp32 product, smallest terms first
NN_D int part_a(const int t) { return (0x001102 >> (4 * t)) & 3; }
NN_D int part_b(const int t) { return (0x010120 >> (4 * t)) & 3; }

// runs of 8 consecutive n of one m out of the accumulator block: quad pair P = 0, 1 (rows 16 P .. 16 P + 15 of the block); the lane's run
// starts at 16 P + 8 (lane >> 5)
template <class E, class ACC>
NN_D void take_run(const ACC& acc, const int P, E (&v)[8]) {
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, (E)acc[8 * P + x]),
                                                    __builtin_bit_cast(unsigned, (E)acc[8 * P + 4 + x]), false, false);
    v[x] = __builtin_bit_cast(E, (unsigned)s[0]);
    v[4 + x] = __builtin_bit_cast(E, (unsigned)s[1]);
  }
}

template <int KIND, int BM, int BN, int WGM, int WGN, int TERMS, bool DUAL, class EPI>
__global__ __launch_bounds__(WGM* WGN * 64, 2) void gemm_kernel(const GemmArgs<EPI> g) {
  typedef Mfma<KIND> MM;
  constexpr int NW = WGM * WGN, MI = BM / WGM / 32, NJ = BN / WGN / 32;
  constexpr int GA = BM / 8 / NW, GB = BN / 8 / NW;  // 1 KiB loads of a wave a step
  constexpr int BUF = (BM + BN) * 128;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && (!DUAL || NJ % 2 == 0), "tile");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;

  // tile of this workgroup
  const unsigned total = gridDim.x, xcd = blockIdx.x & 7u, q8 = total >> 3, r8 = total & 7u;
  unsigned id = xcd * q8 + (xcd < r8 ? xcd : r8) + (blockIdx.x >> 3);
  const unsigned tiles = (unsigned)g.gm * (unsigned)g.gn;
  const int split = (int)(id / tiles);
  id -= (unsigned)split * tiles;
  constexpr unsigned PATCH = 8;
  const unsigned band = id / (PATCH * (unsigned)g.gn), first = band * PATCH;
  const unsigned high = (unsigned)g.gm - first < PATCH ? (unsigned)g.gm - first : PATCH;
  const unsigned in = id - first * (unsigned)g.gn;
  const int tm = (int)(first + in % high), tn = (int)(in / high);
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * (DUAL ? BN / 2 : BN);

  const int lr = lane >> 3, piece = (lane & 7) ^ lr;
  unsigned off_a[GA], off_b[GB];
  __amdgpu_buffer_rsrc_t rs_a = rows_buffer(g.a.p, m0, g.M, g.a.ld, g.kb);
#pragma unroll
  for (int i = 0; i < GA; ++i) off_a[i] = (unsigned)(((i * NW + wave) * 8 + lr) * g.a.ld) + piece * 16;
  __amdgpu_buffer_rsrc_t rs_b[2];
  rs_b[0] = rows_buffer(g.b[0].p, n0, g.N, g.b[0].ld, g.kb);
  rs_b[1] = DUAL ? rows_buffer(g.b[1].p, n0, g.N, g.b[1].ld, g.kb) : rs_b[0];
#pragma unroll
  for (int i = 0; i < GB; ++i) {
    const int grp = i * NW + wave;  // DUAL: blocks of 32 rows alternate between the projections
    const int row = DUAL ? (grp >> 3) * 32 + (grp & 3) * 8 + lr : grp * 8 + lr;
    off_b[i] = (unsigned)(row * (DUAL && ((grp >> 2) & 1) ? g.b[1].ld : g.b[0].ld)) + piece * 16;
  }
  const bool up_wave = NW == 8 && ((wave >> 2) & 1);  // NW == 8: the projection of a load is the wave's, NW == 4: the load's

  const int steps = g.nk * TERMS;
  const int s0 = split * g.per, s1 = s0 + g.per < steps ? s0 + g.per : steps;

  auto issue = [&](const int s, const int buf) __attribute__((always_inline)) {
    const int kc = TERMS == 1 ? s : s / TERMS, t = TERMS == 1 ? 0 : s - kc * TERMS;
    const int k = kc * 128;
    const bool beyond = k + piece * 16 >= g.kb;
    const int pa = TERMS == 1 ? 0 : part_a(t) , pb = TERMS == 1 ? 0 : part_b(t);
    char* base = lds + buf * BUF;
#pragma unroll
    for (int i = 0; i < GA; ++i) {
      const unsigned o = beyond ? 0x80000000u : off_a[i] + k;
      const __amdgpu_buffer_rsrc_t rs = TERMS == 1 ? rs_a : rows_buffer(g.a.p + pa * g.a.plane, m0, g.M, g.a.ld, g.kb);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(base + (i * NW + wave) * 1024), 16, o, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < GB; ++i) {
      const unsigned o = beyond ? 0x80000000u : off_b[i] + k;
      const bool up = DUAL && (NW == 8 ? up_wave : ((i * NW) >> 2) & 1);
      const __amdgpu_buffer_rsrc_t rs =
          TERMS == 1 ? (up ? rs_b[1] : rs_b[0]) : rows_buffer((up ? g.b[1].p : g.b[0].p) + pb * g.b[0].plane, n0, g.N, up ? g.b[1].ld : g.b[0].ld, g.kb);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(base + BM * 128 + (i * NW + wave) * 1024), 16, o, 0, 0, 0);
    }
  };

  typename MM::acc acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  const int hi = lane >> 5, row = lane & 31;
  const int fa = (wm * MI * 32 + row) * 128, fb = BM * 128 + (wn * NJ * 32 + row) * 128;
  if (s0 < s1) issue(s0, 0);
  for (int s = s0; s < s1; ++s) {
    const int buf = (s - s0) & 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // step s has landed for every wave, and nobody reads the other buffer any more
    asm volatile("" ::: "memory");
    if (s + 1 < s1) issue(s + 1, buf ^ 1);
    const char* base = lds + buf * BUF;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const int c = ((kk * 2 + hi) ^ (row & 7)) * 16;
      i32x4 av[MI], bv[NJ];
#pragma unroll
      for (int i = 0; i < MI; ++i) av[i] = *(const i32x4*)(base + fa + i * 4096 + c);
#pragma unroll
      for (int j = 0; j < NJ; ++j) bv[j] = *(const i32x4*)(base + fb + j * 4096 + c);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = MM::run(bv[j], av[i], acc[i][j]);
    }
  }

#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = m0 + (wm * MI + i) * 32 + row;
    if (m >= g.M) continue;
    if constexpr (DUAL) {
#pragma unroll
      for (int j = 0; j < NJ; j += 2)
#pragma unroll
        for (int P = 0; P < 2; ++P) {
          typename MM::el v[8], u[8];
          take_run(acc[i][j], P, v);
          take_run(acc[i][j + 1], P, u);
          g.epi.pair(split, m, n0 + (wn * NJ + j) * 16 + 16 * P + 8 * hi, v, u);
        }
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int P = 0; P < 2; ++P) {
          typename MM::el v[8];
          take_run(acc[i][j], P, v);
          g.epi.one(split, m, n0 + (wn * NJ + j) * 32 + 16 * P + 8 * hi, v);
        }
    }
  }
}

// ---- epilogues: one(split, m, n, v): eight sums of row m from column n on; pair: of both projections.  n may lie beyond the matrix.
// All sums of a split as they are: [split][m][ld] 32-bit words (pair: the second projection at + ld / 2)
struct PartialEpi {
  uint32_t* p;
  int64_t M;
  int64_t ld;  // a multiple of 8: columns padded
  template <class E>
  NN_D void put(uint32_t* q, const E (&v)[8]) const {
    uint4 a, b;
    a.x = __builtin_bit_cast(uint32_t, v[0]), a.y = __builtin_bit_cast(uint32_t, v[1]), a.z = __builtin_bit_cast(uint32_t, v[2]), a.w = __builtin_bit_cast(uint32_t, v[3]);
    b.x = __builtin_bit_cast(uint32_t, v[4]), b.y = __builtin_bit_cast(uint32_t, v[5]), b.z = __builtin_bit_cast(uint32_t, v[6]), b.w = __builtin_bit_cast(uint32_t, v[7]);
    ((uint4*)q)[0] = a;
    ((uint4*)q)[1] = b;
  }
  template <class E>
  NN_D void one(const int split, const int64_t m, const int n, const E (&v)[8]) const {
    if (n < ld) put(p + ((int64_t)split * M + m) * ld + n, v);
  }
  template <class E>
  NN_D void pair(const int split, const int64_t m, const int n, const E (&v)[8], const E (&u)[8]) const {
    if (n >= ld / 2) return;
    uint32_t* q = p + ((int64_t)split * M + m) * ld + n;
    put(q, v);
    put(q + ld / 2, u);
  }
};

// y, or the two halves of one product's rows into two matrices (rows from `split_row` on: the second)
template <int DT>
struct StoreEpi {
  elem_t<DT>*c0, *c1;
  int64_t split_row, rows0, rows1;  // rows [0, rows0) -> c0, [split_row, split_row + rows1) -> c1
  int64_t ld;
  int N;
  NN_D void one(int, const int64_t m, const int n, const float (&v)[8]) const {
    if (n >= N) return;
    elem_t<DT>* q;
    if (m < rows0) q = c0 + m * ld;
    else if (m >= split_row && m < split_row + rows1) q = c1 + (m - split_row) * ld;
    else return;
    store8_n<DT>(q + n, N - n, v);
  }
};

// a = act(g) u into [M][F] rows of the workspace (F a multiple of 64: columns beyond the block's width are zeros, because the weights' rows
// there were read as zeros); g and u beside it where a backward pass will follow
template <int DT>
struct GatedEpi {
  elem_t<DT>*a, *gs, *us;  // gs, us NULL: inference
  int F, act;
  NN_D void pair(int, const int64_t m, const int n, const float (&v)[8], const float (&u)[8]) const {
    if (n >= F) return;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = act_only<DT != SDFNN_F32>(act, v[i]) * u[i];
    store8<DT>(a + m * F + n, o);
    if (gs) {
      store8<DT>(gs + m * F + n, v);
      store8<DT>(us + m * F + n, u);
    }
  }
};

// the gradient of a in, those of g and u out: [M][2 F], dg | du
template <int DT>
struct GatedBwdEpi {
  const elem_t<DT>*gs, *us;
  elem_t<DT>* d;
  int F, act;
  NN_D void one(int, const int64_t m, const int n, const float (&v)[8]) const {
    if (n >= F) return;
    float gv[8], uv[8], dg[8], du[8];
    load8<DT>(gs + m * F + n, gv);
    load8<DT>(us + m * F + n, uv);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float a, s;
      act_both<DT != SDFNN_F32>(act, gv[i], a, s);
      dg[i] = v[i] * uv[i] * s;
      du[i] = v[i] * a;
    }
    store8<DT>(d + m * 2 * F + n, dg);
    store8<DT>(d + m * 2 * F + F + n, du);
  }
};

template <int DT>
struct Int8Epi {
  elem_t<DT>* y;
  const float *sq, *sw, *su, *bias;
  int N, act;
  NN_D void one(int, const int64_t m, const int n, const int (&v)[8]) const {
    if (n >= N) return;
    const float s = sq[m];
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = n + i < N ? n + i : N - 1;
      o[i] = (float)v[i] * s * sw[c] + (bias ? bias[c] : 0.0f);
    }
    store8_n<DT>(y + m * N + n, N - n, o);
  }
  NN_D void pair(int, const int64_t m, const int n, const int (&v)[8], const int (&u)[8]) const {
    if (n >= N) return;
    const float s = sq[m];
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = n + i < N ? n + i : N - 1;
      o[i] = act_only<DT != SDFNN_F32>(act, (float)v[i] * s * sw[c]) * ((float)u[i] * s * su[c]);
    }
    store8_n<DT>(y + m * N + n, N - n, o);
  }
};

// the sums of the splits, added in their order, through the epilogue.  One thread 8 columns.
template <class E, bool DUAL, class EPI>
__global__ __launch_bounds__(256) void split_reduce_kernel(const E* __restrict__ p, const int splits, const int64_t M, const int64_t ld,
                                                           const EPI epi) {
  const int64_t groups = (DUAL ? ld / 2 : ld) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= groups * M) return;
  const int64_t m = i / groups;
  const int n = (int)(i - m * groups) * 8;
  E v[8], u[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0, u[e] = 0;
  for (int s = 0; s < splits; ++s) {
    const E* q = p + ((int64_t)s * M + m) * ld + n;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += q[e];
    if constexpr (DUAL) {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] += q[ld / 2 + e];
    }
  }
  if constexpr (DUAL) epi.pair(0, m, n, v, u);
  else epi.one(0, m, n, v);
}
