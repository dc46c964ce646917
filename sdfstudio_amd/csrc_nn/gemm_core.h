// sdfnn — matrix products C[m, n] = sum_k A[m, k] B[n, k] on the matrix cores.
//
// One scheme serves 16-bit floats (v_mfma_f32_32x32x16), 8-bit integers (v_mfma_i32_32x32x32) and fp32 as three bf16 parts a value: to it a
// step is 128 bytes of k (64 16-bit or 128 8-bit elements), and an operand fragment is 16 bytes a lane whatever they hold.
//   * Tiles go from HBM / L2 to LDS without passing registers (buffer_load_dwordx4 ... lds).  A row past the end of a matrix, and the bytes past
//     k in the last step, lie outside the buffer's range, where the load returns zeros: ragged sizes cost no branch in the loop.
//   * A 16-bit operand may also lie with its k running DOWN the rows (x and dy in a weight's gradient, a weight in dx): its 64 rows of a step go
//     to LDS as they are and ds_read_b64_tr_b16 turns 4 x 16 pieces of them into fragments, so that no transposed copy is ever made.
//   * A fragment read takes one piece of many LDS rows: stored in order they would lie in the same few banks.  The pieces of a row are permuted
//     instead (the permutation is applied to the GLOBAL address of the load, LDS itself is written in order).
//   * The weights' rows (n) are operand A of the instruction and the tokens' rows (m) operand B: a lane then owns ONE m and runs of 4
//     consecutive n, which the epilogue stages through LDS in 16-byte pieces.
//   * fp32: x = p0 + p1 + p2 with p0 = bf16(x), p1 = bf16(x - p0), p2 = bf16(x - p0 - p1) holds all 24 bits; of the nine products of two
//     such sums the six largest are formed (the rest is below 2^-24 of |a b|): six steps for each 64 of k, the small ones first,
//     which differ in the pair of parts they read and add to one fp32 sum, as the steps of a 16-bit product do.
//   * Workgroups are numbered so that the ones that run at the same time on one XCD (ids equal mod 8) form a square-ish patch of tiles and
//     share their operands in that XCD's L2.
//   * Few tiles: k is split over workgroups; raw sums go to the workspace and a second kernel adds them in order and applies the epilogue.
#pragma once
#include "nn_common.h"

struct Operand {
  const char* p;
  int64_t ld;     // bytes between rows
  int64_t plane;  // bytes between the parts of an fp32 matrix
  int64_t rows;   // k along the row: rows of the matrix; k down the rows: k
  int64_t width;  // bytes of a row
};

template <class EPI>
struct GemmArgs {
  Operand a, b[2];  // b[1]: the second projection of a gated product, or what follows b[0] along k from step `turn` on
  int64_t M;
  int N;            // rows of one projection
  int nk;           // steps of k (fp32: each taken six times)
  int turn;
  int per;          // steps of one split (fp32: six for each of k)
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

// the buffer (descriptor words) over the rows of an operand (part `part`) from `row` on: its range ends with the last row's last byte
NN_D i32x4 rows_buffer(const char* p, const int64_t ld, const int64_t rows, const int64_t width, const int64_t row) {
  const int64_t left = rows - row;
  const uint64_t at = (uint64_t)p + (uint64_t)(row * ld);
  int64_t bytes = (left - 1) * ld + width;
  bytes = bytes > 0x7ffffff0 ? 0x7ffffff0 : bytes;
  bytes = left > 0 ? bytes : 0;
  return i32x4{(int)(uint32_t)at, (int)(uint32_t)(at >> 32), (int)bytes, 0x00020000};
}

// 1 KiB, 16 bytes a lane, from the buffer to LDS (byte address `to`, the wavefront's).  Written as an instruction because the compiler, which
// cannot tell the units of the ring apart, waits for every load it knows to write LDS before it reads any of LDS with
// ds_read_b64_tr_b16.  It returns no register, and the loops wait for it by count.  m0 is written here and nowhere else in these kernels.
NN_D void load_lds(const i32x4 buffer, const unsigned offset, const unsigned to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(buffer), "s"(to) : "memory");
}

// the parts multiplied by term t of an fp32 product, smallest terms first
NN_D int part_a(const int t) { return (0x001102 >> (4 * t)) & 3; }
NN_D int part_b(const int t) { return (0x010120 >> (4 * t)) & 3; }

// tile and split of this workgroup
struct TileId {
  int64_t m0;
  int n0, split;
};
template <int BM, int BN, class EPI>
NN_D TileId tile_of(const GemmArgs<EPI>& g) {
  const unsigned total = gridDim.x, xcd = blockIdx.x & 7u, q8 = total >> 3, r8 = total & 7u;
  unsigned id = xcd * q8 + (xcd < r8 ? xcd : r8) + (blockIdx.x >> 3);
  const unsigned tiles = (unsigned)g.gm * (unsigned)g.gn;
  const unsigned split = id / tiles;
  id -= split * tiles;
  constexpr unsigned PATCH = 8;
  const unsigned band = id / (PATCH * (unsigned)g.gn), first = band * PATCH;
  const unsigned high = (unsigned)g.gm - first < PATCH ? (unsigned)g.gm - first : PATCH;
  const unsigned in = id - first * (unsigned)g.gn;
  return {(int64_t)(first + in % high) * BM, (int)(in / high) * BN, (int)split};
}

// The accumulators of a wavefront (rows from m, columns from n on; DUAL: blocks of 32 columns alternate between the projections) through the
// epilogue.  An accumulator block holds one m and scattered n a lane; 32 rows at a time go through the wavefront's own piece of LDS (free
// after the last step; rows 16 bytes longer than their data, so that writes and reads cover all banks) and come back as 8 consecutive n a
// lane, with the lanes side by side along the row: whole lines of every tensor the epilogue reads or writes.  What it reads of other
// tensors (epi.fetch) is requested for several passes before the first is used; what belongs to columns (epi.cols) is read once.
template <int NJ> struct Stage { static constexpr int stride = NJ * 128 + 16, bytes = 32 * stride; };
template <bool DUAL, int NJ, class EPI>
NN_D auto put_cols(const EPI& epi, const int n, const int lane) { return epi.cols(n + (lane % (DUAL ? NJ * 2 : NJ * 4)) * 8); }
template <bool DUAL, class E, int MI, int NJ, class ACC, class EPI, class COLS>
NN_D void put_tile(const ACC (&acc)[MI][NJ], const EPI& epi, const COLS& cols, const int split, const int64_t M, const int64_t m, const int n, const int lane,
                   char* stage) {
  constexpr int W = DUAL ? NJ * 16 : NJ * 32, LPR = W / 8, RPP = 64 / LPR, PASSES = 32 / RPP, STRIDE = Stage<NJ>::stride;
  const int hi = lane >> 5, row = lane & 31;
  const int c = (lane % LPR) * 8, r0 = lane / LPR;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    typename EPI::Row rows[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) rows[p] = epi.fetch(m + i * 32 + p * RPP + r0, M, n + c);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      char* q = stage + row * STRIDE + (DUAL ? (j & 1) * (W * 4) + (j >> 1) * 128 : j * 128) + hi * 16;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        i32x4 v;
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = __builtin_bit_cast(int, (E)acc[i][j][4 * k + x]);
        *(i32x4*)(q + k * 32) = v;
      }
    }
    asm volatile("" ::: "memory");  // one wavefront's LDS accesses happen in program order; the compiler must keep it
#pragma unroll EPI::kUnroll
    for (int p = 0; p < PASSES; ++p) {
      const char* q = stage + (p * RPP + r0) * STRIDE + c * 4;
      E v[8], u[8];
      __builtin_memcpy(v, q, 32);
      if constexpr (DUAL) __builtin_memcpy(u, q + W * 4, 32);
      const int64_t mi = m + i * 32 + p * RPP + r0;
      if (mi < M) {
        if constexpr (DUAL) epi.pair(split, mi, n + c, v, u, cols, rows[p]);
        else epi.one(split, mi, n + c, v, cols, rows[p]);
      }
    }
    asm volatile("" ::: "memory");
  }
}

// ---- one operand's unit of a step in LDS: ROWS matrix rows x 128 bytes of k, moved by loads of 1 KiB, four wavefronts taking turns.
// k along the row: LDS rows are matrix rows, piece c (16 bytes) of row r lies at c ^ ((r >> 1) & 7).
// k down the rows (KM): LDS rows are the 64 k of a step, ROWS 16-bit elements each; piece c (32 bytes = 16 elements) of row r lies at
// c ^ (2 (r & 3) + ((r >> 3) & 1)).  Either way the accesses of one pass over the banks lie in different places.
template <int ROWS, bool KM>
struct Side {
  static constexpr int LOADS = ROWS / 32, RB = KM ? ROWS * 2 : 128;
  // what load i of wavefront `wave` fetches: byte offset of the lane from the unit's first row
  static NN_D unsigned offset(const int i, const int wave, const int lane, const int64_t ld) {
    if constexpr (!KM) {
      const int grp = i * 4 + wave, lr = lane >> 3;
      return (unsigned)((grp * 8 + lr) * ld) + ((lane & 7) ^ ((grp & 1) * 4 + (lr >> 1))) * 16;
    } else {
      constexpr int RPL = 1024 / RB, LPR = 64 / RPL;
      const int r = (i * 4 + wave) * RPL + lane / LPR, c = lane % LPR;
      return (unsigned)(r * ld) + (((c >> 1) ^ ((r & 3) * 2 + ((r >> 3) & 1))) * 2 + (c & 1)) * 16;
    }
  }
  // the lane's address of quarter 0 of block 0 of the wavefront's rows (from `first` on)
  static NN_D int base(const int first, const int lane) {
    if constexpr (!KM) return (first + (lane & 31)) * 128 + (((lane >> 5) ^ ((lane >> 1) & 7)) * 16);
    const int r = (lane >> 5) * 8 + ((lane >> 2) & 3), f = (r & 3) * 2 + (lane >> 5);
    return r * RB + (((first >> 4) + ((lane >> 4) & 1)) ^ f) * 32 + (lane & 3) * 8;
  }
  // the fragment of block i (32 rows), quarter q (32 bytes of k, resp. 16 k)
  static NN_D i32x4 fragment(const char* lds, const int unit, const int base, const int i, const int q) {
    if constexpr (!KM) return *(const i32x4*)(lds + unit + (base ^ (q * 32)) + i * 4096);
    else {
      typedef __attribute__((address_space(3))) s16x4* P;
      const char* p = lds + unit + (base ^ (i * 64)) + q * 16 * RB;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + 4 * RB));
      return __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// loads of one operand.  TURN: it may go over to a second matrix along k
template <int ROWS, bool KM, int TERMS, bool SECOND, bool TURN>
struct Loader {
  unsigned off[Side<ROWS, KM>::LOADS];
  int piece;  // bytes of k in front of the lane's piece (k along the row)
  template <class F>
  NN_D void init(const int wave, const int lane, const int64_t first, F&& ld_of) {  // first: matrix row (KM: column) of the tile
#pragma unroll
    for (int i = 0; i < Side<ROWS, KM>::LOADS; ++i)
      off[i] = Side<ROWS, KM>::offset(i, wave, lane, ld_of(i)) + (KM ? (unsigned)first * 2 : 0);
    piece = ((lane & 7) ^ ((wave & 1) * 4 + (lane >> 4))) * 16;
  }
  // the buffer of step s
  NN_D i32x4 buffer(const Operand& one, const Operand& two, const int turn, const int64_t row, const int s) const {
    const int kc = TERMS == 1 ? s : s / TERMS, t = s - kc * TERMS;
    const int part = TERMS == 1 ? 0 : SECOND ? part_b(t) : part_a(t);
    if constexpr (!KM) return rows_buffer(one.p + part * one.plane, one.ld, one.rows, one.width, row);
    const bool after = TURN && kc >= turn;
    const int64_t at = (int64_t)(after ? kc - turn : kc) * 64;
    return rows_buffer((after ? two.p : one.p) + part * (after ? two.plane : one.plane), one.ld, one.rows, one.width, at);
  }
  // load i of step s; beyond: out of range (buffers end below 2^31), where it writes zeros
  NN_D void issue(const i32x4 buf, const int64_t width, const int s, const bool beyond, const int i, const unsigned to) const {
    const int kc = TERMS == 1 ? s : s / TERMS;
    unsigned o = (KM ? off[i] : off[i] + kc * 128) | (unsigned)beyond << 31;
    if constexpr (!KM) o |= (unsigned)(kc * 128 + piece >= (int)width) << 31;  // past k
    load_lds(buf, o, to);
  }
};

// ---- the product: T x T tiles of four wavefronts, each a quarter of the tile.
//   T = 256  one workgroup a CU (one wavefront a SIMD): a fragment is used for four instructions, so the operand reads take half of LDS's
//            bandwidth; the 256 accumulators leave registers for a second set of fragments.
//   T = 128  two workgroups a CU: more operand traffic, but one's epilogue runs under the other's instructions, and small products
//            have four times the tiles.
// The reads of one quarter step run under the instructions of another.  A step is 128 bytes of k - whole lines, the request that L2 serves at
// full rate - and one operand's T rows of it are the unit of a ring of five in LDS: A0 B0 A1 B1 A2.  Both units of a step are free once the
// last wavefront has taken its fourth quarter into registers; B of the step after next goes into the first of them at once and A of the
// one behind it into the second.  Loads are spread between the instructions, since a load that finds the address unit busy holds back what
// follows it.
constexpr int kRing = 5;
template <int T> struct Unit { static constexpr int bytes = T * 128, ring = kRing * bytes; };
template <int T, int KIND, int TERMS, bool DUAL, bool AK, bool BK, class EPI>
__global__ __launch_bounds__(256, T == 256 ? 1 : 2) void gemm_kernel(const GemmArgs<EPI> g) {
  static_assert(!DUAL || (!AK && !BK), "gated products read k along the rows");
  typedef Mfma<KIND> MM;
  typedef Side<T, AK> SA;
  typedef Side<T, BK> SB;
  constexpr int MI = T / 64, LOADS = T / 32, UNIT = Unit<T>::bytes;  // blocks of a wavefront each way; its loads a unit
  // The last two steps, which load nothing, have code of their own at T = 128, where products of a few steps are at home; at T = 256 a second
  // copy of the loop costs registers, and their loads are out of range instead.
  constexpr bool PEEL = T == 128;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const TileId id = tile_of<T, DUAL ? T / 2 : T>(g);

  Loader<T, AK, TERMS, false, false> la;
  Loader<T, BK, TERMS, true, !AK> lb;
  la.init(wave, lane, id.m0, [&](int) { return g.a.ld; });
  lb.init(wave, lane, id.n0, [&](int i) { return g.b[DUAL ? i & 1 : 0].ld; });
  if constexpr (DUAL) {  // load i brings rows of projection i & 1 (blocks of 32 rows alternate)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) lb.off[i] = (unsigned)(((i >> 1) * 32 + wave * 8 + (lane >> 3)) * g.b[i & 1].ld) + lb.piece;
  }
  const int steps = g.nk * TERMS;
  const int s0 = id.split * g.per, s1 = s0 + g.per < steps ? s0 + g.per : steps;
  const unsigned ring = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds + wave * 1024;
  const std::integral_constant<bool, false> A{};
  const std::integral_constant<bool, true> B{};
  i32x4 buf_a, buf_b[2];  // buffers of the step being loaded
  auto aim = [&](const int s) __attribute__((always_inline)) {
    buf_a = la.buffer(g.a, g.a, 0, id.m0, s);
    buf_b[0] = lb.buffer(g.b[0], g.b[1], g.turn, id.n0, s);
    if constexpr (DUAL) buf_b[1] = lb.buffer(g.b[1], g.b[1], g.turn, id.n0, s);
  };
  auto issue = [&](const int s, auto second, const int i, const int unit) __attribute__((always_inline)) {
    const unsigned to = ring + unit + i * 4096;
    if constexpr (decltype(second)::value) lb.issue(buf_b[DUAL ? i & 1 : 0], g.b[0].width, s, !PEEL && s >= s1, i, to);
    else la.issue(buf_a, g.a.width, s, !PEEL && s >= s1, i, to);
  };

  typename MM::acc acc[MI][MI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < MI; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  const int fa = SA::base(wm * (T / 2), lane), fb = SB::base(wn * (T / 2), lane);
  i32x4 a0[MI], b0[MI], a1[MI], b1[MI];
  // a quarter step: the instructions of the fragments (a, b); between them the reads of quarter nq of the units ua, ub (na, nb) and NL loads
  auto quarter = [&](const i32x4 (&a)[MI], const i32x4 (&b)[MI], const int nq, const int ua, const int ub, i32x4 (&na)[MI], i32x4 (&nb)[MI],
                     auto nl, auto operand, const int ls, const int lf, const int unit) __attribute__((always_inline)) {
    constexpr int NL = decltype(nl)::value;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int j = 0; j < MI / 2; ++j) acc[i][j] = MM::run(b[j], a[i], acc[i][j]);
      if (i < MI / 2) {
        nb[2 * i] = SB::fragment(lds, ub, fb, 2 * i, nq);
        nb[2 * i + 1] = SB::fragment(lds, ub, fb, 2 * i + 1, nq);
        na[i] = SA::fragment(lds, ua, fa, i, nq);
      }
      if (i == MI / 2) {
#pragma unroll
        for (int x = MI / 2; x < MI; ++x) na[x] = SA::fragment(lds, ua, fa, x, nq);
      }
      if constexpr (NL > 0 && NL == LOADS) issue(ls, operand, lf + 2 * i, unit);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = MI / 2; j < MI; ++j) acc[i][j] = MM::run(b[j], a[i], acc[i][j]);
      if constexpr (NL == LOADS) issue(ls, operand, lf + 2 * i + 1, unit);
      if constexpr (NL == LOADS / 2) issue(ls, operand, lf + i, unit);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const std::integral_constant<int, 0> none{};
  auto behind = [](const int unit, const int n) { return unit + n * UNIT >= kRing * UNIT ? unit + (n - kRing) * UNIT : unit + n * UNIT; };

  const int lane_n = id.n0 + wn * (DUAL ? T / 4 : T / 2);
  const auto cols = put_cols<DUAL, MI>(g.epi, lane_n, lane);  // on its way while the product is computed
  if (s0 < s1) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (PEEL && x == 1 && s0 + 1 >= s1) break;
      aim(s0 + x);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) issue(s0 + x, A, i, 2 * x * UNIT);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) issue(s0 + x, B, i, (2 * x + 1) * UNIT);
    }
    if (!PEEL || s0 + 1 < s1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");  // step s0 has landed
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < MI; ++i) a0[i] = SA::fragment(lds, 0, fa, i, 0), b0[i] = SB::fragment(lds, UNIT, fb, i, 0);
    int ua = 0;
    auto step = [&](const int s, auto more) __attribute__((always_inline)) {  // more: step s + 2 exists
      constexpr bool MORE = decltype(more)::value;
      const std::integral_constant<int, MORE ? LOADS / 2 : 0> some{};
      const std::integral_constant<int, MORE ? LOADS : 0> all{};
      const int ub = behind(ua, 1), na = behind(ua, 2), nb = behind(ua, 3), next = behind(ua, 4);
      if constexpr (MORE) aim(s + 2);
      quarter(a0, b0, 1, ua, ub, a1, b1, some, A, s + 2, 0, next);
      quarter(a1, b1, 2, ua, ub, a0, b0, some, A, s + 2, LOADS / 2, next);
      quarter(a0, b0, 3, ua, ub, a1, b1, none, A, 0, 0, 0);
      // own loads of step s + 1 have landed (those of A of s + 2 may be under way), own reads of step s are done: after the barrier both hold
      // for every wavefront
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(MORE ? LOADS : 0) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      quarter(a1, b1, 0, na, nb, a0, b0, all, B, s + 2, 0, ua);  // (the fragments behind the last step are read and not used)
      ua = na;
    };
    int s = s0;
    for (; s + (PEEL ? 2 : 0) < s1; ++s) step(s, std::true_type{});
    if constexpr (PEEL) {
      for (; s < s1; ++s) step(s, std::false_type{});
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may still be on its way into LDS
    }
    __syncthreads();
  }
  static_assert(4 * Stage<MI>::bytes <= Unit<T>::ring, "the epilogue's pieces lie in the ring");
  put_tile<DUAL, typename MM::el>(acc, g.epi, cols, id.split, g.M, id.m0 + wm * (T / 2), lane_n, lane, lds + wave * Stage<MI>::bytes);
}

// ---- epilogues: one(split, m, n, v, cols, row): eight sums of row m from column n on; pair: of both projections.  n may lie beyond the
// matrix (in cols and fetch too), m only in fetch.
// kUnroll: passes of put_tile side by side (few where their code is long).  kCost: ps a column of a 256 x 256 tile's row spends in the epilogue
// with all CUs at it (bytes at ~16 GB/s a CU and ns, or instructions), for the choice of tiles.
struct Nothing {};
// All sums of a split as they are: [split][m][ld] 32-bit words (pair: the second projection at + ld / 2)
struct PartialEpi {
  static constexpr int kCost = 250;
  static constexpr int kUnroll = 8;
  typedef Nothing Row;
  uint32_t* p;
  int64_t M;
  int64_t ld;  // a multiple of 8: columns padded
  NN_D Nothing cols(int) const { return {}; }
  NN_D Nothing fetch(int64_t, int64_t, int) const { return {}; }
  template <class E>
  NN_D void put(uint32_t* q, const E (&v)[8]) const {
    uint4 a, b;
    a.x = __builtin_bit_cast(uint32_t, v[0]), a.y = __builtin_bit_cast(uint32_t, v[1]), a.z = __builtin_bit_cast(uint32_t, v[2]), a.w = __builtin_bit_cast(uint32_t, v[3]);
    b.x = __builtin_bit_cast(uint32_t, v[4]), b.y = __builtin_bit_cast(uint32_t, v[5]), b.z = __builtin_bit_cast(uint32_t, v[6]), b.w = __builtin_bit_cast(uint32_t, v[7]);
    ((uint4*)q)[0] = a;
    ((uint4*)q)[1] = b;
  }
  template <class E>
  NN_D void one(const int split, const int64_t m, const int n, const E (&v)[8], Nothing, Nothing) const {
    if (n < ld) put(p + ((int64_t)split * M + m) * ld + n, v);
  }
  template <class E>
  NN_D void pair(const int split, const int64_t m, const int n, const E (&v)[8], const E (&u)[8], Nothing, Nothing) const {
    if (n >= ld / 2) return;
    uint32_t* q = p + ((int64_t)split * M + m) * ld + n;
    put(q, v);
    put(q + ld / 2, u);
  }
};

// y, or the two halves of one product's rows into two matrices (rows from `split_row` on: the second)
template <int DT>
struct StoreEpi {
  static constexpr int kCost = DT == SDFNN_F32 ? 250 : 120;
  static constexpr int kUnroll = 8;
  typedef Nothing Row;
  elem_t<DT>*c0, *c1;
  int64_t split_row, rows0, rows1;  // rows [0, rows0) -> c0, [split_row, split_row + rows1) -> c1
  int64_t ld;
  int N;
  NN_D Nothing cols(int) const { return {}; }
  NN_D Nothing fetch(int64_t, int64_t, int) const { return {}; }
  NN_D elem_t<DT>* row(const int64_t m) const {
    return m < rows0 ? c0 + m * ld : m >= split_row && m < split_row + rows1 ? c1 + (m - split_row) * ld : nullptr;
  }
  NN_D void one(int, const int64_t m, const int n, const float (&v)[8], Nothing, Nothing) const {
    elem_t<DT>* q = row(m);
    if (q && n < N) store8_n<DT>(q + n, N - n, v);
  }
  NN_D void four(const int64_t m, const int64_t n, const float (&v)[4]) const {
    elem_t<DT>* q = row(m);
    if (!q || n >= N) return;
    if (n + 4 <= N) {
      Bytes<4, 4> raw;
      __builtin_memcpy(&raw, v, 16);
      *reinterpret_cast<Bytes<4, 4>*>(q + n) = raw;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < N) q[n + e] = v[e];
    }
  }
};

// a = act(g) u into [M][F] rows of the workspace (F a multiple of 64: columns beyond the block's width are zeros, because the weights' rows
// there were read as zeros).  Where a backward pass will follow, the two factors it needs beside it: act(g) and u act'(g), formed from the
// sums as they are and kept in fp32 - rounded to 16 bits, g and u alone cost the gradients as much as all their other roundings together
// (error against 64 bits at 8192 x 4096 x 16384 bf16: 0.0031 of the gradients' size, 0.0024 this way, 0.0017 their own last rounding).
// a itself is one number of the type where tiles read it, and so are the gradients of g and u below: each as two numbers would be a third more matrix
// instructions forward and five sixths more backward.  TWO (few rows of 16 bits): two numbers, the rounding of a and what it leaves, which hold a to
// 2^-16 (bf16) and 2^-22.
template <int DT, bool TWO = false>
struct GatedEpi {
  static constexpr int kCost = DT == SDFNN_F32 ? 370 : 300;
  static constexpr int kUnroll = 1;
  typedef Nothing Row;
  elem_t<DT>* a;
  int64_t plane;   // fp32: 0: a as it is; else its three bf16 parts, as the second product reads them, this many bytes apart
  float *fu, *fg;  // factors of du and dg; NULL: inference
  int F, act;
  elem_t<DT>* two = nullptr;  // TWO: [2 M][F], the second numbers `rest` elements behind the first; a: NULL unless a backward pass will follow
  int64_t rest = 0;
  NN_D Nothing cols(int) const { return {}; }
  NN_D Nothing fetch(int64_t, int64_t, int) const { return {}; }
  NN_D void pair(int, const int64_t m, const int n, const float (&v)[8], const float (&u)[8], Nothing, Nothing) const {
    if (n >= F) return;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = v[i];
    if (fu) {
      float q[8];
      act8<DT != SDFNN_F32>(act, o, q);
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] *= u[i];
      store8<SDFNN_F32>(fu + m * F + n, o);
      store8<SDFNN_F32>(fg + m * F + n, q);
    } else {
      act8<DT != SDFNN_F32>(act, o);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= u[i];
    if constexpr (TWO) {
      float p[8], q[8];
      constexpr float top = DT == SDFNN_F16 ? 65504.0f : 0x1.fep127f;  // the first is held there, so that only what is infinite becomes so
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = (float)(elem_t<DT>)__builtin_amdgcn_fmed3f(o[i], -top, top);
        q[i] = o[i] - p[i];
      }
      store8<DT>(two + m * F + n, p);
      store8<DT>(two + rest + m * F + n, q);
      if (!a) return;
    }
    if (DT == SDFNN_F32 && plane) store_parts((char*)a + (m * F + n) * 2, plane, o);
    else store8<DT>(a + m * F + n, o);
  }
};

// the gradient of a in, those of g and u out: [M][2 F], dg | du (fp32 with a plane: as three bf16 parts)
template <int DT>
struct GatedBwdEpi {
  static constexpr int kCost = DT == SDFNN_F32 ? 1250 : 750;
  static constexpr int kUnroll = 8;
  struct Row { float p[8], q[8]; };
  const float *fu, *fg;
  char* d;
  int64_t plane;
  int F;
  NN_D Nothing cols(int) const { return {}; }
  NN_D Row fetch(const int64_t m, const int64_t M, const int n) const {
    Row r{};
    if (m < M && n < F) {
      load8<SDFNN_F32>(fu + m * F + n, r.p);
      load8<SDFNN_F32>(fg + m * F + n, r.q);
    }
    return r;
  }
  NN_D void one(int, const int64_t m, const int n, const float (&v)[8], Nothing, const Row& r) const {
    if (n >= F) return;
    float p[8], q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = r.p[i] * v[i], q[i] = r.q[i] * v[i];
    const int64_t at = m * 2 * F + n;
    if (DT == SDFNN_F32 && plane) {
      store_parts(d + at * 2, plane, q);
      store_parts(d + (at + F) * 2, plane, p);
    } else {
      store8<DT>((elem_t<DT>*)d + at, q);
      store8<DT>((elem_t<DT>*)d + at + F, p);
    }
  }
};

template <int DT>
struct Int8Epi {
  static constexpr int kCost = 190;  // (one for all result types: the workspace query does not know it)
  static constexpr int kUnroll = 8;
  struct Cols { float s[8], t[8]; };  // scales of the columns; t: of the second projection, or the bias
  typedef float Row;
  elem_t<DT>* y;
  const float *sq, *sw, *su, *bias;
  int N, act;
  NN_D Cols cols(const int n) const {
    Cols c;
    const int left = N - n < 0 ? 0 : N - n;
    const float* t = su ? su : bias;
    load8_n<SDFNN_F32>(sw + n, left, c.s);
    if (t) load8_n<SDFNN_F32>(t + n, left, c.t);
    else {
#pragma unroll
      for (int i = 0; i < 8; ++i) c.t[i] = 0.0f;
    }
    return c;
  }
  NN_D float fetch(const int64_t m, const int64_t M, int) const { return sq[m < M ? m : M - 1]; }
  NN_D void one(int, const int64_t m, const int n, const int (&v)[8], const Cols& c, const float s) const {
    if (n >= N) return;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)v[i] * s * c.s[i] + c.t[i];
    store8_n<DT>(y + m * N + n, N - n, o);
  }
  NN_D void pair(int, const int64_t m, const int n, const int (&v)[8], const int (&u)[8], const Cols& c, const float s) const {
    if (n >= N) return;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)v[i] * s * c.s[i];
    act8<DT != SDFNN_F32>(act, o);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= (float)u[i] * s * c.t[i];
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
  if constexpr (DUAL) epi.pair(0, m, n, v, u, epi.cols(n), epi.fetch(m, M, n));
  else epi.one(0, m, n, v, epi.cols(n), epi.fetch(m, M, n));
}
