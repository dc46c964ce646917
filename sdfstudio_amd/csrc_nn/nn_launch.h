// sdfnn — host side of the products: tile choice, workspace layout, launches.
#pragma once
#include <algorithm>

#include "gemm_core.h"
#include "pack_kernels.h"
#include "skinny_kernels.h"

// A call's workspace, carved in the order of use.  With base == nullptr nothing is launched: the same code computes what the call needs.
struct Call {
  char* base;
  int64_t used;
  hipStream_t stream;
  int tile[4], splits[4], products;  // of its products in their order (tile 0: a kernel of few rows), for the queries
  void note(const int t, const int s) { tile[products & 3] = t, splits[products++ & 3] = s; }
  bool dry() const { return base == nullptr; }
  char* take(const int64_t bytes) {
    char* p = base + used;  // dry: never dereferenced
    used += round_up(bytes, 256);
    return p;
  }
};

// A launch larger than 64 KiB of LDS has to ask for it; the attribute is per function and per device and costs a host call of ~1 us.
template <class K>
inline void ask_lds(K kernel, const int bytes) {
  if (bytes > 64 * 1024) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

struct Tiling {
  int tile;  // 256 or 128
  int gm, gn, splits, per;
};
// Which of the two tile sizes (gemm_core.h), and how often k is split: the smallest estimate of
//   256: rounds of workgroups x (steps x 1.3 us + 5 us + the epilogue)
//   128: rounds of pairs    x (max(steps x 1.15 us, two epilogues) + 3 us): one's epilogue runs under the other's steps
// and, where k is split, the join of the raw sums.  Both sides measured (us, 256 / 128): 8192 x 4096 x 16384 bf16, plain store 800 / 1105;
// 524288 x 512 x 256 fp32 with the gated backward's epilogue 1420 / 1420 (bound by HBM), 524288 x 1024 x 256 with the forward's 1950 / 2120; the same
// int8 600 / 460.
inline Tiling choose_tiling(const int64_t M, const int64_t N, const int nk, const int terms, const int cost) {
  Tiling best = {};
  double best_us = 1e30;
  const int steps = nk * terms;
  for (int tile : {256, 128}) {
    const int64_t gm = ceil_div(M, tile), gn = ceil_div(N, tile), tiles = gm * gn;
    if (tile == 128 && tiles >= (int64_t)1 << 24) break;  // a launch has less than 2^32 threads (256 x 256 tiles that would not fit exceed the memory)
    const int64_t slots = tile == 256 ? 256 : 512;
    const int most = (int)std::max<int64_t>(1, std::min<int64_t>(steps / 4, 2 * slots / std::max<int64_t>(tiles, 1)));
    for (int s = 1; s <= most; s = s < 4 ? s + 1 : s + s / 4) {
      const int per = (int)ceil_div(std::max(steps, 1), s);
      const double epilogue = 65536e-6 * (s == 1 ? cost : PartialEpi::kCost);
      const double one = tile == 256 ? per * 1.3 + 5.0 + epilogue : std::max(per * 1.15, epilogue / 2) + 3.0;
      const double join = s == 1 ? 0.0 : 6.0 + (double)(s + 1) * (double)M * (double)N * 4.0 / 3e6;
      const double us = (double)ceil_div(tiles * s, slots) * one + join;
      if (us < best_us) best_us = us, best = {tile, (int)gm, (int)gn, (int)ceil_div(std::max(steps, 1), per), per};
    }
  }
  return best;
}

// k along the rows of an operand, or down them (KM)
enum Sides { kRows, kRowsDown, kDown };  // A B: row row, row down, down down

template <int KIND, int TERMS, bool DUAL, int SIDES, class EPI>
int launch_gemm(Call& c, const Tiling& t, GemmArgs<EPI> g) {
  constexpr bool AK = SIDES == kDown, BK = SIDES != kRows;
  g.gm = t.gm, g.gn = t.gn, g.splits = t.splits, g.per = t.per;
  const unsigned grid = (unsigned)((int64_t)t.gm * t.gn * t.splits);
  if (grid == 0) return 0;
  auto start = [&](auto tile) {
    constexpr int T = decltype(tile)::value;
    auto* k = gemm_kernel<T, KIND, TERMS, DUAL, AK, BK, EPI>;
    ask_lds(k, Unit<T>::ring);
    hipLaunchKernelGGL(k, dim3(grid), dim3(256), Unit<T>::ring, c.stream, g);
  };
  if (t.tile == 256) start(std::integral_constant<int, 256>{});
  else start(std::integral_constant<int, 128>{});
  NN_LAUNCHED("product");
  return 0;
}

// One product through `epi`; k split where the tiles are few.  DUAL: two under a gate.  Otherwise b1 follows b0 along k from step `turn` on.
// nk: steps of 128 bytes of k
template <int KIND, int TERMS, bool DUAL, int SIDES, class EPI>
int product(Call& c, const Operand& a, const Operand& b0, const Operand& b1, const int64_t M, const int64_t N, const int64_t nk, const int64_t turn,
            const EPI& epi) {
  const Tiling t = choose_tiling(M, DUAL ? 2 * N : N, (int)nk, TERMS, EPI::kCost);
  c.note(t.tile, t.splits);
  const int64_t ld = (DUAL ? 2 : 1) * round_up(N, 64);
  char* part = t.splits > 1 ? c.take((int64_t)t.splits * M * ld * 4) : nullptr;
  if (c.dry() || M == 0 || N == 0) return 0;
  NN_REQUIRE((int64_t)t.gm * t.gn * t.splits < (int64_t)1 << 24 && nk * TERMS < 0x7fffffff, "too many tiles");
  if (t.splits == 1) {
    GemmArgs<EPI> g{a, {b0, b1}, M, (int)N, (int)nk, (int)turn, 0, 0, 0, 0, epi};
    return launch_gemm<KIND, TERMS, DUAL, SIDES>(c, t, g);
  }
  PartialEpi pe{(uint32_t*)part, M, ld};
  GemmArgs<PartialEpi> g{a, {b0, b1}, M, (int)N, (int)nk, (int)turn, 0, 0, 0, 0, pe};
  if (const int rc = launch_gemm<KIND, TERMS, DUAL, SIDES>(c, t, g)) return rc;
  const int64_t groups = round_up(N, 64) / 8 * M;
  hipLaunchKernelGGL((split_reduce_kernel<typename Mfma<KIND>::el, DUAL, EPI>), dim3((unsigned)ceil_div(groups, 256)), dim3(256), 0, c.stream,
                     (const typename Mfma<KIND>::el*)part, t.splits, M, ld, epi);
  NN_LAUNCHED("split sum");
  return 0;
}

// Rows up to which a product streams its weights (skinny_kernels.h).  fp32, whose tiles first have to split the weights into parts, stays with it
// longer: 64 x 4096 -> 2 x 16384 -> 4096 takes 714 us on tiles and 391 here, its backward pass 1076 and 710 (16 rows: 1045 and 435).
constexpr int64_t few_rows(const int kind) { return kind == 3 ? 64 : 32; }

// the same for at most few_rows(KIND) rows.  cols: columns that the epilogue writes (>= N).  PAIR: M rows of a, each result the sum of two
template <int KIND, bool DUAL, bool PAIR = false, class EPI>
int skinny(Call& c, const Operand& a, const Operand& b0, const Operand& b1, const int64_t M, const int64_t N, const int64_t cols, const EPI& epi) {
  c.note(0, 1);
  if (c.dry() || M == 0 || N == 0) return 0;
  GemmArgs<EPI> g{a, {b0, b1}, M, (int)N, 0, 0, 0, 0, 0, 0, epi};
  const dim3 grid((unsigned)ceil_div(cols, 16)), block(kSkinnyWaves * 64);
  if (M <= 16) hipLaunchKernelGGL((skinny_kernel<KIND, 1, DUAL, PAIR, EPI>), grid, block, 0, c.stream, g);
  else if (M <= 32) hipLaunchKernelGGL((skinny_kernel<KIND, 2, DUAL, PAIR, EPI>), grid, block, 0, c.stream, g);
  else if constexpr (few_rows(KIND) > 32) hipLaunchKernelGGL((skinny_kernel<KIND, 4, DUAL, PAIR, EPI>), grid, block, 0, c.stream, g);
  NN_LAUNCHED("product of few rows");
  return 0;
}

// y[m, n] = sum_k a[m, k] b[k, n] of at most few_rows(3) fp32 rows; b1 follows b0 along k from row `turn` on, K: all rows of k
template <class EPI>
int skinny_down(Call& c, const Operand& a, const Operand& b0, const Operand& b1, const int64_t M, const int64_t N, const int64_t K, const int64_t turn,
                const EPI& epi) {
  const int64_t cols = ceil_div(N, 64), units = ceil_div(K, 16);
  // four workgroups a CU, each with two turns of its wavefronts or more
  const int64_t want = std::max<int64_t>(1, std::min(units / (2 * kDownWaves), 1024 / cols)), per = ceil_div(units, want), splits = ceil_div(units, per);
  const int64_t ld = round_up(N, 64);
  char* part = splits > 1 ? c.take(splits * M * ld * 4) : nullptr;
  c.note(0, (int)splits);
  if (c.dry() || M == 0) return 0;
  auto start = [&](const auto& e) {
    typedef std::remove_cv_t<std::remove_reference_t<decltype(e)>> E;
    const GemmArgs<E> g{a, {b0, b1}, M, (int)N, (int)units, (int)turn, (int)per, 0, 0, 0, e};
    const dim3 grid((unsigned)cols, (unsigned)splits), block(kDownWaves * 64);
    if (M <= 16) hipLaunchKernelGGL((skinny_down_kernel<1, E>), grid, block, 0, c.stream, g);
    else if (M <= 32) hipLaunchKernelGGL((skinny_down_kernel<2, E>), grid, block, 0, c.stream, g);
    else hipLaunchKernelGGL((skinny_down_kernel<4, E>), grid, block, 0, c.stream, g);
  };
  if (splits == 1) {
    start(epi);
    NN_LAUNCHED("product of few rows");
    return 0;
  }
  start(PartialEpi{(uint32_t*)part, M, ld});
  NN_LAUNCHED("product of few rows");
  hipLaunchKernelGGL((split_reduce_kernel<float, false, EPI>), dim3((unsigned)ceil_div(ld / 8 * M, 256)), dim3(256), 0, c.stream, (const float*)part,
                     (int)splits, M, ld, epi);
  NN_LAUNCHED("split sum");
  return 0;
}
// w[r, c] = sum_m p[m, r] x[m, c] of few fp32 rows into `to`; R rows r (both halves of `to` with what lies between)
inline int outer(Call& c, const Operand& p, const Operand& x, const int64_t M, const int64_t R, const StoreEpi<SDFNN_F32>& to) {
  c.note(0, 1);
  if (c.dry() || R == 0) return 0;
  hipLaunchKernelGGL(outer_kernel, dim3((unsigned)ceil_div(to.N, 256), (unsigned)ceil_div(R, 64)), dim3(256), 0, c.stream, OuterArgs{p, x, M, to});
  NN_LAUNCHED("outer product");
  return 0;
}

// Copies of operands with rows of whole steps, gathered and made in one launch.  ES: bytes of an element (4: three bf16 parts)
template <int ES>
struct Packs {
  PackBatch b{};
  int64_t blocks = 0;
  // to: where the copy goes; NULL: into the workspace
  Operand add(Call& c, const void* src, const int64_t ld, const int64_t rows, const int64_t cols, const int64_t pad, char* to = nullptr) {
    const int64_t es = ES == 1 ? 1 : 2, plane = rows * pad * 2;
    char* dst = to ? to : c.take(ES == 4 ? 3 * plane : rows * pad * es);
    if (rows > 0 && pad > 0) {
      b.a[b.count] = {src, ld, rows, cols, dst, pad, plane, pad};
      b.first[b.count++] = (unsigned)blocks;
      blocks += std::min<int64_t>(ceil_div(rows * (pad / 8), 256), 1 << 21);
    }
    return {dst, pad * es, plane, rows, pad * es};
  }
  int launch(Call& c) {
    if (c.dry() || b.count == 0) return 0;
    b.first[b.count] = (unsigned)blocks;
    hipLaunchKernelGGL((pack_rows_kernel<ES>), dim3((unsigned)blocks), dim3(256), 0, c.stream, b);
    NN_LAUNCHED("operand copy");
    return 0;
  }
};
