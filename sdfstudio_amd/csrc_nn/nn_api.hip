// libsdfnn.so: the gated feed-forward block's operators (include/sdfnn.h).  gfx950 only.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "nn_launch.h"
#include "norm_kernels.h"

namespace {
thread_local char g_err[512] = "";
}
void sdfnn_set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}

#define NN_TRY(expr)                \
  do {                              \
    if (const int rc_ = (expr)) return rc_; \
  } while (0)

namespace {

constexpr int64_t kMaxRows = 0x7fffffff, kMaxDim = (int64_t)1 << 24;

bool aligned16(const void* p, const int64_t ld_bytes) { return ((uintptr_t)p & 15) == 0 && (ld_bytes & 15) == 0; }

// Tiles reach the rows of an operand that they read in place through 31-bit offsets (gemm_core.h): 256 of them lie below 2^31 bytes
#define NN_REACH(what, ld, es) NN_REQUIRE((ld) <= ((int64_t)1 << 23) / (es) - 1, "%s: rows %lld bytes apart: less than 8 MiB", what, (long long)((ld) * (es)))

// ---------------------------------------------------------------------------------------------- norm
// f(IC<TPR>, IC<NV>, IC<U>) for the row width: how many threads and registers hold a row, how many rows at a time (norm_kernels.h); wide()
// for rows that they do not hold
template <int N> using IC = std::integral_constant<int, N>;
template <class F, class W>
void pick_row(const int64_t dim, F&& f, W&& wide) {
  if (dim <= 64) f(IC<8>{}, IC<1>{}, IC<2>{});
  else if (dim <= 128) f(IC<16>{}, IC<1>{}, IC<2>{});
  else if (dim <= 256) f(IC<32>{}, IC<1>{}, IC<2>{});
  else if (dim <= 512) f(IC<64>{}, IC<1>{}, IC<2>{});
  else if (dim <= 1024) f(IC<64>{}, IC<2>{}, IC<1>{});
  else if (dim <= 2048) f(IC<64>{}, IC<4>{}, IC<1>{});
  else if (dim <= 4096) f(IC<256>{}, IC<2>{}, IC<1>{});
  else if (dim <= 8192) f(IC<256>{}, IC<4>{}, IC<1>{});
  else wide();
}
// rows that a workgroup of that shape takes at a time
constexpr int64_t rows_at_once(const int tpr, const int u) { return (tpr > 256 ? 1 : 256 / tpr) * u; }
dim3 row_grid(const int64_t rows, const int tpr, const int u) { return dim3((unsigned)ceil_div(rows, rows_at_once(tpr, u))); }
// f(arguments) for pieces of the rows, each of less than the 2^32 threads that a launch may have
template <int DT, class F>
void row_pieces(const NormArgs& a, const int tpr, const int u, F&& f) {
  typedef elem_t<DT> T;
  const int64_t most = tpr > 256 ? (int64_t)1 << 21 : rows_at_once(tpr, u) << 23;
  for (int64_t at = 0; at < a.rows; at += most) {
    NormArgs b = a;
    b.rows = std::min(most, a.rows - at);
    b.x = (const T*)a.x + at * a.ldx;
    if (a.r) b.r = (const T*)a.r + at * a.ldr;
    if (a.dy) b.dy = (const T*)a.dy + at * a.lddy;
    if (a.dh) b.dh = (const T*)a.dh + at * a.lddh;
    if (a.y) b.y = (T*)a.y + at * a.dim;
    if (a.h) b.h = (T*)a.h + at * a.dim;
    if (a.dx) b.dx = (T*)a.dx + at * a.dim;
    if (a.inv) b.inv = a.inv + at;
    if (a.q) b.q = a.q + at * a.dim;
    if (a.scales) b.scales = a.scales + at;
    f(b);
  }
}

int check_norm(const char* what, const void* x, const int64_t ldx, const void* residual, const int64_t ldr, const int32_t dtype,
               const int64_t rows, const int64_t dim) {
  NN_REQUIRE(dtype >= SDFNN_F32 && dtype <= SDFNN_F16, "%s: dtype %d", what, dtype);
  NN_REQUIRE(rows >= 0 && rows <= kMaxRows, "%s: %lld rows", what, (long long)rows);
  NN_REQUIRE(dim >= 1 && dim <= kMaxDim, "%s: rows of %lld elements (1 .. 2^24)", what, (long long)dim);
  NN_REQUIRE(x, "%s: null tensor", what);
  NN_REQUIRE(ldx >= dim && (!residual || ldr >= dim), "%s: a row stride is smaller than the row", what);
  return 0;
}

#define NN_ROW_SHAPE constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, U = decltype(u)::value
template <int DT>
int norm_forward(const NormArgs& a, hipStream_t s) {
  pick_row(a.dim, [&](auto tpr, auto nv, auto u) {
    NN_ROW_SHAPE;
    row_pieces<DT>(a, TPR, U, [&](const NormArgs& b) {
      hipLaunchKernelGGL((rms_norm_fwd_kernel<DT, TPR, NV, U>), row_grid(b.rows, TPR, U), dim3(256), 0, s, b);
    });
  }, [&] {
    row_pieces<DT>(a, kWide, 1, [&](const NormArgs& b) {
      hipLaunchKernelGGL((rms_norm_fwd_wide_kernel<DT>), row_grid(b.rows, kWide, 1), dim3(kWide), 0, s, b);
    });
  });
  NN_LAUNCHED("rms_norm_forward");
  return 0;
}
template <int DT>
int norm_quantize(const NormArgs& a, hipStream_t s) {
  pick_row(a.dim, [&](auto tpr, auto nv, auto u) {
    NN_ROW_SHAPE;
    row_pieces<DT>(a, TPR, U, [&](const NormArgs& b) {
      const dim3 grid = row_grid(b.rows, TPR, U), block(256);
      if (!b.w && !b.r) hipLaunchKernelGGL((rms_norm_quant_kernel<DT, TPR, NV, U, true>), grid, block, 0, s, b);
      else hipLaunchKernelGGL((rms_norm_quant_kernel<DT, TPR, NV, U, false>), grid, block, 0, s, b);
    });
  }, [&] {
    row_pieces<DT>(a, kWide, 1, [&](const NormArgs& b) {
      hipLaunchKernelGGL((rms_norm_quant_wide_kernel<DT>), row_grid(b.rows, kWide, 1), dim3(kWide), 0, s, b);
    });
  });
  NN_LAUNCHED("rms_norm_quantize");
  return 0;
}

// workgroups of the backward pass (= partial sums of dweight): enough to fill the chip, but with at least two turns of rows each, so that their
// sums stay small beside the tensors
int64_t bwd_groups(const int64_t rows, const int64_t dim) {
  int64_t groups = std::min<int64_t>(rows, 256);
  pick_row(dim, [&](auto tpr, auto, auto u) {
    groups = std::min<int64_t>(ceil_div(rows, 2 * rows_at_once(decltype(tpr)::value, decltype(u)::value)), dim <= 8192 ? 1024 : 256);
  }, [] {});
  return std::max<int64_t>(1, groups);
}
template <int DT>
int norm_backward(NormArgs a, elem_t<DT>* dw, hipStream_t s) {
  const int64_t groups = bwd_groups(a.rows, a.dim);
  if (a.rows > 0)
    pick_row(a.dim, [&](auto tpr, auto nv, auto u) {
      NN_ROW_SHAPE;
      if (dw) hipLaunchKernelGGL((rms_norm_bwd_kernel<DT, TPR, NV, U, true>), dim3((unsigned)groups), dim3(256), 0, s, a);
      else row_pieces<DT>(a, TPR, U, [&](const NormArgs& b) {
        hipLaunchKernelGGL((rms_norm_bwd_kernel<DT, TPR, NV, U, false>), row_grid(b.rows, TPR, U), dim3(256), 0, s, b);
      });
    }, [&] {
      if (a.dx) row_pieces<DT>(a, kWide, 1, [&](const NormArgs& b) {
        hipLaunchKernelGGL((rms_norm_bwd_wide_kernel<DT>), row_grid(b.rows, kWide, 1), dim3(kWide), 0, s, b);
      });
      if (dw) hipLaunchKernelGGL((rms_norm_dw_wide_kernel<DT>), dim3((unsigned)ceil_div(a.dim, 256), (unsigned)groups), dim3(256), 0, s, a);
    });
  NN_LAUNCHED("rms_norm_backward");
  if (!dw) return 0;
  hipLaunchKernelGGL((rms_norm_dw_reduce_kernel<DT>), dim3((unsigned)ceil_div(a.dim, 32)), dim3(1024), 0, s, a.partial,
                     a.rows > 0 ? (int)groups : 0, a.dim, dw);
  NN_LAUNCHED("rms_norm_backward (weight)");
  return 0;
}

// ---------------------------------------------------------------------------------------------- 8-bit products
template <int DT, bool DUAL>
int int8_products(Call& c, const int8_t* q, const int64_t ldq, const int8_t* w0, const int64_t ld0, const int8_t* w1, const int64_t ld1,
                  const int64_t rows, const int64_t n, const int64_t k, const Int8Epi<DT>& epi) {
  Operand a{(const char*)q, ldq, 0, rows, k}, b0{(const char*)w0, ld0, 0, n, k}, b1{(const char*)w1, ld1, 0, n, k};
  if (rows <= few_rows(2)) return skinny<2, DUAL>(c, a, b0, b1, rows, n, n, epi);
  if (k % 16) {  // the tiles read 16 bytes at a time
    Packs<1> packs;
    const int64_t pad = round_up(k, 128);
    a = packs.add(c, q, ldq, rows, k, pad);
    b0 = packs.add(c, w0, ld0, n, k, pad);
    if (DUAL) b1 = packs.add(c, w1, ld1, n, k, pad);
    NN_TRY(packs.launch(c));
  }
  const int64_t nk = ceil_div(k, 128);
  return product<2, 1, DUAL, kRows>(c, a, b0, b1, rows, n, nk, nk, epi);
}

int check_int8(const char* what, const int8_t* q, const int64_t ldq, const int8_t* w0, const int64_t ld0, const int8_t* w1, const int64_t ld1,
               const int32_t dtype, const int64_t rows, const int64_t n, const int64_t k) {
  NN_REQUIRE(dtype >= SDFNN_F32 && dtype <= SDFNN_F16, "%s: dtype %d", what, dtype);
  NN_REQUIRE(rows >= 0 && rows <= kMaxRows, "%s: %lld rows", what, (long long)rows);
  NN_REQUIRE(n >= 1 && n <= kMaxDim, "%s: %lld channels (1 .. 2^24)", what, (long long)n);
  NN_REQUIRE(k >= 1 && k <= 131072, "%s: k = %lld: the 32-bit sum is exact for 1 .. 131072", what, (long long)k);
  NN_REQUIRE(q && w0 && w1, "%s: null tensor", what);
  NN_REQUIRE(ldq >= k && ld0 >= k && ld1 >= k, "%s: a row stride is smaller than the row", what);
  if (rows > few_rows(2) && k % 16 == 0) {
    for (const int64_t ld : {ldq, ld0, ld1}) NN_REACH(what, ld, 1);
    NN_REQUIRE(aligned16(q, ldq) && aligned16(w0, ld0) && aligned16(w1, ld1),
               "%s: with k a multiple of 16 rows have to start at 16-byte boundaries", what);
  }
  return 0;
}

template <class F>
int by_dtype(const int32_t dtype, F&& f) {
  if (dtype == SDFNN_F32) return f(IC<SDFNN_F32>{});
  if (dtype == SDFNN_BF16) return f(IC<SDFNN_BF16>{});
  return f(IC<SDFNN_F16>{});
}

// ---------------------------------------------------------------------------------------------- gated MLP
template <int DT> struct Kind {  // of the tile and of the few-row product
  static constexpr int tile = DT == SDFNN_F16 ? 1 : 0, few = DT == SDFNN_F32 ? 3 : DT == SDFNN_F16 ? 1 : 0;
  static constexpr int terms = DT == SDFNN_F32 ? 6 : 1, es = elem_size(DT);
  static constexpr bool f32 = DT == SDFNN_F32;
};

// [rows, cols] where it lies if the tiles can read it there (16-bit rows of a multiple of 8), else a copy with rows of whole steps
template <int DT>
Operand operand(Call& c, Packs<Kind<DT>::es>& packs, const void* p, const int64_t ld, const int64_t rows, const int64_t cols, char* to = nullptr) {
  if (!Kind<DT>::f32 && cols % 8 == 0) return {(const char*)p, ld * 2, 0, rows, cols * 2};
  return packs.add(c, p, ld, rows, cols, round_up(cols, 64), to);
}

// what a forward pass keeps: fu, fg [rows][Fp] fp32 (GatedEpi), then a [rows][Fp]: 16-bit types and few rows of fp32 as it is, else as the
// three bf16 parts that the products read; behind them the parts of x, which the backward reads again (to split x once more takes 223 us of
// 8.4 ms at 524288 x 256 x 512)
template <int DT>
struct Saved {
  float *fu, *fg;
  char *a, *x;
  int64_t plane;
  Saved(void* p, const int64_t M, const int64_t Fp)
      : fu((float*)p), fg(fu + M * Fp), a((char*)(fg + M * Fp)), x(a + a_size(M, Fp)), plane(parts(M) ? M * Fp * 2 : 0) {}
  static bool parts(const int64_t M) { return Kind<DT>::f32 && M > few_rows(Kind<DT>::few); }
  static int64_t a_size(const int64_t M, const int64_t Fp) { return M * Fp * (parts(M) ? 6 : Kind<DT>::es); }
  static int64_t size(const int64_t M, const int64_t D, const int64_t Fp) {
    return M * Fp * 8 + a_size(M, Fp) + (parts(M) ? M * round_up(D, 64) * 6 : 0);
  }
};

template <int DT>
int gated_forward(Call& c, const void* x, const int64_t ldx, const void* wg, const void* wu, const void* wd, const int act, const int64_t M,
                  const int64_t D, const int64_t F, const int64_t O, void* saved, void* y) {
  typedef elem_t<DT> T;
  typedef Kind<DT> K;
  const int64_t Fp = round_up(F, 64), es = K::es;
  Saved<DT> sv(saved, M, Fp);
  // Up to 16 rows of 16 bits the hidden row goes into the second product as two numbers (GatedEpi): they fit the few-row product's 32 rows, which is bound
  // by the weights.  4096 x 16384 bf16, one number / two: 1 row 84 / 84 us, 8 rows 88 / 90, 16 rows 90 / 103; 17 rows 97 / 111, 32 rows 114 / 140
  // (the operand rows, read by every workgroup, are the time by then).
  const bool few = M <= few_rows(K::few), two = !K::f32 && 2 * M <= few_rows(K::few);
  if (!saved) sv.fu = sv.fg = nullptr, sv.a = two ? nullptr : c.take(Saved<DT>::a_size(M, Fp));
  const StoreEpi<DT> se{(T*)y, nullptr, M, M, 0, O, (int)O};
  if (few) {
    const Operand xo{(const char*)x, ldx * es, 0, M, D * es}, g{(const char*)wg, D * es, 0, F, D * es}, u{(const char*)wu, D * es, 0, F, D * es};
    const Operand d{(const char*)wd, F * es, 0, O, F * es};
    if constexpr (!K::f32)
      if (two) {
        char* a2 = c.take(2 * M * Fp * es);
        const GatedEpi<DT, true> ge{(T*)sv.a, 0, sv.fu, sv.fg, (int)Fp, act, (T*)a2, M * Fp};
        NN_TRY((skinny<K::few, true>(c, xo, g, u, M, F, Fp, ge)));
        return skinny<K::few, false, true>(c, {a2, Fp * es, 0, 2 * M, F * es}, d, d, 2 * M, O, O, se);
      }
    const GatedEpi<DT> ge{(T*)sv.a, 0, sv.fu, sv.fg, (int)Fp, act};
    NN_TRY((skinny<K::few, true>(c, xo, g, u, M, F, Fp, ge)));
    return skinny<K::few, false>(c, {sv.a, Fp * es, 0, M, F * es}, d, d, M, O, O, se);
  }
  const GatedEpi<DT> ge{(T*)sv.a, sv.plane, sv.fu, sv.fg, (int)Fp, act};
  Packs<K::es> packs;
  const Operand xo = operand<DT>(c, packs, x, ldx, M, D, saved && K::f32 ? sv.x : nullptr), g = operand<DT>(c, packs, wg, D, F, D), u = operand<DT>(c, packs, wu, D, F, D);
  const Operand d = operand<DT>(c, packs, wd, F, O, F);
  NN_TRY(packs.launch(c));
  const int64_t nd = ceil_div(D, 64), nf = Fp / 64;
  NN_TRY((product<K::tile, K::terms, true, kRows>(c, xo, g, u, M, F, nd, nd, ge)));
  const Operand ao{sv.a, Fp * 2, sv.plane, M, Fp * 2};
  return product<K::tile, K::terms, false, kRows>(c, ao, d, d, M, O, nf, nf, se);
}

// up to few_rows fp32 rows: no operand is copied or split
int gated_backward_few(Call& c, const char* x, const int64_t ldx, const char* wg, const char* wu, const char* wd, const Saved<SDFNN_F32>& sv,
                       const char* dy, const int64_t lddy, const int64_t M, const int64_t D, const int64_t F, const int64_t O, float* dx, float* dwg,
                       float* dwu, float* dwd) {
  const int64_t Fp = round_up(F, 64);
  const Operand dgu{c.take(M * Fp * 8), Fp * 8, 0, M, Fp * 8}, dyo{dy, lddy * 4, 0, M, O * 4};
  if (dx || dwg) {
    const Operand d{wd, F * 4, 0, O, F * 4};
    const GatedBwdEpi<SDFNN_F32> be{sv.fu, sv.fg, const_cast<char*>(dgu.p), 0, (int)Fp};
    NN_TRY(skinny_down(c, dyo, d, d, M, F, O, round_up(O, 16), be));
  }
  if (dx) {
    const Operand g{wg, D * 4, 0, F, D * 4}, u{wu, D * 4, 0, F, D * 4};
    const StoreEpi<SDFNN_F32> se{dx, nullptr, M, M, 0, D, (int)D};
    NN_TRY(skinny_down(c, dgu, g, u, M, D, 2 * Fp, Fp, se));
  }
  if (dwd) NN_TRY(outer(c, dyo, {sv.a, Fp * 4, 0, M, F * 4}, M, O, {dwd, nullptr, O, O, 0, F, (int)F}));
  if (dwg) NN_TRY(outer(c, dgu, {x, ldx * 4, 0, M, D * 4}, M, 2 * Fp, {dwg, dwu, Fp, F, F, D, (int)D}));
  return 0;
}

template <int DT>
int gated_backward(Call& c, const void* x, const int64_t ldx, const void* wg, const void* wu, const void* wd, const void* saved, const void* dy,
                   const int64_t lddy, const int64_t M, const int64_t D, const int64_t F, const int64_t O, void* dx, void* dwg, void* dwu,
                   void* dwd) {
  typedef elem_t<DT> T;
  typedef Kind<DT> K;
  const int64_t Fp = round_up(F, 64);
  const Saved<DT> sv(const_cast<void*>(saved), M, Fp);
  if constexpr (K::f32)
    if (!Saved<DT>::parts(M)) return gated_backward_few(c, (const char*)x, ldx, (const char*)wg, (const char*)wu, (const char*)wd, sv, (const char*)dy, lddy, M, D, F, O, (float*)dx,
                                                        (float*)dwg, (float*)dwu, (float*)dwd);
  // gradients of g and u, side by side
  const int64_t dplane = M * 2 * Fp * 2;
  const Operand dgu{c.take((K::f32 ? 3 : 1) * dplane), 2 * Fp * 2, dplane, M, 2 * Fp * 2};
  const int64_t nm = ceil_div(M, 64), nf = Fp / 64;
  Packs<K::es> packs;
  const Operand dyo = operand<DT>(c, packs, dy, lddy, M, O);
  Operand d{}, g{}, u{}, xo{};
  const Operand a{sv.a, Fp * 2, sv.plane, M, Fp * 2};
  if (dx || dwg) d = operand<DT>(c, packs, wd, F, O, F);
  if (dx) g = operand<DT>(c, packs, wg, D, F, D), u = operand<DT>(c, packs, wu, D, F, D);
  const int64_t Dp = round_up(D, 64);
  if (dwg) xo = Saved<DT>::parts(M) ? Operand{sv.x, Dp * 2, M * Dp * 2, M, Dp * 2} : operand<DT>(c, packs, x, ldx, M, D);
  NN_TRY(packs.launch(c));
  const int64_t start = c.used;  // the split sums of one product make room for those of the next
  int64_t most = start;
  auto next = [&]() { most = std::max(most, c.used), c.used = start; };
  if (dx || dwg) {
    const GatedBwdEpi<DT> be{sv.fu, sv.fg, const_cast<char*>(dgu.p), dgu.plane, (int)Fp};
    const int64_t no = ceil_div(O, 64);
    NN_TRY((product<K::tile, K::terms, false, kRowsDown>(c, dyo, d, d, M, F, no, no, be)));
    next();
  }
  if (dx) {
    const StoreEpi<DT> se{(T*)dx, nullptr, M, M, 0, D, (int)D};
    NN_TRY((product<K::tile, K::terms, false, kRowsDown>(c, dgu, g, u, M, D, 2 * nf, nf, se)));
    next();
  }
  if (dwd) {
    const StoreEpi<DT> se{(T*)dwd, nullptr, O, O, 0, F, (int)F};
    NN_TRY((product<K::tile, K::terms, false, kDown>(c, dyo, a, a, O, F, nm, nm, se)));
    next();
  }
  if (dwg) {
    const StoreEpi<DT> se{(T*)dwg, (T*)dwu, Fp, F, F, D, (int)D};
    NN_TRY((product<K::tile, K::terms, false, kDown>(c, dgu, xo, xo, 2 * Fp, D, nm, nm, se)));
    next();
  }
  c.used = most;
  return 0;
}

int check_gated(const char* what, const int32_t dtype, const int32_t act, const int64_t rows, const int64_t dim, const int64_t hidden,
                const int64_t out) {
  NN_REQUIRE(dtype >= SDFNN_F32 && dtype <= SDFNN_F16, "%s: dtype %d", what, dtype);
  NN_REQUIRE(act >= SDFNN_SILU && act <= SDFNN_RELU, "%s: activation %d", what, act);
  NN_REQUIRE(rows >= 0 && rows <= kMaxRows, "%s: %lld rows", what, (long long)rows);
  NN_REQUIRE(dim >= 1 && hidden >= 1 && out >= 1 && dim <= 1 << 20 && hidden <= 1 << 20 && out <= 1 << 20,
             "%s: widths %lld, %lld, %lld (1 .. 2^20)", what, (long long)dim, (long long)hidden, (long long)out);
  return 0;
}

// What a call needs and which kernels it takes, without launching anything
int plan_int8(Call& c, const int64_t rows, const int64_t n, const int64_t k, const int32_t projections) {
  if (rows < 0 || rows > kMaxRows || n < 1 || n > kMaxDim || k < 1 || k > 131072 || projections < 1 || projections > 2) return -1;
  const Int8Epi<SDFNN_F32> epi{};
  if (projections == 1) return int8_products<SDFNN_F32, false>(c, nullptr, k, nullptr, k, nullptr, k, rows, n, k, epi);
  return int8_products<SDFNN_F32, true>(c, nullptr, k, nullptr, k, nullptr, k, rows, n, k, epi);
}
int plan_gated(Call& c, const char* what, const int32_t dtype, const int64_t rows, const int64_t dim, const int64_t hidden, const int64_t out,
               const int32_t backward) {
  NN_TRY(check_gated(what, dtype, 0, rows, dim, hidden, out));
  char some = 0;
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (backward) return gated_backward<DT>(c, nullptr, dim, nullptr, nullptr, nullptr, nullptr, nullptr, out, rows, dim, hidden, out, &some, &some, &some, &some);
    return gated_forward<DT>(c, nullptr, dim, nullptr, nullptr, nullptr, 0, rows, dim, hidden, out, nullptr, nullptr);
  });
}
int32_t product_of(const Call& c, const int32_t index, int32_t* splits) {
  NN_REQUIRE(index >= 0 && index < c.products, "product %d of %d", (int)index, c.products);
  if (splits) *splits = c.splits[index];
  return c.tile[index];
}

}  // namespace

extern "C" {

int sdfnn_version(void) { return 101; }  // 101: sdfnn_int8_product, sdfnn_gated_product
const char* sdfnn_last_error(void) { return g_err; }

int sdfnn_rms_norm_forward(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int32_t dtype, int64_t rows,
                           int64_t dim, float eps, void* y, void* h, float* inv, sdfnn_stream_t stream) {
  NN_TRY(check_norm("rms_norm_forward", x, ldx, residual, ldr, dtype, rows, dim));
  NN_REQUIRE(weight && y, "rms_norm_forward: null tensor");
  NN_REQUIRE(eps >= 0.0f && eps < INFINITY, "rms_norm_forward: eps %g", (double)eps);
  if (rows == 0) return 0;
  NormArgs a{};
  a.x = x, a.ldx = ldx, a.r = residual, a.ldr = ldr, a.w = weight, a.rows = rows, a.dim = dim, a.eps = eps;
  a.y = y, a.h = residual ? h : nullptr, a.inv = inv;
  return by_dtype(dtype, [&](auto dt) { return norm_forward<decltype(dt)::value>(a, (hipStream_t)stream); });
}

int64_t sdfnn_rms_norm_backward_workspace_size(int64_t rows, int64_t dim) {
  if (rows < 0 || rows > kMaxRows || dim < 1 || dim > kMaxDim) return -1;
  return bwd_groups(rows, dim) * dim * 4;
}

int sdfnn_rms_norm_backward(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, const float* inv,
                            const void* dy, int64_t lddy, const void* dh, int64_t lddh, int32_t dtype, int64_t rows, int64_t dim, void* dx,
                            void* dweight, void* workspace, int64_t workspace_bytes, sdfnn_stream_t stream) {
  NN_TRY(check_norm("rms_norm_backward", x, ldx, residual, ldr, dtype, rows, dim));
  NN_REQUIRE(weight && inv, "rms_norm_backward: null tensor");
  NN_REQUIRE(dy || dh, "rms_norm_backward: neither output has a gradient");
  NN_REQUIRE((!dy || lddy >= dim) && (!dh || lddh >= dim), "rms_norm_backward: a row stride is smaller than the row");
  NN_REQUIRE(!dweight || (workspace && workspace_bytes >= sdfnn_rms_norm_backward_workspace_size(rows, dim)),
             "rms_norm_backward: the workspace is too small");
  if (!dx && !dweight) return 0;
  NormArgs a{};
  a.x = x, a.ldx = ldx, a.r = residual, a.ldr = ldr, a.w = weight, a.rows = rows, a.dim = dim;
  a.dy = dy, a.lddy = lddy, a.dh = dh, a.lddh = lddh, a.dx = dx, a.inv = const_cast<float*>(inv), a.partial = (float*)workspace;
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return norm_backward<DT>(a, (elem_t<DT>*)dweight, (hipStream_t)stream);
  });
}

int sdfnn_rms_norm_quantize(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int32_t dtype, int64_t rows,
                            int64_t dim, float eps, int8_t* q, float* scales, void* h, sdfnn_stream_t stream) {
  NN_TRY(check_norm("rms_norm_quantize", x, ldx, residual, ldr, dtype, rows, dim));
  NN_REQUIRE(q && scales, "rms_norm_quantize: null tensor");
  NN_REQUIRE(!weight || (eps >= 0.0f && eps < INFINITY), "rms_norm_quantize: eps %g", (double)eps);
  if (rows == 0) return 0;
  NormArgs a{};
  a.x = x, a.ldx = ldx, a.r = residual, a.ldr = ldr, a.w = weight, a.rows = rows, a.dim = dim, a.eps = eps;
  a.q = q, a.scales = scales, a.h = residual ? h : nullptr;
  return by_dtype(dtype, [&](auto dt) { return norm_quantize<decltype(dt)::value>(a, (hipStream_t)stream); });
}

int64_t sdfnn_int8_linear_workspace_size(int64_t rows, int64_t n, int64_t k, int32_t projections) {
  Call c{};
  return plan_int8(c, rows, n, k, projections) ? -1 : c.used;
}

int32_t sdfnn_int8_product(int64_t rows, int64_t n, int64_t k, int32_t projections, int32_t* splits) {
  Call c{};
  return plan_int8(c, rows, n, k, projections) ? -1 : product_of(c, 0, splits);
}

int sdfnn_int8_linear(const int8_t* q, int64_t ldq, const float* sq, const int8_t* w, int64_t ldw, const float* sw, const float* bias,
                      int32_t dtype, int64_t rows, int64_t n, int64_t k, void* y, void* workspace, int64_t workspace_bytes,
                      sdfnn_stream_t stream) {
  NN_TRY(check_int8("int8_linear", q, ldq, w, ldw, w, ldw, dtype, rows, n, k));
  NN_REQUIRE(sq && sw && y, "int8_linear: null tensor");
  const int64_t need = sdfnn_int8_linear_workspace_size(rows, n, k, 1);
  NN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "int8_linear: the workspace is too small (%lld of %lld bytes)",
             (long long)workspace_bytes, (long long)need);
  if (rows == 0) return 0;
  Call c{workspace ? (char*)workspace : (char*)y, 0, (hipStream_t)stream};
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const Int8Epi<DT> epi{(elem_t<DT>*)y, sq, sw, nullptr, bias, (int)n, 0};
    return int8_products<DT, false>(c, q, ldq, w, ldw, w, ldw, rows, n, k, epi);
  });
}

int sdfnn_int8_gated_linear(const int8_t* q, int64_t ldq, const float* sq, const int8_t* w_gate, int64_t ldg, const float* s_gate,
                            const int8_t* w_up, int64_t ldu, const float* s_up, int32_t act, int32_t dtype, int64_t rows, int64_t n,
                            int64_t k, void* y, void* workspace, int64_t workspace_bytes, sdfnn_stream_t stream) {
  NN_TRY(check_int8("int8_gated_linear", q, ldq, w_gate, ldg, w_up, ldu, dtype, rows, n, k));
  NN_REQUIRE(act >= SDFNN_SILU && act <= SDFNN_RELU, "int8_gated_linear: activation %d", act);
  NN_REQUIRE(sq && s_gate && s_up && y, "int8_gated_linear: null tensor");
  const int64_t need = sdfnn_int8_linear_workspace_size(rows, n, k, 2);
  NN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "int8_gated_linear: the workspace is too small (%lld of %lld bytes)",
             (long long)workspace_bytes, (long long)need);
  if (rows == 0) return 0;
  Call c{workspace ? (char*)workspace : (char*)y, 0, (hipStream_t)stream};
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const Int8Epi<DT> epi{(elem_t<DT>*)y, sq, s_gate, s_up, nullptr, (int)n, act};
    return int8_products<DT, true>(c, q, ldq, w_gate, ldg, w_up, ldu, rows, n, k, epi);
  });
}

int64_t sdfnn_gated_saved_size(int32_t dtype, int64_t rows, int64_t dim, int64_t hidden) {
  if (check_gated("gated_saved_size", dtype, 0, rows, dim, hidden, 1)) return -1;
  const int64_t Fp = round_up(hidden, 64);
  return dtype == SDFNN_F32 ? Saved<SDFNN_F32>::size(rows, dim, Fp) : Saved<SDFNN_BF16>::size(rows, dim, Fp);
}

int64_t sdfnn_gated_workspace_size(int32_t dtype, int64_t rows, int64_t dim, int64_t hidden, int64_t out, int32_t backward) {
  Call c{};
  return plan_gated(c, "gated_workspace_size", dtype, rows, dim, hidden, out, backward) ? -1 : c.used;
}

int32_t sdfnn_gated_product(int32_t dtype, int64_t rows, int64_t dim, int64_t hidden, int64_t out, int32_t backward, int32_t index, int32_t* splits) {
  Call c{};
  return plan_gated(c, "gated_product", dtype, rows, dim, hidden, out, backward) ? -1 : product_of(c, index, splits);
}

int sdfnn_gated_forward(const void* x, int64_t ldx, const void* w_gate, const void* w_up, const void* w_down, int32_t dtype, int32_t act,
                        int64_t rows, int64_t dim, int64_t hidden, int64_t out, void* saved, void* y, void* workspace,
                        int64_t workspace_bytes, sdfnn_stream_t stream) {
  NN_TRY(check_gated("gated_forward", dtype, act, rows, dim, hidden, out));
  NN_REQUIRE(x && w_gate && w_up && w_down && y, "gated_forward: null tensor");
  NN_REQUIRE(ldx >= dim, "gated_forward: a row stride is smaller than the row");
  const int64_t es = elem_size(dtype);
  if (rows > few_rows(0) && es == 2) {
    NN_REQUIRE(dim % 8 || (aligned16(x, ldx * es) && aligned16(w_gate, 0) && aligned16(w_up, 0)),
               "gated_forward: with dim a multiple of 8 rows have to start at 16-byte boundaries");
    NN_REQUIRE(hidden % 8 || aligned16(w_down, 0), "gated_forward: with hidden a multiple of 8 w_down has to start at a 16-byte boundary");
    if (dim % 8 == 0) NN_REACH("gated_forward", ldx, es);
  }
  NN_REQUIRE(!saved || aligned16(saved, 0), "gated_forward: saved has to start at a 16-byte boundary");
  const int64_t need = sdfnn_gated_workspace_size(dtype, rows, dim, hidden, out, 0);
  NN_REQUIRE(rows == 0 || (workspace && aligned16(workspace, 0) && workspace_bytes >= need),
             "gated_forward: the workspace is too small or not aligned (%lld of %lld bytes)", (long long)workspace_bytes, (long long)need);
  if (rows == 0) return 0;
  Call c{(char*)workspace, 0, (hipStream_t)stream};
  return by_dtype(dtype, [&](auto dt) {
    return gated_forward<decltype(dt)::value>(c, x, ldx, w_gate, w_up, w_down, act, rows, dim, hidden, out, saved, y);
  });
}

int sdfnn_gated_backward(const void* x, int64_t ldx, const void* w_gate, const void* w_up, const void* w_down, const void* saved,
                         const void* dy, int64_t lddy, int32_t dtype, int64_t rows, int64_t dim, int64_t hidden, int64_t out,
                         void* dx, void* dw_gate, void* dw_up, void* dw_down, void* workspace, int64_t workspace_bytes,
                         sdfnn_stream_t stream) {
  NN_TRY(check_gated("gated_backward", dtype, 0, rows, dim, hidden, out));
  NN_REQUIRE(x && w_gate && w_up && w_down && dy && saved, "gated_backward: null tensor");
  NN_REQUIRE(ldx >= dim && lddy >= out, "gated_backward: a row stride is smaller than the row");
  NN_REQUIRE(!dw_gate == !dw_up, "gated_backward: dw_gate and dw_up are computed together");
  const int64_t es = elem_size(dtype);
  NN_REQUIRE(es == 4 || ((out % 8 || aligned16(dy, lddy * es)) && (hidden % 8 || aligned16(w_down, 0)) &&
                         (dim % 8 || (aligned16(x, ldx * es) && aligned16(w_gate, 0) && aligned16(w_up, 0)))),
             "gated_backward: rows of a multiple of 8 elements have to start at 16-byte boundaries");
  if (es == 2 && dim % 8 == 0) NN_REACH("gated_backward", ldx, es);
  if (es == 2 && out % 8 == 0) NN_REACH("gated_backward", lddy, es);
  NN_REQUIRE(aligned16(saved, 0), "gated_backward: saved has to start at a 16-byte boundary");
  const int64_t need = sdfnn_gated_workspace_size(dtype, rows, dim, hidden, out, 1);
  NN_REQUIRE(need == 0 || (workspace && aligned16(workspace, 0) && workspace_bytes >= need),
             "gated_backward: the workspace is too small or not aligned (%lld of %lld bytes)", (long long)workspace_bytes, (long long)need);
  Call c{workspace ? (char*)workspace : (char*)saved, 0, (hipStream_t)stream};
  return by_dtype(dtype, [&](auto dt) {
    return gated_backward<decltype(dt)::value>(c, x, ldx, w_gate, w_up, w_down, saved, dy, lddy, rows, dim, hidden, out, dx, dw_gate,
                                               dw_up, dw_down);
  });
}

}  // extern "C"
