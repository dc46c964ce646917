// sdfnn — root-mean-square norm with the residual's addition: forward, 8-bit output, backward.
//
//   h = x + r     inv = (mean(h^2) + eps)^(-1/2)     y = h inv w
//   q = round(127 v / max|v|),  v = h w,  scale = inv max|v| / 127        (inv > 0 divides out of the codes)
//   u = dy w,  n = h inv:   dx = dr = inv (u - n mean(u n)) + dh,   dw = sum over rows of dy n
//
// All three are bound by HBM: every tensor is read or written once.  A row stays in the registers of its threads between the passes that
// the statistic needs (NV groups of 8 elements a thread); the backward forms h from x and r again instead of reading a stored h, because
// the stored one is rounded to the type.
//
// Eight to 64 lanes a row up to 2048 elements (no barrier and no LDS: the sums are joined by lane permutations), U rows of narrow ones at a
// time; a workgroup of 256 threads a row above.  Every workgroup of a forward pass takes its rows once: a loop over rows saves the loads of the weight
// but waits for its own stores before the next rows' loads arrive (the counter of both is one), 202 us where the launch below takes 177.  The backward
// pass has to walk: it keeps the sums of dw.  Rows beyond 8192 elements go through kernels of their own that read them twice (the second time
// from L2).  bf16, 524288 x 256 with a residual: forward 177 us = 6.1 TB/s, backward 259 us = 5.2 TB/s; fp16 to codes 89 us = 4.5 TB/s.
#pragma once
#include "nn_common.h"

struct NormArgs {
  const void *x, *r, *w, *dy, *dh;
  int64_t ldx, ldr, lddy, lddh;
  int64_t rows, dim;
  float eps;
  void *y, *h, *dx;
  float* inv;      // forward: written (may be NULL); backward: read
  int8_t* q;
  float* scales;
  float* partial;  // backward: [gridDim.x][dim] sums of dy n
};

// ---- joining a value over the threads of a row
// the value of the lane across: 1, 2: by quads, 4, 8: mirrored (the nearer lanes agree by then), 16, 32: rows of lanes swapped
template <int CTRL>
NN_D uint32_t lane_dpp(const uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
template <int D>
NN_D void lane_pair(const uint32_t v, uint32_t& a, uint32_t& b) {
  if constexpr (D == 32) {
    const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    a = s[0], b = s[1];
  } else if constexpr (D == 16) {
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    a = s[0], b = s[1];
  } else {
    a = v;
    b = lane_dpp<D == 1 ? 0xb1 : D == 2 ? 0x4e : D == 4 ? 0x141 : 0x140>(v);
  }
}
template <int D, class T, class OP>
NN_D T lane_step(const T v, OP op) {
  if constexpr (sizeof(T) == 4) {
    uint32_t a, b;
    lane_pair<D>(__builtin_bit_cast(uint32_t, v), a, b);
    return op(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
  } else {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    uint32_t al, bl, ah, bh;
    lane_pair<D>((uint32_t)u, al, bl);
    lane_pair<D>((uint32_t)(u >> 32), ah, bh);
    return op(__builtin_bit_cast(T, (unsigned long long)ah << 32 | al), __builtin_bit_cast(T, (unsigned long long)bh << 32 | bl));
  }
}
template <int TPR, class T, class OP>
NN_D T row_join(T v, OP op, T* lds) {
  v = lane_step<1>(v, op);
  v = lane_step<2>(v, op);
  v = lane_step<4>(v, op);
  if constexpr (TPR >= 16) v = lane_step<8>(v, op);
  if constexpr (TPR >= 32) v = lane_step<16>(v, op);
  if constexpr (TPR >= 64) v = lane_step<32>(v, op);
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    __syncthreads();  // lds may still be read by the join before this one
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) v = op(v, lds[i]);
  }
  return v;
}
struct AddF { NN_D float operator()(float a, float b) const { return a + b; } };
struct MaxF { NN_D float operator()(float a, float b) const { return fmaxf(a, b); } };
// largest |v| by its bits: as unsigned integers inf lies above every finite value and NaN above inf, so a NaN in a row survives the join
struct MaxBits { template <class T> NN_D T operator()(T a, T b) const { return a > b ? a : b; } };

// f(group index i, first column c, valid elements n) over a thread's groups of 8 columns
template <int TPR, int NV, class F>
NN_D void row_loop(const int64_t dim, const int t, F&& f) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * 8;
    if (c < dim) f(i, (int64_t)c, (int)(dim - c < 8 ? dim - c : 8));
  }
}
NN_D void fill8(float (&v)[8], const float x) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x;
}
constexpr int kWide = 1024;  // threads of a row in the kernels for wide rows
template <class F>
NN_D void wide_loop(const int64_t dim, F&& f) {
  for (int64_t c = (int64_t)threadIdx.x * 8; c < dim; c += kWide * 8) f(c, (int)(dim - c < 8 ? dim - c : 8));
}
template <int DT>
NN_D void load_h(const elem_t<DT>* x, const elem_t<DT>* r, const int64_t c, const int n, float (&h)[8]) {
  load8_n<DT>(x + c, n, h);
  if (r) {
    float t[8];
    load8_n<DT>(r + c, n, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] += t[e];
  }
}

// U rows from `first` on: load(row, u) fetches a row into registers, work(first) handles them
template <int U, class LOAD, class WORK>
NN_D void take_rows(const int64_t rows, const int64_t first, LOAD&& load, WORK&& work) {
  if (first >= rows) return;
#pragma unroll
  for (int u = 0; u < U; ++u) load(first + u < rows ? first + u : rows - 1, u);
  work(first);
}

// ---- forward.  TPR threads a row, GRP rows of them a workgroup, U such rows at a time
template <int DT, int TPR, int NV, int U>
__global__ __launch_bounds__(256) void rms_norm_fwd_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  constexpr int GRP = 256 / TPR;
  __shared__ float lds[16];
  const int t = threadIdx.x % TPR;
  const T *x = (const T*)a.x, *r = (const T*)a.r, *w = (const T*)a.w;
  Raw8<DT> wr[NV], xr[U][NV], rr[U][NV];
  row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) { wr[i] = raw8_n<DT>(w + c, n); });
  take_rows<U>(a.rows, ((int64_t)blockIdx.x * GRP + threadIdx.x / TPR) * U, [&](const int64_t row, const int u) {
    row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
      xr[u][i] = raw8_n<DT>(x + row * a.ldx + c, n);
      if (r) rr[u][i] = raw8_n<DT>(r + row * a.ldr + c, n);
    });
  }, [&](const int64_t first) {
    float h[U][NV][8], ss[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ss[u] = 0.0f;
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t, const int) {
        widen8<DT>(xr[u][i], h[u][i]);
        if (r) {
          float b[8];
          widen8<DT>(rr[u][i], b);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[u][i][e] += b[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) ss[u] = fmaf(h[u][i][e], h[u][i][e], ss[u]);
      });
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float inv = 1.0f / sqrtf(row_join<TPR>(ss[u], AddF{}, lds) / (float)a.dim + a.eps);
      const int64_t row = first + u;
      if (row >= a.rows) continue;  // (U > 1: the threads of a row leave together, and no barrier follows)
      if (t == 0 && a.inv) a.inv[row] = inv;
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
        if (a.h) store8_n<DT>((T*)a.h + row * a.dim + c, n, h[u][i]);
        float o[8];
        widen8<DT>(wr[i], o);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= h[u][i][e] * inv;
        store8_n<DT>((T*)a.y + row * a.dim + c, n, o);
      });
    }
  });
}
template <int DT>
__global__ __launch_bounds__(kWide) void rms_norm_fwd_wide_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  __shared__ float lds[16];
  const int64_t row = blockIdx.x;
  const T *x = (const T*)a.x + row * a.ldx, *r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  float ss = 0.0f;
  wide_loop(a.dim, [&](const int64_t c, const int n) {
    float h[8];
    load_h<DT>(x, r, c, n, h);
    if (a.h) store8_n<DT>((T*)a.h + row * a.dim + c, n, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(h[e], h[e], ss);
  });
  const float inv = 1.0f / sqrtf(row_join<kWide>(ss, AddF{}, lds) / (float)a.dim + a.eps);
  if (threadIdx.x == 0 && a.inv) a.inv[row] = inv;
  wide_loop(a.dim, [&](const int64_t c, const int n) {
    float h[8], o[8];
    load_h<DT>(x, r, c, n, h);
    load8_n<DT>((const T*)a.w + c, n, o);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= h[e] * inv;
    store8_n<DT>((T*)a.y + row * a.dim + c, n, o);
  });
}

// ---- 8-bit output.  The code of v is round(127 v / top) with v = (x + r) w and top = max|v| exact.  In fp32 the quotient is off by two half steps
// (7.6e-6 each, of 127), two more where there is a residual and two more where there is a weight, so only a value that close to the border between
// two codes - one in ten thousand - can go wrong: a row that holds one finds its largest magnitude in 64 bits (among the few values next to the
// largest in fp32; without residual and weight it is known) and decides such values there, each alone.  Ties exist (half the largest value is
// one) and are decided by the quotient of exact numbers, so that they go to even.
NN_D int code_of(const double v, const double top) {
  double c = __builtin_rint(v * 127.0 / top);
  c = c > 127.0 ? 127.0 : c;
  c = c < -127.0 ? -127.0 : c;
  return c == c ? (int)c : 0;
}
// eight values of a row as they were read
template <int DT>
struct Eight {
  Raw8<DT> x, r, w;
  NN_D void load(const elem_t<DT>* px, const elem_t<DT>* pr, const elem_t<DT>* pw, const int64_t c, const int n) {
    x = raw8_n<DT>(px + c, n);
    if (pr) r = raw8_n<DT>(pr + c, n);
    if (pw) w = raw8_n<DT>(pw + c, n);
  }
  NN_D void sum(const bool has_r, float (&h)[8]) const {
    widen8<DT>(x, h);
    if (has_r) {
      float b[8];
      widen8<DT>(r, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] += b[e];
    }
  }
  NN_D void values(const bool has_w, float (&v)[8]) const {  // from h
    if (has_w) {
      float b[8];
      widen8<DT>(w, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= b[e];
    }
  }
  NN_D void exact(const bool has_r, const bool has_w, double (&v)[8]) const {
    float a[8], b[8], k[8];
    widen8<DT>(x, a);
    if (has_r) widen8<DT>(r, b);
    else fill8(b, 0.0f);
    if (has_w) widen8<DT>(w, k);
    else fill8(k, 1.0f);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ((double)a[e] + (double)b[e]) * (double)k[e];
  }
  // the codes of those among v that fp32 cannot decide
  NN_D void decide(const bool has_r, const bool has_w, const float (&v)[8], const float per, const float edge, const double top, int (&q)[8]) const {
    double d[8];
    exact(has_r, has_w, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float k = v[e] * per;
      if (!(fabsf(k - __builtin_rintf(k)) <= edge)) q[e] = code_of(d[e], top);
    }
  }
};
NN_D void largest(const float (&v)[8], uint32_t& big) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu;
    big = b > big ? b : big;
  }
}
// the largest magnitude exactly: the fp32 values are off by two half steps (2^-23, or some of the smallest steps there are), so it is among those
// from top (1 - 2^-21) on
NN_D void largest_exact(const float (&v)[8], const double (&d)[8], const float top, unsigned long long& big) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (fabsf(v[e]) < top * (1.0f - 0x1p-21f) - 0x1p-146f) continue;
    const unsigned long long b = (unsigned long long)__double_as_longlong(d[e]) & 0x7fffffffffffffffull;
    big = b > big ? b : big;
  }
}
// codes in fp32; off: how far the farthest value lies from its code
NN_D void codes8(const float (&v)[8], const float per, int (&q)[8], float& off) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float k = v[e] * per, z = __builtin_rintf(k);
    off = fmaxf(off, fabsf(k - z));
    q[e] = (int)z;
  }
}
NN_D void store_codes(int8_t* out, const int n, const int (&q)[8]) {
  if (n >= 8) {
    Bytes<2, 1> raw;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      raw.w[k] = (uint32_t)(q[4 * k] & 255) | (uint32_t)(q[4 * k + 1] & 255) << 8 | (uint32_t)(q[4 * k + 2] & 255) << 16 | (uint32_t)q[4 * k + 3] << 24;
    *reinterpret_cast<Bytes<2, 1>*>(out) = raw;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) out[e] = (int8_t)q[e];
  }
}
// 127 / top (0: a row of zeros, or one that is not finite: codes 0), and how far from its code a value may lie for fp32 to decide (where 127 / top
// may overflow: nowhere)
NN_D float codes_per(const float top) { return top > 0.0f && top < INFINITY ? 127.0f / top : 0.0f; }
NN_D float codes_edge(const float top, const NormArgs& a) {
  return top > 0.0f && top < 1e-30f ? -1.0f : 0.5f - 2e-5f - (a.r ? 1.55e-5f : 0.0f) - (a.w ? 1.55e-5f : 0.0f);
}
// inv in fp32 as the forward pass has it (every wavefront computes a row's scale in one lane: 64-bit roots and quotients took as long as the codes)
NN_D float scale_of(const float top, const float ss, const NormArgs& a) {
  if (!a.w) return top / 127.0f;
  return (float)((double)top * (double)(1.0f / sqrtf(ss / (float)a.dim + a.eps)) * (1.0 / 127.0));
}

// PLAIN: neither weight nor residual
template <int DT, int TPR, int NV, int U, bool PLAIN>
__global__ __launch_bounds__(256) void rms_norm_quant_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  constexpr int GRP = 256 / TPR;
  __shared__ float ldss[16], ldso[16];
  __shared__ uint32_t ldsb[16];
  __shared__ unsigned long long ldsd[16];
  const int t = threadIdx.x % TPR;
  const T *x = (const T*)a.x, *r = PLAIN ? nullptr : (const T*)a.r, *w = PLAIN ? nullptr : (const T*)a.w;
  Raw8<DT> wr[NV];
  Eight<DT> in[U][NV];
  if (w) row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) { wr[i] = raw8_n<DT>(w + c, n); });
  take_rows<U>(a.rows, ((int64_t)blockIdx.x * GRP + threadIdx.x / TPR) * U, [&](const int64_t row, const int u) {
    row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
      in[u][i].load(x + row * a.ldx, r ? r + row * a.ldr : nullptr, nullptr, c, n);
      if (!PLAIN) in[u][i].w = wr[i];
    });
  }, [&](const int64_t first) {
    float v[U][NV][8], ss[U];
    uint32_t big[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ss[u] = 0.0f, big[u] = 0;
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
        in[u][i].sum(r != nullptr, v[u][i]);
        if (!PLAIN && a.h && first + u < a.rows) store8_n<DT>((T*)a.h + (first + u) * a.dim + c, n, v[u][i]);
        if (w) {
#pragma unroll
          for (int e = 0; e < 8; ++e) ss[u] = fmaf(v[u][i][e], v[u][i][e], ss[u]);
        }
        in[u][i].values(w != nullptr, v[u][i]);
        largest(v[u][i], big[u]);
      });
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float sum = w ? row_join<TPR>(ss[u], AddF{}, ldss) : 0.0f;
      const float top = __builtin_bit_cast(float, row_join<TPR>(big[u], MaxBits{}, ldsb)), per = codes_per(top);
      int q[NV][8];
      float off = 0.0f;
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t, const int) { codes8(v[u][i], per, q[i], off); });
      const float edge = codes_edge(top, a);
      double exact = top;
      if (r || w) {
        if (row_join<TPR>(off, MaxF{}, ldso) > edge) {  // (all threads of the row alike)
          unsigned long long b = 0;
          row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t, const int) {
            double d[8];
            in[u][i].exact(r != nullptr, w != nullptr, d);
            largest_exact(v[u][i], d, top, b);
          });
          exact = __longlong_as_double((long long)row_join<TPR>(b, MaxBits{}, ldsd));
        }
      }
      if (off > edge)
        row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t, const int) {
          in[u][i].decide(r != nullptr, w != nullptr, v[u][i], per, edge, exact, q[i]);
        });
      const int64_t row = first + u;
      if (row >= a.rows) continue;  // (U > 1: the threads of a row leave together, and no barrier follows)
      if (t == 0) a.scales[row] = scale_of(top, sum, a);
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) { store_codes(a.q + row * a.dim + c, n, q[i]); });
    }
  });
}
template <int DT>
__global__ __launch_bounds__(kWide) void rms_norm_quant_wide_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  __shared__ float ldss[16];
  __shared__ uint32_t ldsb[16];
  __shared__ unsigned long long ldsd[16];
  const bool has_r = a.r != nullptr, has_w = a.w != nullptr;
  const int64_t row = blockIdx.x;
  const T *x = (const T*)a.x + row * a.ldx, *r = has_r ? (const T*)a.r + row * a.ldr : nullptr, *w = (const T*)a.w;
  auto take = [&](const int64_t c, const int n, Eight<DT>& in, float (&h)[8], float (&v)[8]) {
    in.load(x, r, w, c, n);
    in.sum(has_r, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = h[e];
    in.values(has_w, v);
  };
  float ss = 0.0f;
  uint32_t big = 0;
  wide_loop(a.dim, [&](const int64_t c, const int n) {
    Eight<DT> in;
    float h[8], v[8];
    take(c, n, in, h, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(h[e], h[e], ss);
    largest(v, big);
    if (a.h) store8_n<DT>((T*)a.h + row * a.dim + c, n, h);
  });
  ss = row_join<kWide>(ss, AddF{}, ldss);
  const float top = __builtin_bit_cast(float, row_join<kWide>(big, MaxBits{}, ldsb)), per = codes_per(top);
  const float edge = codes_edge(top, a);
  double exact = top;
  if (has_r || has_w) {
    unsigned long long b = 0;
    wide_loop(a.dim, [&](const int64_t c, const int n) {
      Eight<DT> in;
      float h[8], v[8];
      double d[8];
      take(c, n, in, h, v);
      in.exact(has_r, has_w, d);
      largest_exact(v, d, top, b);
    });
    exact = __longlong_as_double((long long)row_join<kWide>(b, MaxBits{}, ldsd));
  }
  if (threadIdx.x == 0) a.scales[row] = scale_of(top, ss, a);
  wide_loop(a.dim, [&](const int64_t c, const int n) {
    Eight<DT> in;
    float h[8], v[8], off = 0.0f;
    int q[8];
    take(c, n, in, h, v);
    codes8(v, per, q, off);
    if (off > edge) in.decide(has_r, has_w, v, per, edge, exact, q);
    store_codes(a.q + row * a.dim + c, n, q);
  });
}

// ---- backward.  The workgroups walk the rows and keep their threads' columns of dw in registers; their partial sums are added in a fixed order by the
// second kernel, so the result does not depend on which finished first.
template <int DT, int TPR, int NV, int U, bool DW>
__global__ __launch_bounds__(256) void rms_norm_bwd_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  constexpr int GRP = 256 / TPR;
  __shared__ float lds[16];
  __shared__ float ldw[DW && GRP > 1 ? 256 * 8 : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const T *x = (const T*)a.x, *r = (const T*)a.r, *w = (const T*)a.w, *dy = (const T*)a.dy, *dh = (const T*)a.dh;
  Raw8<DT> wr[NV], xr[U][NV], rr[U][NV], yr[U][NV], hr[U][NV];
  float inv[U], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) fill8(dw[i], 0.0f);
  row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) { wr[i] = raw8_n<DT>(w + c, n); });
  for (int64_t at = ((int64_t)blockIdx.x * GRP + sub) * U; at < a.rows; at += (int64_t)gridDim.x * GRP * U)
    take_rows<U>(a.rows, at, [&](const int64_t row, const int u) {
      inv[u] = a.inv[row];
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
        xr[u][i] = raw8_n<DT>(x + row * a.ldx + c, n);
        if (r) rr[u][i] = raw8_n<DT>(r + row * a.ldr + c, n);
        if (dy) yr[u][i] = raw8_n<DT>(dy + row * a.lddy + c, n);
        if (dh) hr[u][i] = raw8_n<DT>(dh + row * a.lddh + c, n);
      });
    }, [&](const int64_t first) {
      float nn[U][NV][8], g[U][NV][8], un[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        un[u] = 0.0f;
        const bool there = first + u < a.rows;
        row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t, const int) {
          float b[8], k[8];
          widen8<DT>(xr[u][i], nn[u][i]);
          if (r) {
            widen8<DT>(rr[u][i], b);
#pragma unroll
            for (int e = 0; e < 8; ++e) nn[u][i][e] += b[e];
          }
          if (dy) widen8<DT>(yr[u][i], g[u][i]);
          else fill8(g[u][i], 0.0f);
          widen8<DT>(wr[i], k);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            nn[u][i][e] *= inv[u];
            if constexpr (DW) dw[i][e] = fmaf(there ? g[u][i][e] : 0.0f, nn[u][i][e], dw[i][e]);
            g[u][i][e] *= k[e];
            un[u] = fmaf(g[u][i][e], nn[u][i][e], un[u]);
          }
        });
      }
      if (!a.dx) return;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float mean = row_join<TPR>(un[u], AddF{}, lds) / (float)a.dim;
        const int64_t row = first + u;
        if (row >= a.rows) continue;  // (U > 1: the threads of a row leave together, and no barrier follows)
        row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
          float d[8];
          if (dh) widen8<DT>(hr[u][i], d);
          else fill8(d, 0.0f);
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = fmaf(inv[u], g[u][i][e] - nn[u][i][e] * mean, d[e]);
          store8_n<DT>((T*)a.dx + row * a.dim + c, n, d);
        });
      }
    });
  if constexpr (DW) {
    float* out = a.partial + (int64_t)blockIdx.x * a.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = ((int64_t)i * TPR + t) * 8;
      if constexpr (GRP > 1) {  // the workgroup's rows first (every thread takes part: the loop bounds are uniform)
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) ldw[(sub * 8 + e) * TPR + t] = dw[i][e];
        __syncthreads();
        if (sub == 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < GRP; ++k) s += ldw[(k * 8 + e) * TPR + t];
            if (c + e < a.dim) out[c + e] = s;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < a.dim) out[c + e] = dw[i][e];
      }
    }
  }
}
template <int DT>
__global__ __launch_bounds__(kWide) void rms_norm_bwd_wide_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  __shared__ float lds[16];
  const int64_t row = blockIdx.x;
  const T *x = (const T*)a.x + row * a.ldx, *r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  const float inv = a.inv[row];
  auto load = [&](const int64_t c, const int n, float (&nn)[8], float (&u)[8]) {
    float k[8];
    load_h<DT>(x, r, c, n, nn);
    if (a.dy) load8_n<DT>((const T*)a.dy + row * a.lddy + c, n, u);
    else fill8(u, 0.0f);
    load8_n<DT>((const T*)a.w + c, n, k);
#pragma unroll
    for (int e = 0; e < 8; ++e) nn[e] *= inv, u[e] *= k[e];
  };
  float un = 0.0f;
  wide_loop(a.dim, [&](const int64_t c, const int n) {
    float nn[8], u[8];
    load(c, n, nn, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) un = fmaf(u[e], nn[e], un);
  });
  const float mean = row_join<kWide>(un, AddF{}, lds) / (float)a.dim;
  wide_loop(a.dim, [&](const int64_t c, const int n) {
    float nn[8], u[8], d[8];
    load(c, n, nn, u);
    if (a.dh) load8_n<DT>((const T*)a.dh + row * a.lddh + c, n, d);
    else fill8(d, 0.0f);
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = fmaf(inv, u[e] - nn[e] * mean, d[e]);
    store8_n<DT>((T*)a.dx + row * a.dim + c, n, d);
  });
}

// rows too wide for the registers of a workgroup: dw by columns.  One thread a column, the rows split over blockIdx.y
template <int DT>
__global__ __launch_bounds__(256) void rms_norm_dw_wide_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.dim) return;
  float s = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float h = (float)((const T*)a.x)[row * a.ldx + c];
    if (a.r) h += (float)((const T*)a.r)[row * a.ldr + c];
    s = fmaf(a.dy ? (float)((const T*)a.dy)[row * a.lddy + c] : 0.0f, h * a.inv[row], s);
  }
  a.partial[(int64_t)blockIdx.y * a.dim + c] = s;
}

// dweight[c] = sum over the parts, 32 columns a workgroup, 32 threads a column: each takes every 32nd part, eight at a time, then a fixed order
template <int DT>
__global__ __launch_bounds__(1024) void rms_norm_dw_reduce_kernel(const float* __restrict__ partial, const int parts, const int64_t dim,
                                                                 elem_t<DT>* __restrict__ dw) {
  __shared__ float lds[32][33];
  const int col = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + col;
  float s = 0.0f;
  if (c < dim) {
    int p = g;
    for (; p + 7 * 32 < parts; p += 8 * 32) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = partial[(int64_t)(p + k * 32) * dim + c];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    for (; p < parts; p += 32) s += partial[(int64_t)p * dim + c];
  }
  lds[g][col] = s;
  __syncthreads();
  if (g == 0 && c < dim) {
    float tot = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) tot += lds[i][col];
    dw[c] = (elem_t<DT>)tot;
  }
}
