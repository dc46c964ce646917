// sdfnn — root-mean-square norm with the residual's addition: forward, 8-bit output, backward.
//
//   h = x + r     inv = (mean(h^2) + eps)^(-1/2)     y = h inv w
//   q = round(127 v / max|v|),  v = h w,  scale = inv max|v| / 127        (inv > 0 divides out of the codes)
//   u = dy w,  n = h inv:   dx = dr = inv (u - n mean(u n)) + dh,   dw = sum over rows of dy n
//
// All three are bound by HBM: every tensor is read or written once.  A row stays in the registers of its threads between the two passes
// that the statistic needs (NV groups of 8 elements a thread); the backward forms h from x and r again instead of reading a stored h,
// because the stored one is rounded to the type.
//
// One wavefront a row up to 2048 elements (four rows a workgroup: no barrier, a shuffle tree joins the sums), one workgroup of 256 or 1024
// threads a row above; a row beyond 32768 elements is read a second time (NV = 0: it comes back from L2).
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
template <int TPR, class T, class OP>
NN_D T row_join(T v, OP op, T* lds) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = op(v, __shfl_xor(v, d, 64));
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
// largest |v| by its bits: as unsigned integers inf lies above every finite value and NaN above inf, so a NaN in a row survives the join
struct MaxBits { NN_D unsigned long long operator()(unsigned long long a, unsigned long long b) const { return a > b ? a : b; } };

template <int DT, int TPR, int NV>
struct RowLoop {
  // f(group index i, first column c, valid elements n) over this thread's groups
  template <class F>
  static NN_D void run(const int64_t dim, const int t, F&& f) {
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t c = ((int64_t)i * TPR + t) * 8;
        if (c < dim) f(i, c, (int)(dim - c < 8 ? dim - c : 8));
      }
    } else {
      for (int64_t c = (int64_t)t * 8; c < dim; c += TPR * 8) f(0, c, (int)(dim - c < 8 ? dim - c : 8));
    }
  }
};

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

// ---- forward.  TPR threads a row, RPB rows a workgroup
template <int DT, int TPR, int NV, int RPB>
__global__ __launch_bounds__(TPR * RPB) void rms_norm_fwd_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  __shared__ float lds[16];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;  // RPB > 1: a whole wavefront, which meets no barrier; RPB == 1: never
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  const T* w = (const T*)a.w;
  T* y = (T*)a.y + row * a.dim;
  T* ho = a.h ? (T*)a.h + row * a.dim : nullptr;
  float h[NV > 0 ? NV : 1][8];
  float ss = 0.0f;
  RowLoop<DT, TPR, NV>::run(a.dim, t, [&](const int i, const int64_t c, const int n) {
    load_h<DT>(x, r, c, n, h[i]);
    if (ho) store8_n<DT>(ho + c, n, h[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(h[i][e], h[i][e], ss);
  });
  ss = row_join<TPR>(ss, AddF{}, lds);
  const float inv = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  if (t == 0 && a.inv) a.inv[row] = inv;
  RowLoop<DT, TPR, NV>::run(a.dim, t, [&](const int i, const int64_t c, const int n) {
    float wv[8];
    load8_n<DT>(w + c, n, wv);
    if constexpr (NV == 0) load_h<DT>(x, r, c, n, h[0]);
#pragma unroll
    for (int e = 0; e < 8; ++e) wv[e] *= h[i][e] * inv;
    store8_n<DT>(y + c, n, wv);
  });
}

// ---- 8-bit output.  v and its largest magnitude are held in 64 bits: x + r and the product with w then lose nothing that could move a
// value across the border between two codes, and gfx950 adds and multiplies doubles at the rate of single floats, which HBM hides
// (16384 x 4096 fp16 with a residual: DESIGN.md has the figures).
NN_D int code_of(const double v, const double top, const double per) {
  double c = v * per;
  // Ties exist (half the largest value is one) and their rounding to even must not hang on the last bit of a reciprocal: next to a border
  // the quotient itself decides, which is exact where it is a tie.
  if (__builtin_fabs(c - __builtin_floor(c) - 0.5) < 1e-9) c = v * 127.0 / top;
  c = __builtin_rint(c);
  c = c > 127.0 ? 127.0 : c;
  c = c < -127.0 ? -127.0 : c;
  return c == c ? (int)c : 0;
}

template <int DT, int TPR, int NV, int RPB>
__global__ __launch_bounds__(TPR * RPB) void rms_norm_quant_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  __shared__ float lds[16];
  __shared__ unsigned long long ldsm[16];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  const T* w = (const T*)a.w;
  T* ho = a.h ? (T*)a.h + row * a.dim : nullptr;
  int8_t* q = a.q + row * a.dim;
  float xs[NV > 0 ? NV : 1][8], rs[NV > 0 ? NV : 1][8];
  float ss = 0.0f;
  unsigned long long top = 0;
  auto value = [&](const int i, const int e, const float wv) {
    return ((double)xs[i][e] + (double)rs[i][e]) * (double)wv;
  };
  RowLoop<DT, TPR, NV>::run(a.dim, t, [&](const int i, const int64_t c, const int n) {
    load8_n<DT>(x + c, n, xs[i]);
    if (r) load8_n<DT>(r + c, n, rs[i]);
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) rs[i][e] = 0.0f;
    }
    float wv[8], h[8];
    if (w) load8_n<DT>(w + c, n, wv);
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) wv[e] = 1.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[e] = xs[i][e] + rs[i][e];
      ss = fmaf(h[e], h[e], ss);
      const unsigned long long b = (unsigned long long)__double_as_longlong(value(i, e, wv[e])) & 0x7fffffffffffffffull;
      top = b > top ? b : top;
    }
    if (ho) store8_n<DT>(ho + c, n, h);
  });
  if (w) ss = row_join<TPR>(ss, AddF{}, lds);
  top = row_join<TPR>(top, MaxBits{}, ldsm);
  const double largest = __longlong_as_double((long long)top);
  const double per = largest > 0.0 ? 127.0 / largest : 0.0;  // (a row of zeros, or one with a NaN: codes 0)
  const float inv = w ? 1.0f / sqrtf(ss / (float)a.dim + a.eps) : 1.0f;
  if (t == 0) a.scales[row] = (float)(largest / 127.0 * (double)inv);
  RowLoop<DT, TPR, NV>::run(a.dim, t, [&](const int i, const int64_t c, const int n) {
    if constexpr (NV == 0) {
      load8_n<DT>(x + c, n, xs[0]);
      if (r) load8_n<DT>(r + c, n, rs[0]);
    }
    float wv[8];
    if (w) load8_n<DT>(w + c, n, wv);
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) wv[e] = 1.0f;
    }
    int8_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = (int8_t)code_of(value(i, e, wv[e]), largest, per);
    if (n >= 8) {
      Bytes<2, 1> raw;
      __builtin_memcpy(&raw, b, 8);
      *reinterpret_cast<Bytes<2, 1>*>(q + c) = raw;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) q[c + e] = b[e];
    }
  });
}

// ---- backward.  A workgroup walks rows blockIdx.x, + gridDim.x, ... and keeps its threads' columns of dw in registers; the partial sums
// of the workgroups are added in a fixed order by the second kernel, so the result does not depend on which finished first.
template <int DT, int TPR, int NV, int RPB, bool DW>
__global__ __launch_bounds__(TPR * RPB) void rms_norm_bwd_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  constexpr int N = NV > 0 ? NV : 1;
  __shared__ float lds[16];
  __shared__ float ldw[RPB > 1 ? RPB * TPR * 8 : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const T* w = (const T*)a.w;
  float dw[N][8];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.0f;
  for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < a.rows; row += (int64_t)gridDim.x * RPB) {
    const T* x = (const T*)a.x + row * a.ldx;
    const T* r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
    const T* dy = a.dy ? (const T*)a.dy + row * a.lddy : nullptr;
    const T* dh = a.dh ? (const T*)a.dh + row * a.lddh : nullptr;
    T* dx = a.dx ? (T*)a.dx + row * a.dim : nullptr;
    const float inv = a.inv[row];
    float nn[N][8], u[N][8];
    float un = 0.0f;
    RowLoop<DT, TPR, NV>::run(a.dim, t, [&](const int i, const int64_t c, const int n) {
      float g[8], wv[8];
      load_h<DT>(x, r, c, n, nn[i]);
      load8_n<DT>(w + c, n, wv);
      if (dy) load8_n<DT>(dy + c, n, g);
      else {
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        nn[i][e] *= inv;
        u[i][e] = g[e] * wv[e];
        un = fmaf(u[i][e], nn[i][e], un);
        if constexpr (DW && NV > 0) dw[i][e] = fmaf(g[e], nn[i][e], dw[i][e]);
      }
    });
    un = row_join<TPR>(un, AddF{}, lds) / (float)a.dim;
    if (dx) {
      RowLoop<DT, TPR, NV>::run(a.dim, t, [&](const int i, const int64_t c, const int n) {
        if constexpr (NV == 0) {
          float wv[8];
          load_h<DT>(x, r, c, n, nn[0]);
          load8_n<DT>(w + c, n, wv);
#pragma unroll
          for (int e = 0; e < 8; ++e) u[0][e] = 0.0f;
          if (dy) load8_n<DT>(dy + c, n, u[0]);
#pragma unroll
          for (int e = 0; e < 8; ++e) nn[0][e] *= inv, u[0][e] *= wv[e];
        }
        float d[8], o[8];
        if (dh) load8_n<DT>(dh + c, n, d);
        else {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = fmaf(inv, u[i][e] - nn[i][e] * un, d[e]);
        store8_n<DT>(dx + c, n, o);
      });
    }
  }
  if constexpr (DW && NV > 0) {
    float* out = a.partial + (int64_t)blockIdx.x * a.dim;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t c = ((int64_t)i * TPR + t) * 8;
      if constexpr (RPB > 1) {  // the workgroup's rows first (every thread takes part: the loop bounds are uniform)
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) ldw[(sub * 8 + e) * TPR + t] = dw[i][e];
        __syncthreads();
        if (sub == 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < RPB; ++k) s += ldw[(k * 8 + e) * TPR + t];
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

// dweight[c] = sum over the parts, 64 columns a workgroup, 16 threads a column: each takes every 16th part, then a fixed order
template <int DT>
__global__ __launch_bounds__(1024) void rms_norm_dw_reduce_kernel(const float* __restrict__ partial, const int parts, const int64_t dim,
                                                                 elem_t<DT>* __restrict__ dw) {
  __shared__ float lds[16][64];
  const int col = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + col;
  float s = 0.0f;
  if (c < dim)
    for (int p = g; p < parts; p += 16) s += partial[(int64_t)p * dim + c];
  lds[g][col] = s;
  __syncthreads();
  if (g == 0 && c < dim) {
    float tot = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) tot += lds[i][col];
    dw[c] = (elem_t<DT>)tot;
  }
}
