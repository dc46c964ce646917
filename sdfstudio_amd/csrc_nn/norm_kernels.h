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
// Eight to 64 lanes a row up to 2048 elements (no barrier: a shuffle tree joins the sums), U rows of narrow ones at a time so that enough loads
// are under way; a workgroup of 256 or 1024 threads a row above; a row beyond 16384 elements is read a second time (NV = 0: it comes
// back from L2).  Workgroups walk the rows and keep the weight in registers.
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
  for (int d = (TPR < 64 ? TPR : 64) / 2; d >= 1; d >>= 1) v = op(v, __shfl_xor(v, d, 64));
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
struct MaxBits { template <class T> NN_D T operator()(T a, T b) const { return a > b ? a : b; } };

// f(group index i, first column c, valid elements n) over a thread's groups of 8 columns
template <int TPR, int NV, class F>
NN_D void row_loop(const int64_t dim, const int t, F&& f) {
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * 8;
      if (c < dim) f(i, (int64_t)c, (int)(dim - c < 8 ? dim - c : 8));
    }
  } else {
    for (int64_t c = (int64_t)t * 8; c < dim; c += TPR * 8) f(0, c, (int)(dim - c < 8 ? dim - c : 8));
  }
}
NN_D void fill8(float (&v)[8], const float x) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x;
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
constexpr int some(const int nv) { return nv > 0 ? nv : 1; }

// ---- forward.  TPR threads a row, GRP rows of them a workgroup, U such rows at a time
template <int DT, int TPR, int NV, int U>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_norm_fwd_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  constexpr int GRP = TPR > 256 ? 1 : 256 / TPR, N = some(NV);
  __shared__ float lds[16];
  const int t = threadIdx.x % TPR;
  const T* w = (const T*)a.w;
  float wv[N][8];
  if constexpr (NV > 0) row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) { load8_n<DT>(w + c, n, wv[i]); });
  for (int64_t first = ((int64_t)blockIdx.x * GRP + threadIdx.x / TPR) * U; first < a.rows; first += (int64_t)gridDim.x * GRP * U) {
    float h[U][N][8], ss[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ss[u] = 0.0f;
      const int64_t row = first + u < a.rows ? first + u : a.rows - 1;
      const T* x = (const T*)a.x + row * a.ldx;
      const T* r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
        load_h<DT>(x, r, c, n, h[u][i]);
        if constexpr (NV == 0) {
          if (a.h) store8_n<DT>((T*)a.h + row * a.dim + c, n, h[u][0]);
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
        if constexpr (NV == 0) {
          load8_n<DT>(w + c, n, wv[0]);
          load_h<DT>((const T*)a.x + row * a.ldx, a.r ? (const T*)a.r + row * a.ldr : nullptr, c, n, h[u][0]);
        } else if (a.h) store8_n<DT>((T*)a.h + row * a.dim + c, n, h[u][i]);
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = h[u][i][e] * inv * wv[i][e];
        store8_n<DT>((T*)a.y + row * a.dim + c, n, o);
      });
    }
  }
}

// ---- 8-bit output.  The code of v is round(127 v / top) with v = (x + r) w and top = max|v| exact: in fp32 the quotient is off by at most five
// half steps of 127 (4e-5), so only a value within 5e-5 of the border between two codes - one in ten thousand - is computed again
// in 64 bits, and so is the largest magnitude, from the few values next to the largest in fp32.  (All of it in 64 bits: 168 us instead
// of 110 for 16384 x 4096 fp16 with a residual.)  Ties exist (half the largest value is one) and their rounding to even must not hang on the last
// bit of a reciprocal: there the quotient of exact numbers decides.
NN_D int code_of(const double v, const double top) {
  double c = __builtin_rint(v * 127.0 / top);
  c = c > 127.0 ? 127.0 : c;
  c = c < -127.0 ? -127.0 : c;
  return c == c ? (int)c : 0;
}

template <int DT, int TPR, int NV, int U>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_norm_quant_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  constexpr int GRP = TPR > 256 ? 1 : 256 / TPR, N = some(NV);
  __shared__ float ldss[16];
  __shared__ uint32_t ldsb[16];
  __shared__ unsigned long long ldsd[16];
  const int t = threadIdx.x % TPR;
  const T* w = (const T*)a.w;
  float wv[N][8];
  auto load_w = [&](const int i, const int64_t c, const int n) {
    if (w) load8_n<DT>(w + c, n, wv[i]);
    else fill8(wv[i], 1.0f);
  };
  if constexpr (NV > 0) row_loop<TPR, NV>(a.dim, t, load_w);
  for (int64_t first = ((int64_t)blockIdx.x * GRP + threadIdx.x / TPR) * U; first < a.rows; first += (int64_t)gridDim.x * GRP * U) {
    float xs[U][N][8], rs[U][N][8], ss[U];
    uint32_t big[U];
    auto load = [&](const int u, const int64_t row, const int i, const int64_t c, const int n) {
      load8_n<DT>((const T*)a.x + row * a.ldx + c, n, xs[u][i]);
      if (a.r) load8_n<DT>((const T*)a.r + row * a.ldr + c, n, rs[u][i]);
      else fill8(rs[u][i], 0.0f);
      if constexpr (NV == 0) load_w(i, c, n);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ss[u] = 0.0f, big[u] = 0;
      const int64_t row = first + u < a.rows ? first + u : a.rows - 1;
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
        load(u, row, i, c, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float h = xs[u][i][e] + rs[u][i][e];
          ss[u] = fmaf(h, h, ss[u]);
          const uint32_t b = __builtin_bit_cast(uint32_t, h * wv[i][e]) & 0x7fffffffu;
          big[u] = b > big[u] ? b : big[u];
        }
      });
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = first + u < a.rows ? first + u : a.rows - 1;
      const float sum = w ? row_join<TPR>(ss[u], AddF{}, ldss) : 0.0f;
      const float topf = __builtin_bit_cast(float, row_join<TPR>(big[u], MaxBits{}, ldsb));
      // the largest magnitude exactly: fp32 values are off by two half steps (2^-23), so it is among those from here on (a NaN passes on)
      const float near = topf * (1.0f - 0x1p-21f);
      unsigned long long tb = 0;
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
        if constexpr (NV == 0) load(u, row, i, c, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (fabsf((xs[u][i][e] + rs[u][i][e]) * wv[i][e]) < near) continue;
          const double v = ((double)xs[u][i][e] + (double)rs[u][i][e]) * (double)wv[i][e];
          const unsigned long long b = (unsigned long long)__double_as_longlong(v) & 0x7fffffffffffffffull;
          tb = b > tb ? b : tb;
        }
      });
      const double top = __longlong_as_double((long long)row_join<TPR>(tb, MaxBits{}, ldsd));
      if (first + u >= a.rows) continue;  // (U > 1: the threads of a row leave together, and no barrier follows)
      if (t == 0) a.scales[row] = (float)(top / 127.0 * (w ? 1.0 / sqrt((double)sum / (double)a.dim + (double)a.eps) : 1.0));
      const float per = topf > 0.0f && topf < INFINITY ? 127.0f / topf : 0.0f;  // (a row of zeros, or one that is not finite: codes 0)
      const float edge = topf > 0.0f && topf < 1e-30f ? -1.0f : 0.49995f;      // (where 127 / topf may overflow: all in 64 bits)
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
        if constexpr (NV == 0) load(u, row, i, c, n);
        float h[8], off = 0.0f;
        int q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          h[e] = xs[u][i][e] + rs[u][i][e];
          const float k = h[e] * wv[i][e] * per, z = __builtin_rintf(k);
          off = fmaxf(off, fabsf(k - z));
          q[e] = (int)z;
        }
        if (off > edge) {
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] = code_of(((double)xs[u][i][e] + (double)rs[u][i][e]) * (double)wv[i][e], top);
        }
        if (a.h) store8_n<DT>((T*)a.h + row * a.dim + c, n, h);
        int8_t* out = a.q + row * a.dim + c;
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
      });
    }
  }
}

// ---- backward.  The workgroups walk the rows and keep their threads' columns of dw in registers; their partial sums are added in a fixed order by the
// second kernel, so the result does not depend on which finished first.
template <int DT, int TPR, int NV, int U, bool DW>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_norm_bwd_kernel(const NormArgs a) {
  typedef elem_t<DT> T;
  constexpr int GRP = TPR > 256 ? 1 : 256 / TPR, N = some(NV);
  __shared__ float lds[16];
  __shared__ float ldw[DW && GRP > 1 ? 256 * 8 : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const T* w = (const T*)a.w;
  float dw[N][8], wv[N][8];
#pragma unroll
  for (int i = 0; i < N; ++i) fill8(dw[i], 0.0f);
  if constexpr (NV > 0) row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) { load8_n<DT>(w + c, n, wv[i]); });
  for (int64_t first = ((int64_t)blockIdx.x * GRP + sub) * U; first < a.rows; first += (int64_t)gridDim.x * GRP * U) {
    float nn[U][N][8], g[U][N][8], un[U];
    auto load = [&](const int u, const int64_t row, const int i, const int64_t c, const int n) {
      load_h<DT>((const T*)a.x + row * a.ldx, a.r ? (const T*)a.r + row * a.ldr : nullptr, c, n, nn[u][i]);
      if (a.dy) load8_n<DT>((const T*)a.dy + row * a.lddy + c, n, g[u][i]);
      else fill8(g[u][i], 0.0f);
      if constexpr (NV == 0) load8_n<DT>(w + c, n, wv[0]);
      const float inv = a.inv[row];
#pragma unroll
      for (int e = 0; e < 8; ++e) nn[u][i][e] *= inv;
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      un[u] = 0.0f;
      const bool there = first + u < a.rows;
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
        load(u, there ? first + u : a.rows - 1, i, c, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (DW && NV > 0) dw[i][e] = fmaf(there ? g[u][i][e] : 0.0f, nn[u][i][e], dw[i][e]);
          un[u] = fmaf(g[u][i][e] * wv[i][e], nn[u][i][e], un[u]);
        }
      });
    }
    if (!a.dx) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float mean = row_join<TPR>(un[u], AddF{}, lds) / (float)a.dim;
      const int64_t row = first + u;
      if (row >= a.rows) continue;  // (U > 1: the threads of a row leave together, and no barrier follows)
      const float inv = a.inv[row];
      row_loop<TPR, NV>(a.dim, t, [&](const int i, const int64_t c, const int n) {
        if constexpr (NV == 0) load(u, row, i, c, n);
        float d[8];
        if (a.dh) load8_n<DT>((const T*)a.dh + row * a.lddh + c, n, d);
        else fill8(d, 0.0f);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = fmaf(inv, g[u][i][e] * wv[i][e] - nn[u][i][e] * mean, d[e]);
        store8_n<DT>((T*)a.dx + row * a.dim + c, n, d);
      });
    }
  }
  if constexpr (DW && NV > 0) {
    float* out = a.partial + (int64_t)blockIdx.x * a.dim;
#pragma unroll
    for (int i = 0; i < N; ++i) {
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
