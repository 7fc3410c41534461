// Layer norm over the last dimension, forward and backward:
//   xh = (x - mean) rstd   y = xh w + b   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   g = dy w   dx = rstd (g - mean(g) - xh mean(g xh))   dw = sum_rows dy xh   db = sum_rows dy
// All sums in binary32 in a fixed order, one rounding of each result.
//
// Bound by memory.  A row lies in the registers of one wave, of a workgroup of 4 or of one of 16
// (up to 32 columns a thread), so that x is read once for the mean, the squares and the result; wider
// rows are read again.  The backward's workgroups walk over rows with the columns of dw and db in
// registers, and leave one partial sum each, which a second kernel adds.
#include "otx_common.h"

namespace otx {

namespace {

constexpr int kCols = 32;  // columns a thread holds

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float* f) {
  if constexpr (V == 1) {
    f[0] = Elem<T>::ld(p);
  } else {
    const uint4 w = *(const uint4*)p;
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = Elem<T>::get(w, i);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float* f) {
  struct {
    T e[V];
  } v;
#pragma unroll
  for (int i = 0; i < V; i++) v.e[i] = Elem<T>::put(f[i]);
  if constexpr (V == 1)
    *p = v.e[0];
  else
    *(uint4*)p = __builtin_bit_cast(uint4, v);
}

// The sum of N values over the threads of a row (WR waves), the same in every thread.
template <int N, int WR>
__device__ __forceinline__ void row_sum(float (&v)[N], float* lds) {
#pragma unroll
  for (int m = 32; m; m >>= 1)
#pragma unroll
    for (int i = 0; i < N; i++) v[i] += __shfl_xor(v[i], m);
  if constexpr (WR > 1) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    __syncthreads();  // the last sums have been read
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < N; i++) lds[i * WR + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
      v[i] = lds[i * WR];
#pragma unroll
      for (int k = 1; k < WR; k++) v[i] += lds[i * WR + k];
    }
  }
}

template <typename T, int V, int WR>  // WR waves to a row
__global__ void __launch_bounds__(WR == 1 ? 256 : WR * 64)
    layer_norm_fwd_kernel(const T* x, const T* w, const T* b, T* y, float* mean, float* rstd, long rows, int D,
                          float eps) {
  constexpr int NT = WR * 64, RPB = WR == 1 ? 4 : 1, NC = kCols / V;
  __shared__ float lds[WR];
  const int tid = WR == 1 ? threadIdx.x & 63 : threadIdx.x, steps = (D + NT * V - 1) / (NT * V);
  const float inv = 1.0f / (float)D;
  for (long r = (long)blockIdx.x * RPB + (WR == 1 ? threadIdx.x >> 6 : 0); r < rows; r += (long)gridDim.x * RPB) {
    const T* xr = x + r * D;
    T* yr = y + r * D;
    float v[kCols], sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const int c = (i * NT + tid) * V;
      if (c < D) {
        load<T, V>(xr + c, v + i * V);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) v[i * V + e] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < kCols; i++) sum[0] += v[i];
    for (int i = NC; i < steps; i++) {
      const int c = (i * NT + tid) * V;
      float f[V];
      if (c < D) {
        load<T, V>(xr + c, f);
#pragma unroll
        for (int e = 0; e < V; e++) sum[0] += f[e];
      }
    }
    row_sum<1, WR>(sum, lds);
    const float mu = sum[0] * inv;
    sum[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; i++)
      if ((i * NT + tid) * V < D)
#pragma unroll
        for (int e = 0; e < V; e++) sum[0] = __builtin_fmaf(v[i * V + e] - mu, v[i * V + e] - mu, sum[0]);
    for (int i = NC; i < steps; i++) {
      const int c = (i * NT + tid) * V;
      float f[V];
      if (c < D) {
        load<T, V>(xr + c, f);
#pragma unroll
        for (int e = 0; e < V; e++) sum[0] = __builtin_fmaf(f[e] - mu, f[e] - mu, sum[0]);
      }
    }
    row_sum<1, WR>(sum, lds);
    const float rs = 1.0f / __builtin_sqrtf(__builtin_fmaf(sum[0], inv, eps));
    if (tid == 0) mean[r] = mu, rstd[r] = rs;
    auto write = [&](int c, const float* f) {
      float g[V], wf[V], bf[V];
      load<T, V>(w + c, wf);
      if (b) load<T, V>(b + c, bf);
#pragma unroll
      for (int e = 0; e < V; e++) g[e] = __builtin_fmaf((f[e] - mu) * rs, wf[e], b ? bf[e] : 0.0f);
      store<T, V>(yr + c, g);
    };
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const int c = (i * NT + tid) * V;
      if (c < D) write(c, v + i * V);
    }
    for (int i = NC; i < steps; i++) {
      const int c = (i * NT + tid) * V;
      float f[V];
      if (c < D) {
        load<T, V>(xr + c, f);
        write(c, f);
      }
    }
  }
}

// dx, and the workgroup's partial dw and db: part[0 .. G)[D], part[G .. 2 G)[D].  `held`: the row fits
// the registers; otherwise dx alone (layer_norm_cols_kernel forms the column sums).
template <typename T, int V, int WR>
__global__ void __launch_bounds__(WR == 1 ? 256 : WR * 64)
    layer_norm_bwd_kernel(const T* x, const T* w, const float* mean, const float* rstd, const T* dy, T* dx, float* part,
                          long rows, int D) {
  constexpr int NT = WR * 64, RPB = WR == 1 ? 4 : 1, NC = kCols / V;
  __shared__ float lds[WR == 1 ? 2 * 64 * kCols : 2 * WR];
  const int tid = WR == 1 ? threadIdx.x & 63 : threadIdx.x, wave = threadIdx.x >> 6;
  const float inv = 1.0f / (float)D;
  float wf[kCols], dw[kCols], db[kCols];
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const int c = (i * NT + tid) * V;
    if (c < D) {
      load<T, V>(w + c, wf + i * V);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++) wf[i * V + e] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kCols; i++) dw[i] = db[i] = 0.0f;
  for (long r = (long)blockIdx.x * RPB + (WR == 1 ? wave : 0); r < rows; r += (long)gridDim.x * RPB) {
    const float mu = mean[r], rs = rstd[r];
    float xh[kCols], g[kCols], sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const int c = (i * NT + tid) * V;
      if (c < D) {
        load<T, V>(x + r * D + c, xh + i * V);
        load<T, V>(dy + r * D + c, g + i * V);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) xh[i * V + e] = mu, g[i * V + e] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < kCols; i++) {
      xh[i] = (xh[i] - mu) * rs;
      dw[i] = __builtin_fmaf(g[i], xh[i], dw[i]);
      db[i] += g[i];
      g[i] *= wf[i];
      sum[0] += g[i];
      sum[1] = __builtin_fmaf(g[i], xh[i], sum[1]);
    }
    row_sum<2, WR>(sum, lds);
    const float m1 = sum[0] * inv, m2 = sum[1] * inv;
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const int c = (i * NT + tid) * V;
      if (c < D) {
        float f[V];
#pragma unroll
        for (int e = 0; e < V; e++) f[e] = rs * (g[i * V + e] - m1 - xh[i * V + e] * m2);
        store<T, V>(dx + r * D + c, f);
      }
    }
  }
  if constexpr (WR == 1) {  // the four waves' sums, in order
    for (int k = 1; k < 4; k++) {
      __syncthreads();
      if (wave == k)
#pragma unroll
        for (int i = 0; i < kCols; i++) lds[i * 64 + tid] = dw[i], lds[(kCols + i) * 64 + tid] = db[i];
      __syncthreads();
      if (wave == 0)
#pragma unroll
        for (int i = 0; i < kCols; i++) dw[i] += lds[i * 64 + tid], db[i] += lds[(kCols + i) * 64 + tid];
    }
    if (wave) return;
  }
  float* p = part + (long)blockIdx.x * D;
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const int c = (i * NT + tid) * V;
    if (c < D)
#pragma unroll
      for (int e = 0; e < V; e++) p[c + e] = dw[i * V + e], p[(long)gridDim.x * D + c + e] = db[i * V + e];
  }
}

// Rows wider than the registers of a workgroup: dx from two readings.
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_dx_wide_kernel(const T* x, const T* w, const float* mean,
                                                                  const float* rstd, const T* dy, T* dx, long rows,
                                                                  int D) {
  __shared__ float lds[32];
  const float inv = 1.0f / (float)D;
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mu = mean[r], rs = rstd[r];
    float sum[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < D; c += 1024) {
      const float g = Elem<T>::ld(dy + r * D + c) * Elem<T>::ld(w + c);
      sum[0] += g;
      sum[1] = __builtin_fmaf(g, (Elem<T>::ld(x + r * D + c) - mu) * rs, sum[1]);
    }
    row_sum<2, 16>(sum, lds);
    const float m1 = sum[0] * inv, m2 = sum[1] * inv;
    for (int c = threadIdx.x; c < D; c += 1024) {
      const float g = Elem<T>::ld(dy + r * D + c) * Elem<T>::ld(w + c);
      dx[r * D + c] = Elem<T>::put(rs * (g - m1 - (Elem<T>::ld(x + r * D + c) - mu) * rs * m2));
    }
  }
}

// Their column sums: a thread walks one column over the rows of its part of the grid.
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_cols_kernel(const T* x, const float* mean, const float* rstd,
                                                              const T* dy, float* part, long rows, int D) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= D) return;
  float dw = 0.0f, db = 0.0f;
  for (long r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = Elem<T>::ld(dy + r * D + c);
    dw = __builtin_fmaf(g, (Elem<T>::ld(x + r * D + c) - mean[r]) * rstd[r], dw);
    db += g;
  }
  part[(long)blockIdx.y * D + c] = dw;
  part[((long)gridDim.y + blockIdx.y) * D + c] = db;
}

// The sum of G partial rows: a workgroup takes 64 columns, each wave every 16th row.
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_join_kernel(const float* part, T* dw, T* db, int G, int D) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  const float* p = part + (blockIdx.y ? (long)G * D : 0);
  float sum = 0.0f;
  if (c < D)
    for (int g = wave; g < G; g += 16) sum += p[(long)g * D + c];
  lds[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < D) {
    for (int k = 1; k < 16; k++) sum += lds[k][lane];
    (blockIdx.y ? db : dw)[c] = Elem<T>::put(sum);
  }
}

int waves_of(int D) { return D <= 64 * kCols ? 1 : D <= 256 * kCols ? 4 : 16; }

}  // namespace

// Workgroups of the backward, which is the number of partial column sums.
int layer_norm_parts(long rows, int D) {
  const int w = waves_of(D);
  const long blocks = w == 1 ? (rows + 3) / 4 : rows, most = w == 16 ? otx_cu_count() : 2 * otx_cu_count();
  return (int)(blocks < most ? blocks : most);
}

template <typename T, int V>
static hipError_t ln_fwd(const T* x, const T* w, const T* b, T* y, float* mean, float* rstd, long rows, int D,
                         float eps, hipStream_t st) {
  const int wr = waves_of(D);
  const long blocks = wr == 1 ? (rows + 3) / 4 : rows, most = 16L * otx_cu_count();
  const int grid = (int)(blocks < most ? blocks : most);
  if (wr == 1)
    layer_norm_fwd_kernel<T, V, 1><<<grid, 256, 0, st>>>(x, w, b, y, mean, rstd, rows, D, eps);
  else if (wr == 4)
    layer_norm_fwd_kernel<T, V, 4><<<grid, 256, 0, st>>>(x, w, b, y, mean, rstd, rows, D, eps);
  else
    layer_norm_fwd_kernel<T, V, 16><<<grid, 1024, 0, st>>>(x, w, b, y, mean, rstd, rows, D, eps);
  return hipGetLastError();
}

template <typename T, int V>
static hipError_t ln_bwd(const T* x, const T* w, const float* mean, const float* rstd, const T* dy, T* dx, float* part,
                         long rows, int D, hipStream_t st) {
  const int wr = waves_of(D), G = layer_norm_parts(rows, D);
  if (D > 1024 * kCols) {
    layer_norm_dx_wide_kernel<T><<<G, 1024, 0, st>>>(x, w, mean, rstd, dy, dx, rows, D);
    layer_norm_cols_kernel<T><<<dim3((D + 255) / 256, G), 256, 0, st>>>(x, mean, rstd, dy, part, rows, D);
  } else if (wr == 1) {
    layer_norm_bwd_kernel<T, V, 1><<<G, 256, 0, st>>>(x, w, mean, rstd, dy, dx, part, rows, D);
  } else if (wr == 4) {
    layer_norm_bwd_kernel<T, V, 4><<<G, 256, 0, st>>>(x, w, mean, rstd, dy, dx, part, rows, D);
  } else {
    layer_norm_bwd_kernel<T, V, 16><<<G, 1024, 0, st>>>(x, w, mean, rstd, dy, dx, part, rows, D);
  }
  return hipGetLastError();
}

// wide: rows start at 16-byte boundaries and hold whole 16-byte vectors.
hipError_t launch_layer_norm_fwd(int dtype, bool wide, const void* x, const void* w, const void* b, void* y,
                                 float* mean, float* rstd, long rows, int D, float eps, hipStream_t st) {
#define OTX_LN(T, V) ln_fwd<T, V>((const T*)x, (const T*)w, (const T*)b, (T*)y, mean, rstd, rows, D, eps, st)
  if (dtype == 1) return wide ? OTX_LN(uint16_t, 8) : OTX_LN(uint16_t, 1);
  return wide ? OTX_LN(float, 4) : OTX_LN(float, 1);
#undef OTX_LN
}

hipError_t launch_layer_norm_bwd(int dtype, bool wide, const void* x, const void* w, const float* mean,
                                 const float* rstd, const void* dy, void* dx, void* dw, void* db, int wdtype,
                                 float* part, long rows, int D, hipStream_t st) {
#define OTX_LN(T, V) ln_bwd<T, V>((const T*)x, (const T*)w, mean, rstd, (const T*)dy, (T*)dx, part, rows, D, st)
  hipError_t e;
  if (dtype == 1)
    e = wide ? OTX_LN(uint16_t, 8) : OTX_LN(uint16_t, 1);
  else
    e = wide ? OTX_LN(float, 4) : OTX_LN(float, 1);
#undef OTX_LN
  if (e != hipSuccess) return e;
  const int G = layer_norm_parts(rows, D);
  const dim3 grid((D + 63) / 64, db ? 2 : 1);
  if (wdtype == 1)
    layer_norm_join_kernel<uint16_t><<<grid, 1024, 0, st>>>(part, (uint16_t*)dw, (uint16_t*)db, G, D);
  else
    layer_norm_join_kernel<float><<<grid, 1024, 0, st>>>(part, (float*)dw, (float*)db, G, D);
  return hipGetLastError();
}

}  // namespace otx
