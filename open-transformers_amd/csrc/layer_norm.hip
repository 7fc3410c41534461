// Layer norm over the last dimension, forward and backward:
//   xh = (x - mean) rstd   y = xh w + b   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   g = dy w   dx = rstd (g - mean(g) - xh mean(g xh))   dw = sum_rows dy xh   db = sum_rows dy
// All sums in binary32 in a fixed order, one rounding of each result.
//
// Bound by memory.  A row lies in the registers of 8 to 1024 threads, as vectors of 16 bytes a thread, so
// that x is read once for the mean, the squares and the result; rows that do not fit are read again.  The
// backward's workgroups walk over rows with the columns of dw and db in registers, and leave one partial
// sum each, which a second kernel adds.  Vectors need no alignment but their elements' (the memory pipeline
// takes them at any address): rows of odd widths are read as wide as others, and only a row's last vector
// may be cut.  16384 x 2048 bf16: forward 27 us (4.9 TB/s), backward 37 (5.5), join 4; 4099 x 5005 binary32
// 31, 45 and 6 (5.3 and 5.5 TB/s; 54 and 60 us element by element).  A large copy reaches 5.2.
#include "otx_common.h"

namespace otx {

namespace {

constexpr int kMost = 1024;  // the most threads that hold a row

constexpr int threads_of(int nt) { return nt < 256 ? 256 : nt; }

// A vector of the row at p, of which the first `left` elements exist; the others are 0.
template <typename T>
__device__ __forceinline__ uint4 fetch(const T* p, int left) {
  constexpr int V = Elem<T>::VEC;
  uint4 w = make_uint4(0, 0, 0, 0);
  if (left >= V) {
    __builtin_memcpy(&w, p, 16);
  } else if (left > 0) {
    struct {
      T e[V];
    } v;
#pragma unroll
    for (int e = 0; e < V; e++) v.e[e] = e < left ? p[e] : (T)0;
    w = __builtin_bit_cast(uint4, v);
  }
  return w;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& w, float* f) {
#pragma unroll
  for (int i = 0; i < Elem<T>::VEC; i++) f[i] = Elem<T>::get(w, i);
}

template <typename T>
__device__ __forceinline__ void store(T* p, int left, const float* f) {
  constexpr int V = Elem<T>::VEC;
  struct {
    T e[V];
  } v;
#pragma unroll
  for (int i = 0; i < V; i++) v.e[i] = Elem<T>::put(f[i]);
  if (left >= V) {
    typedef uint32_t Four __attribute__((ext_vector_type(4)));
    typedef Four Words __attribute__((aligned(2)));  // of any element's alignment
    *(Words*)p = __builtin_bit_cast(Four, v);
  } else {
    asm volatile("");  // keeps these stores from being merged with the one above, which would split it
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < left) p[i] = v.e[i];
  }
}

// The sum of N values over the NT threads of a row, the same in each of them.
template <int N, int NT>
__device__ __forceinline__ void row_sum(float (&v)[N], float* lds) {
  constexpr int W = NT / 64;
#pragma unroll
  for (int m = NT < 64 ? NT / 2 : 32; m; m >>= 1)
#pragma unroll
    for (int i = 0; i < N; i++) v[i] += __shfl_xor(v[i], m);
  if constexpr (W > 1) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    __syncthreads();  // the last sums have been read
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < N; i++) lds[i * W + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
      v[i] = lds[i * W];
#pragma unroll
      for (int k = 1; k < W; k++) v[i] += lds[i * W + k];
    }
  }
}

// NT threads to a row, C columns of it in a thread's registers.
template <typename T, int NT, int C>
__global__ void __launch_bounds__(threads_of(NT))
    layer_norm_fwd_kernel(const T* x, const T* w, const T* b, T* y, float* mean, float* rstd, long rows, int D,
                          float eps) {
  constexpr int V = Elem<T>::VEC, RPB = threads_of(NT) / NT, NC = C / V;
  __shared__ float lds[NT / 64 + 1];
  const int tid = threadIdx.x % NT;
  const int steps = NT < kMost ? NC : (D + NT * V - 1) / (NT * V);  // past NC: read again
  const float inv = 1.0f / (float)D;
  for (long r = (long)blockIdx.x * RPB + threadIdx.x / NT; r < rows; r += (long)gridDim.x * RPB) {
    const T* xr = x + r * D;
    T* yr = y + r * D;
    uint4 raw[NC];
    float v[C], sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NC; i++) raw[i] = fetch(xr + (i * NT + tid) * V, D - (i * NT + tid) * V);
#pragma unroll
    for (int i = 0; i < NC; i++) unpack<T>(raw[i], v + i * V);
#pragma unroll
    for (int i = 0; i < C; i++) sum[0] += v[i];
    for (int i = NC; i < steps; i++) {
      const int c = (i * NT + tid) * V;
      float f[V];
      unpack<T>(fetch(xr + c, D - c), f);
#pragma unroll
      for (int e = 0; e < V; e++) sum[0] += f[e];
    }
    row_sum<1, NT>(sum, lds);
    const float mu = sum[0] * inv;
    sum[0] = 0.0f;
    auto squares = [&](int c, const float* f) {
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float d = c + e < D ? f[e] - mu : 0.0f;
        sum[0] = __builtin_fmaf(d, d, sum[0]);
      }
    };
#pragma unroll
    for (int i = 0; i < NC; i++) squares((i * NT + tid) * V, v + i * V);
    for (int i = NC; i < steps; i++) {
      const int c = (i * NT + tid) * V;
      float f[V];
      unpack<T>(fetch(xr + c, D - c), f);
      squares(c, f);
    }
    row_sum<1, NT>(sum, lds);
    const float rs = 1.0f / __builtin_sqrtf(__builtin_fmaf(sum[0], inv, eps));
    if (tid == 0) mean[r] = mu, rstd[r] = rs;
    auto write = [&](int c, const float* f) {
      float g[V], wf[V], bf[V];
      unpack<T>(fetch(w + c, D - c), wf);
      if (b) unpack<T>(fetch(b + c, D - c), bf);
#pragma unroll
      for (int e = 0; e < V; e++) g[e] = __builtin_fmaf((f[e] - mu) * rs, wf[e], b ? bf[e] : 0.0f);
      store(yr + c, D - c, g);
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
        unpack<T>(fetch(xr + c, D - c), f);
        write(c, f);
      }
    }
  }
}

// dx, and the workgroup's partial dw and db: part[0 .. G)[D], part[G .. 2 G)[D].
template <typename T, int NT, int C>
__global__ void __launch_bounds__(threads_of(NT))
    layer_norm_bwd_kernel(const T* x, const T* w, const float* mean, const float* rstd, const T* dy, T* dx, float* part,
                          long rows, int D) {
  constexpr int V = Elem<T>::VEC, RPB = threads_of(NT) / NT, NC = C / V;
  __shared__ float lds[NT <= 64 ? 2 * NT * C : NT / 32];
  const int tid = threadIdx.x % NT;
  const float inv = 1.0f / (float)D;
  float dw[C], db[C];
  uint4 wr[NC];
#pragma unroll
  for (int i = 0; i < NC; i++) wr[i] = fetch(w + (i * NT + tid) * V, D - (i * NT + tid) * V);
#pragma unroll
  for (int i = 0; i < C; i++) dw[i] = db[i] = 0.0f;
  for (long r = (long)blockIdx.x * RPB + threadIdx.x / NT; r < rows; r += (long)gridDim.x * RPB) {
    const float mu = mean[r], rs = rstd[r];
    const T *xr = x + r * D, *gr = dy + r * D;
    uint4 xw[NC], gw[NC];
    float xh[C], g[C], sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NC; i++) {
      xw[i] = fetch(xr + (i * NT + tid) * V, D - (i * NT + tid) * V);
      gw[i] = fetch(gr + (i * NT + tid) * V, D - (i * NT + tid) * V);
    }
#pragma unroll
    for (int i = 0; i < NC; i++) {
      unpack<T>(xw[i], xh + i * V);
      unpack<T>(gw[i], g + i * V);
    }
#pragma unroll
    for (int i = 0; i < C; i++) {  // past the row's end w and dy are 0 and x - mean is finite
      xh[i] = (xh[i] - mu) * rs;
      dw[i] = __builtin_fmaf(g[i], xh[i], dw[i]);
      db[i] += g[i];
      g[i] *= Elem<T>::get(wr[i / V], i % V);
      sum[0] += g[i];
      sum[1] = __builtin_fmaf(g[i], xh[i], sum[1]);
    }
    row_sum<2, NT>(sum, lds);
    const float m1 = sum[0] * inv, m2 = sum[1] * inv;
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const int c = (i * NT + tid) * V;
      if (c < D) {
        float f[V];
#pragma unroll
        for (int e = 0; e < V; e++) f[e] = rs * (g[i * V + e] - m1 - xh[i * V + e] * m2);
        store(dx + r * D + c, D - c, f);
      }
    }
  }
  if constexpr (NT <= 64) {  // the sums of a wave's rows, then of the four waves, in order
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int m = 32; m >= NT; m >>= 1)
#pragma unroll
      for (int i = 0; i < C; i++) dw[i] += __shfl_xor(dw[i], m), db[i] += __shfl_xor(db[i], m);
    for (int k = 1; k < 4; k++) {
      __syncthreads();
      if (wave == k && lane < NT)
#pragma unroll
        for (int i = 0; i < C; i++) lds[i * NT + lane] = dw[i], lds[(C + i) * NT + lane] = db[i];
      __syncthreads();
      if (wave == 0 && lane < NT)
#pragma unroll
        for (int i = 0; i < C; i++) dw[i] += lds[i * NT + lane], db[i] += lds[(C + i) * NT + lane];
    }
    if (threadIdx.x >= NT) return;
  }
  float *pw = part + (long)blockIdx.x * D, *pb = pw + (long)gridDim.x * D;
#pragma unroll
  for (int i = 0; i < NC; i++)
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const int c = (i * NT + tid) * V + e;
      if (c < D) store(pw + c, D - c, dw + i * V + e), store(pb + c, D - c, db + i * V + e);
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
    row_sum<2, 1024>(sum, lds);
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

// The sum of G partial rows: a workgroup takes 16 columns, 64 threads each.
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_join_kernel(const float* part, T* dw, T* db, int G, int D) {
  __shared__ float lds[64][16];
  const int col = threadIdx.x & 15, at = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  const float* p = part + (blockIdx.y ? (long)G * D : 0);
  float sum = 0.0f;
  if (c < D)
#pragma unroll 8
    for (int g = at; g < G; g += 64) sum += p[(long)g * D + c];
  lds[at][col] = sum;
#pragma unroll
  for (int n = 32; n; n >>= 1) {
    __syncthreads();
    if (at < n) lds[at][col] = sum += lds[at + n][col];
  }
  if (at == 0 && c < D) (blockIdx.y ? db : dw)[c] = Elem<T>::put(sum);
}

struct Shape {
  int threads, cols;
};
// The fewest threads that hold a row in 8 columns each, then a wave and more with up to 32: one
// wave's sums need no barrier.  262144 rows of 64 bf16, forward and backward: 14 and 20 us with 8
// threads to a row, 66 and 75 with 64; 8192 of 2048: 15 and 22 us with 64, 18 and 26 with 256,
// 67 and 49 with 1024.
Shape shape_of(int D) {
  if (D <= 512) return {D <= 64 ? 8 : D <= 128 ? 16 : D <= 256 ? 32 : 64, 8};
  if (D <= 2048) return {64, D <= 1024 ? 16 : 32};
  if (D <= 8192) return {256, D <= 4096 ? 16 : 32};
  return {512, 32};
}

}  // namespace

// Workgroups of the backward, which is the number of partial column sums: as many as the registers let
// stay at once, or half of that for the 16 columns a thread (twice as many: as fast, and a join twice as long).
int layer_norm_parts(long rows, int D) {
  const Shape s = shape_of(D);
  const int n = threads_of(s.threads) / s.threads;
  const long blocks = (rows + n - 1) / n;
  const long most = (s.threads > 256 ? 1 : s.cols == 8 ? 4 : 2) * otx_cu_count();
  return (int)(blocks < most ? blocks : most);
}

#define OTX_LN_SHAPES(X) X(8, 8) X(16, 8) X(32, 8) X(64, 8) X(64, 16) X(64, 32) X(256, 16) X(256, 32)

template <typename T>
static hipError_t ln_fwd(const T* x, const T* w, const T* b, T* y, float* mean, float* rstd, long rows, int D,
                         float eps, hipStream_t st) {
  const Shape s = shape_of(D);
  const int n = threads_of(s.threads) / s.threads;
  const long blocks = (rows + n - 1) / n, most = 16L * otx_cu_count();
  const int grid = (int)(blocks < most ? blocks : most);
#define OTX_LN(N, C) \
  if (s.threads == N && s.cols == C) \
    layer_norm_fwd_kernel<T, N, C><<<grid, threads_of(N), 0, st>>>(x, w, b, y, mean, rstd, rows, D, eps);
  OTX_LN_SHAPES(OTX_LN)
#undef OTX_LN
  // 16 columns each leave room for two workgroups: 1024 rows of 16384 binary32 31 us, with 512 threads 37.
  if (s.threads == 512) layer_norm_fwd_kernel<T, kMost, 16><<<grid, kMost, 0, st>>>(x, w, b, y, mean, rstd, rows, D, eps);
  return hipGetLastError();
}

template <typename T>
static hipError_t ln_bwd(const T* x, const T* w, const float* mean, const float* rstd, const T* dy, T* dx, float* part,
                         long rows, int D, hipStream_t st) {
  const Shape s = shape_of(D);
  const int G = layer_norm_parts(rows, D);
  if (D > s.threads * s.cols) {
    layer_norm_dx_wide_kernel<T><<<G, 1024, 0, st>>>(x, w, mean, rstd, dy, dx, rows, D);
    layer_norm_cols_kernel<T><<<dim3((D + 255) / 256, G), 256, 0, st>>>(x, mean, rstd, dy, part, rows, D);
    return hipGetLastError();
  }
#define OTX_LN(N, C) \
  if (s.threads == N && s.cols == C) \
    layer_norm_bwd_kernel<T, N, C><<<G, threads_of(N), 0, st>>>(x, w, mean, rstd, dy, dx, part, rows, D);
  OTX_LN_SHAPES(OTX_LN)
#undef OTX_LN
  if (s.threads == 512) layer_norm_bwd_kernel<T, 512, 32><<<G, 512, 0, st>>>(x, w, mean, rstd, dy, dx, part, rows, D);
  return hipGetLastError();
}

hipError_t launch_layer_norm_fwd(int dtype, const void* x, const void* w, const void* b, void* y,
                                 float* mean, float* rstd, long rows, int D, float eps, hipStream_t st) {
#define OTX_LN(T) ln_fwd<T>((const T*)x, (const T*)w, (const T*)b, (T*)y, mean, rstd, rows, D, eps, st)
  if (dtype == 1) return OTX_LN(uint16_t);
  return OTX_LN(float);
#undef OTX_LN
}

hipError_t launch_layer_norm_bwd(int dtype, const void* x, const void* w, const float* mean,
                                 const float* rstd, const void* dy, void* dx, void* dw, void* db, int wdtype,
                                 float* part, long rows, int D, hipStream_t st) {
#define OTX_LN(T) ln_bwd<T>((const T*)x, (const T*)w, mean, rstd, (const T*)dy, (T*)dx, part, rows, D, st)
  hipError_t e;
  if (dtype == 1)
    e = OTX_LN(uint16_t);
  else
    e = OTX_LN(float);
#undef OTX_LN
  if (e != hipSuccess) return e;
  const int G = layer_norm_parts(rows, D);
  const dim3 grid((D + 15) / 16, db ? 2 : 1);
  if (wdtype == 1)
    layer_norm_join_kernel<uint16_t><<<grid, 1024, 0, st>>>(part, (uint16_t*)dw, (uint16_t*)db, G, D);
  else
    layer_norm_join_kernel<float><<<grid, 1024, 0, st>>>(part, (float*)dw, (float*)db, G, D);
  return hipGetLastError();
}

}  // namespace otx
