// Rotary positions in both pair layouts, over part of the head, with gathered positions:
//   y1 = x1 c - x2 s,  y2 = x1 s + x2 c   with c, s = cos, sin of the row's position, in binary32,
// one rounding to the storage type.  Pairs are (2 i, 2 i + 1) or (i, i + R / 2); columns R .. D - 1
// are copied.  The gradient is the transpose, the same kernel with -s.
//
// Bound by memory: x is read once and written once, in the other order of heads and rows.  A thread
// takes one unit of V pairs (two accesses of 16 bytes) of a row, and the same unit of several heads,
// so that the position, c and s are read once for all of them.
#include "otx_args.h"
#include "otx_common.h"

namespace otx {

namespace {

template <typename T, int V>
struct Vec {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = Elem<T>::ld(p);
  } else {
    const uint4 w = *(const uint4*)p;
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = Elem<T>::get(w, i);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; i++) v.e[i] = Elem<T>::put(f[i]);
  if constexpr (V == 1)
    *p = v.e[0];
  else
    *(uint4*)p = __builtin_bit_cast(uint4, v);
}

template <int V>
__device__ __forceinline__ void load_table(const float* p, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = *p;
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 w = *(const float4*)(p + i);
      f[i] = w.x, f[i + 1] = w.y, f[i + 2] = w.z, f[i + 3] = w.w;
    }
  }
}

template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a, int heads, uint32_t units, uint32_t total) {
  const uint32_t turned = a.R / (2 * V);
  const int h0 = blockIdx.y * heads, h1 = min(h0 + heads, a.H);
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
    const uint32_t row = i / units, u = i % units, b = row / a.T, t = row % a.T;
    const T* x = (const T*)a.x + b * a.sx[0] + t * a.sx[1];
    T* y = (T*)a.y + b * a.sy[0] + t * a.sy[1];
    if (u >= turned) {  // columns that are not turned
      const int first = a.R + (int)(u - turned) * 2 * V;
      for (int h = h0; h < h1; h++) {
        float f[V];
        load<T, V>(x + h * a.sx[2] + first, f);
        store<T, V>(y + h * a.sy[2] + first, f);
        if (first + V < a.D) {
          load<T, V>(x + h * a.sx[2] + first + V, f);
          store<T, V>(y + h * a.sy[2] + first + V, f);
        }
      }
      continue;
    }
    const int at = a.positions ? a.positions[row] : (int)t;
    float c[V], s[V];
    if (at >= 0 && at < a.P) {
      load_table<V>(a.cosv + (long)at * (a.R / 2) + u * V, c);
      load_table<V>(a.sinv + (long)at * (a.R / 2) + u * V, s);
#pragma unroll
      for (int e = 0; e < V; e++) s[e] *= a.sign;
    } else {  // no such position
#pragma unroll
      for (int e = 0; e < V; e++) c[e] = s[e] = __builtin_nanf("");
    }
    const int p1 = HALF ? u * V : u * 2 * V, p2 = p1 + (HALF ? a.R / 2 : V);
#pragma unroll 4
    for (int h = h0; h < h1; h++) {
      float f[V], g[V];
      load<T, V>(x + h * a.sx[2] + p1, f);
      load<T, V>(x + h * a.sx[2] + p2, g);
      if constexpr (HALF || V == 1) {
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float x1 = f[e], x2 = g[e];
          f[e] = __builtin_fmaf(x1, c[e], -(x2 * s[e]));
          g[e] = __builtin_fmaf(x1, s[e], x2 * c[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V / 2; e++) {
          float x1 = f[2 * e], x2 = f[2 * e + 1];
          f[2 * e] = __builtin_fmaf(x1, c[e], -(x2 * s[e]));
          f[2 * e + 1] = __builtin_fmaf(x1, s[e], x2 * c[e]);
          x1 = g[2 * e], x2 = g[2 * e + 1];
          g[2 * e] = __builtin_fmaf(x1, c[V / 2 + e], -(x2 * s[V / 2 + e]));
          g[2 * e + 1] = __builtin_fmaf(x1, s[V / 2 + e], x2 * c[V / 2 + e]);
        }
      }
      store<T, V>(y + h * a.sy[2] + p1, f);
      store<T, V>(y + h * a.sy[2] + p2, g);
    }
  }
}

template <typename T, int V>
hipError_t rotary_of(const RotaryArgs& a, bool half, hipStream_t st) {
  const uint32_t units = a.R / (2 * V) + (a.D - a.R + 2 * V - 1) / (2 * V);
  const uint32_t total = (uint32_t)a.B * a.T * units;
  // Heads a thread takes: as many as leave the device two workgroups per compute unit.
  int heads = a.H;
  while (heads > 1 && (long)((total + 255) / 256) * ((a.H + heads - 1) / heads) < 2 * otx_cu_count())
    heads = (heads + 1) / 2;
  const dim3 grid(total / 256 + 1 < (1u << 20) ? (total + 255) / 256 : 1u << 20, (a.H + heads - 1) / heads);
  if (half)
    rotary_kernel<T, V, true><<<grid, 256, 0, st>>>(a, heads, units, total);
  else
    rotary_kernel<T, V, false><<<grid, 256, 0, st>>>(a, heads, units, total);
  return hipGetLastError();
}

}  // namespace

// wide: every access can be of 16 bytes (V elements divide D, 2 V divide R, aligned rows).
hipError_t launch_rotary(int dtype, const RotaryArgs& a, bool half, bool wide, hipStream_t st) {
  if (dtype == 1) return wide ? rotary_of<uint16_t, 8>(a, half, st) : rotary_of<uint16_t, 1>(a, half, st);
  return wide ? rotary_of<float, 4>(a, half, st) : rotary_of<float, 1>(a, half, st);
}

}  // namespace otx
