// Rotary positions in both pair layouts, over part of the head, with gathered positions:
//   y1 = x1 c - x2 s,  y2 = x1 s + x2 c   with c, s = cos, sin of the row's position, in binary32,
// one rounding to the storage type.  Pairs are (2 i, 2 i + 1) or (i, i + R / 2); columns R .. D - 1
// are copied.  The gradient is the transpose, the same kernel with -s.
//
// Bound by memory: x is read once and written once, in the other order of heads and rows.  A thread takes
// one unit of V pairs (two accesses of up to 16 bytes, at any address) of a row, and the same unit of several
// heads, so that the position, c and s are read once for all of them.  4 x 4096 rows of 16 heads of 128 bf16
// columns, pairs interleaved: 30 us for 134 MB and the tables, 4.5 TB/s (a large copy reaches 5.2).
#include "otx_args.h"
#include "otx_common.h"

namespace otx {

namespace {

// N bytes, to be read and written at any address.
template <int N> struct Bytes { typedef uint32_t __attribute__((ext_vector_type(N / 4))) V; typedef V At __attribute__((aligned(2))); };
template <> struct Bytes<4> { typedef uint32_t V; typedef V At __attribute__((aligned(2))); };
template <> struct Bytes<2> { typedef uint16_t V, At; };

template <typename T, int V>
struct Vec {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&f)[V]) {
  typedef Bytes<V * sizeof(T)> Raw;
  const auto v = __builtin_bit_cast(Vec<T, V>, (typename Raw::V)*(const typename Raw::At*)p);
#pragma unroll
  for (int i = 0; i < V; i++) f[i] = Elem<T>::ld(v.e + i);
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  typedef Bytes<V * sizeof(T)> Raw;
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; i++) v.e[i] = Elem<T>::put(f[i]);
  *(typename Raw::At*)p = __builtin_bit_cast(typename Raw::V, v);
}

template <int V>
__device__ __forceinline__ void load_table(const float* p, float (&f)[V]) {
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int i = 0; i < V; i += W) load<float, W>(p + i, *(float (*)[W])(f + i));
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
      const int second = first + V < a.D ? first + V : first;
#pragma unroll 4
      for (int h = h0; h < h1; h++) {
        float f[V], g[V];
        load<T, V>(x + h * a.sx[2] + first, f);
        load<T, V>(x + h * a.sx[2] + second, g);
        store<T, V>(y + h * a.sy[2] + first, f);
        store<T, V>(y + h * a.sy[2] + second, g);
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

// Wide accesses where the turned and the copied columns divide into them.  8192 rows of 16 heads, 24 of
// 96 bf16 columns turned: 15 us by 4, 22 by 1 (by 2, as 20 of 80 allows, 20 and 22: not worth its code);
// 128 of 128 by 8: 13 us, its traffic at 5.2 TB/s.
hipError_t launch_rotary(int dtype, const RotaryArgs& a, bool half, hipStream_t st) {
  const int odd = a.R / 2 | (a.D - a.R);  // V divides both
  if (dtype == 1) {
    if (odd % 8 == 0) return rotary_of<uint16_t, 8>(a, half, st);
    return odd % 4 == 0 ? rotary_of<uint16_t, 4>(a, half, st) : rotary_of<uint16_t, 1>(a, half, st);
  }
  return odd % 4 == 0 ? rotary_of<float, 4>(a, half, st) : rotary_of<float, 1>(a, half, st);
}

}  // namespace otx
