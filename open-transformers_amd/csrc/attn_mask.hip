// Masked flash attention: document and prefix masks, padding, windows of any size, tanh-capped
// scores and a linear distance bias, forward and backward, for any sequence length.
//
//   t_ij = cap tanh(sigma q_i.k_j / cap)  (or sigma q_i.k_j)      sigma = 1 / sqrt(D)
//   u_ij = t_ij - slope_h |i - j|
//   O_i  = sum_j p_ij v_j,  p_i = softmax of u_i over the visible j; a row that sees nothing is 0
//   visible(i, j): doc_i == doc_j >= 0 and ((j <= i and (window == 0 or i - j < window)) or j < prefix_b)
//
//   D_i = dO_i.O_i   dU = P (dO V^T - D)   dS = dU (1 - (t / cap)^2)
//   dQ = sigma dS K   dK = sigma dS^T Q   dV = P^T dO
//
// One pass over the keys with a running maximum and sum, all statistics and accumulators in
// binary32.  The products run on the matrix units in the storage type: v_mfma_f32_32x32x16_bf16,
// or v_mfma_f32_32x32x2_f32 for binary32 tensors.  P and dS are rounded to bf16 where they are
// the operand of a bf16 product (half a step, 2^-8 relative, unbiased; the accumulation is
// binary32).  No atomics: dQ and dK/dV are separate kernels that each own their output rows and
// form S and dP themselves, so results repeat bit for bit.
//
// Layout.  A wave owns 32 rows (queries, or keys in the dK/dV kernel) and holds them as the
// matrix unit's B operand; the other side's tile lies in LDS.  S^T = K Q^T then leaves every
// lane with one query (lane % 32) and 16 keys of each 32-key block, so the softmax needs one
// exchange between half-waves, and the result registers are, as they are, the B operand of the
// next product O^T = V^T P^T: the k index of a product may be permuted when both operands are,
// and the A operand is read from LDS with the same permutation (transposing reads,
// ds_read_b64_tr_b16, for bf16).  P and dS never pass through LDS.
//
// D_i is formed from O with eight more bits than its bf16 holds, which the forward keeps where a gradient
// will be wanted: rounded to bf16, O would alone cost gradients of 2^-8 relative where rows see few keys
// (documents of two tokens, dQ: 0.0036 of its norm off binary64 instead of 0.0026, of which 0.0017 is the
// rounding of the result), and a byte an element is what it takes.
//
// Masked pairs contribute nothing, whatever their rows hold.  A weight of 0 times a NaN or an
// infinity is NaN, so a tile that some rows of the workgroup do not see whole is checked for
// non-finite values, and a workgroup that finds one does its rows over, one at a time
// (careful_row), with products of visible pairs only.
#include "otx_args.h"
#include "otx_common.h"

namespace otx {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kTab = 64;  // tokens per entry of the block table
constexpr int kThreads = 256;

// ---- matrix products of a storage type -----------------------------------------------------
// Rows of a tile lie in LDS with D * sizeof(T) bytes each, cut into 16-byte chunks; chunk c of
// row r is kept at position c ^ swizzle(r).  All of a lane's addresses in a tile are one base
// with a constant exclusive-or and a constant offset.
template <typename T, int D>
struct Tile {
  static constexpr int NC = D * (int)sizeof(T) / 16;  // chunks in a row
  static constexpr int KS = NC / 2;                   // steps over D of a row product (a chunk for each half-wave)
  static constexpr int DT = D / 32;
  static constexpr int RB = D * (int)sizeof(T);
  static constexpr int SUB = 32 * RB;  // bytes of 32 rows

  // A row product reads the same chunk of 16 rows at a time, and a transposing read four neighbouring
  // chunks of four rows: both spread over all 64 banks.  (Row & 15 alone makes the transposing reads
  // 2.3 times slower: 6.8 clocks against 3.0, measured on 8 waves that read nothing else.)  Binary32
  // column reads take half the banks from row r and half from row r + 4.
  static constexpr int SW = NC == 32 ? 7 : 15;  // the swizzle repeats after SW + 1 rows
  __device__ static __forceinline__ int swizzle(int row) {
    if constexpr (sizeof(T) == 4 && NC == 32) return (row & 3) | (row & 4) << 1;
    if constexpr (sizeof(T) == 4) return (row & 3) | (row & 4) << 1 | (row & 8) >> 1;
    if constexpr (NC == 16) return (row & 3) << 2 | ((row >> 2) & 3);
    return (row & 2) << 1 | ((row >> 2) & 3);
  }
  __device__ static __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ swizzle(row)) << 4); }

  // Row fragments: lane l takes row l % 32 of 32, chunks 2 ks + l / 32.
  __device__ static __forceinline__ uint32_t row_base(uint32_t lds, int lane) { return lds + at(lane & 31, lane >> 5); }
  // Column fragments of 32 rows: see cols().
  __device__ static __forceinline__ uint32_t col_base(uint32_t lds, int lane) {
    if constexpr (sizeof(T) == 2) {
      const int col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      return lds + at(4 * (lane >> 5) + ((lane & 15) >> 2), col >> 3) + (col & 7) * 2;
    } else {
      return lds + at(4 * (lane >> 5), (lane & 31) >> 2) + (lane & 3) * 4;
    }
  }
};

template <typename V>
__device__ __forceinline__ V lds_at(uint32_t address) {
  return *(const __attribute__((address_space(3))) V*)address;
}

// The row fragments of 32 tile rows.
template <typename T, int D>
struct Rows {
  using L = Tile<T, D>;
  u32x4 f[L::KS];
  __device__ __forceinline__ void read(uint32_t base, int ks) { f[ks] = lds_at<u32x4>(base ^ (ks << 5)); }
  __device__ __forceinline__ void read(uint32_t base) {
#pragma unroll
    for (int ks = 0; ks < L::KS; ks++) read(base, ks);
  }
};

template <typename T>
__device__ __forceinline__ f32x16 mma_rows(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  } else {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(otx_u2f(a.x), otx_u2f(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(otx_u2f(a.y), otx_u2f(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(otx_u2f(a.z), otx_u2f(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x2f32(otx_u2f(a.w), otx_u2f(b.w), c, 0, 0, 0);
  }
}

// The transposed fragments of 32 tile rows X[k], for acc[dt][d][n] += sum_k X[k][32 dt + d] W[k][n]
// with W in result layout: element r of a lane in half-wave h is row otx_row(r, h).
template <typename T, int D>
struct Cols;

template <int D>
struct Cols<uint16_t, D> {
  using L = Tile<uint16_t, D>;
  using W = bf16x8;
  s16x4 f[2][L::DT][2];
  // 16 lanes of a transposing read take rows k .. k + 3, columns 16 g .. 16 g + 15: lane i addresses
  // row k + i / 4, columns 4 (i % 4) .., and receives column i of the four rows.
  __device__ __forceinline__ void read(uint32_t base, int s, int dt) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
#pragma unroll
    for (int g = 0; g < 2; g++)
      f[s][dt][g] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4*)((base ^ (dt << 6 | g << 5)) + (16 * s + 8 * g) * L::RB));
  }
  __device__ __forceinline__ void read(uint32_t base) {
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int dt = 0; dt < L::DT; dt++) read(base, s, dt);
  }
  __device__ __forceinline__ static bf16x8 weights(const f32x16& w, int s) {
    bf16x8 b;
#pragma unroll
    for (int j = 0; j < 8; j++) b[j] = (__bf16)w[8 * s + j];
    return b;
  }
  __device__ __forceinline__ void mma(f32x16 (&acc)[L::DT], bf16x8 b, int s, int dt) const {
    const s16x8 a = __builtin_shufflevector(f[s][dt][0], f[s][dt][1], 0, 1, 2, 3, 4, 5, 6, 7);
    acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), b, acc[dt], 0, 0, 0);
  }
  __device__ __forceinline__ void mma(f32x16 (&acc)[L::DT], const f32x16& w) const {
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const bf16x8 b = weights(w, s);
#pragma unroll
      for (int dt = 0; dt < L::DT; dt++) mma(acc, b, s, dt);
    }
  }
};

template <int D>
struct Cols<float, D> {
  using L = Tile<float, D>;
  using W = f32x8;
  float f[2][L::DT][8];
  __device__ __forceinline__ void read(uint32_t base, int s, int dt) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int row = otx_row(8 * s + j, 0);
      f[s][dt][j] = lds_at<float>((base ^ (dt << 7 | L::swizzle(row) << 4)) + row * L::RB);
    }
  }
  __device__ __forceinline__ void read(uint32_t base) {
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int dt = 0; dt < L::DT; dt++) read(base, s, dt);
  }
  __device__ __forceinline__ static W weights(const f32x16& w, int s) {
    W b;
#pragma unroll
    for (int j = 0; j < 8; j++) b[j] = w[8 * s + j];
    return b;
  }
  __device__ __forceinline__ void mma(f32x16 (&acc)[L::DT], W b, int s, int dt) const {
#pragma unroll
    for (int j = 0; j < 8; j++) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(f[s][dt][j], b[j], acc[dt], 0, 0, 0);
  }
  __device__ __forceinline__ void mma(f32x16 (&acc)[L::DT], const f32x16& w) const {
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const W b = weights(w, s);
#pragma unroll
      for (int j = 0; j < 8; j++)  // the accumulators in turn
#pragma unroll
        for (int dt = 0; dt < L::DT; dt++)
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(f[s][dt][j], b[j], acc[dt], 0, 0, 0);
    }
  }
};

// Step i of KS: the column fragments are read while row fragments are used, into the registers that those leave.
template <typename T, int D>
__device__ __forceinline__ void read_step(Cols<T, D>& c, uint32_t base, int i) {
  constexpr int EACH = Tile<T, D>::KS / (2 * Tile<T, D>::DT);
  if (i % EACH == 0) c.read(base, i / EACH / Tile<T, D>::DT, i / EACH % Tile<T, D>::DT);
}

// Reads above it are in flight before the products below it begin.
__device__ __forceinline__ void fence_schedule() { __builtin_amdgcn_sched_barrier(0); }

template <typename T>
__device__ __forceinline__ float element(const u32x4& v, int e) {
  if constexpr (sizeof(T) == 4) return otx_u2f(v[e]);
  return otx_u2f((e & 1) ? (v[e >> 1] & 0xffff0000u) : (v[e >> 1] << 16));
}

// The largest magnitude seen, as bits: from which an infinity or a NaN is told.
template <typename T>
struct Largest {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  uint32_t m = 0;
  __device__ __forceinline__ void take(const u32x4& v) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (sizeof(T) == 2)
        m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                                   __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu)));
      else
        m = __builtin_elementwise_max(m, v[i] & 0x7fffffffu);
    }
  }
  __device__ __forceinline__ bool nonfinite() const {
    if constexpr (sizeof(T) == 2) return (m & 0xffffu) >= 0x7f80u || m >> 16 >= 0x7f80u;
    return m >= 0x7f800000u;
  }
};

// x, as a value that is formed here: what rarely run code makes of it does not wait in registers
// through the loops (it did, and cost them up to 40).
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// For branches off the common path: registers are kept for the other side.
__device__ __forceinline__ bool rare(bool x) { return __builtin_expect(x, 0); }

// ---- which tiles take part -------------------------------------------------------------------
struct Band {  // the mask of one batch row, apart from documents
  int S, window, prefix;
  __device__ __forceinline__ bool any(int q0, int q1, int k0, int k1) const {  // some pair of the rectangle
    return (k0 <= q1 && (window == 0 || k1 > q0 - window)) || k0 < prefix;
  }
  __device__ __forceinline__ bool all(int q0, int q1, int k0, int k1) const {  // every pair
    return (k1 <= q0 && (window == 0 || k0 > q1 - window)) || k1 < prefix;
  }
};

struct Docs {  // documents of a range of tokens
  int lo, hi, pad;
};
__device__ __forceinline__ Docs docs_of(const i32x4* table, int first, int last, int nb) {
  if (!table) return {0, 0, 0};
  Docs d = {0x7fffffff, -1, 0};
  for (int i = first; i <= last && i < nb; i++) {
    const i32x4 t = table[i];
    d.lo = min(d.lo, t.x);
    d.hi = max(d.hi, t.y);
    d.pad |= t.z;
  }
  return d;
}

// The tiles of BT tokens that a range of `own` tokens meets, 64 at a time (a lane tests one): of these
// first the ones that all of the range sees whole, then those that the mask cuts, so that the loop over
// whole tiles holds no mask.
template <int BT, bool OWN_QUERIES, bool TEAM>  // TEAM: every fourth tile, dealt to the waves in turn
struct TileIter {
  uint64_t whole, part, docs;  // docs: tiles whose pairs need not be of one document
  uint64_t whole0, part0;
  int base, n, o0, o1, seen;
  bool cut, mixed;  // of the tile that next() returned
  Docs own;
  __device__ __forceinline__ void init(int own0, int own1, const Docs& d, int ntiles) {
    o0 = own0, o1 = own1, own = d, n = ntiles, whole = part = 0, base = -64, cut = mixed = false, seen = 0;
  }
  // Starts over for the same range.
  __device__ __forceinline__ void again() {
    base = n <= 64 ? 0 : -64;
    whole = n <= 64 ? whole0 : 0;
    part = n <= 64 ? part0 : 0;
  }
  __device__ __forceinline__ bool load(const Band& band, const i32x4* table, int nb, int lane) {
    base += 64;
    if (base >= n) return false;
    const int t = base + lane, t0 = t * BT, t1 = t0 + BT - 1;
    bool a = false, all = false, d = false;
    if (t < n) {
      a = OWN_QUERIES ? band.any(o0, o1, t0, t1) : band.any(t0, t1, o0, o1);
      all = OWN_QUERIES ? band.all(o0, o1, t0, t1) : band.all(t0, t1, o0, o1) && t1 < band.S;
      if (a && table) {
        const Docs x = docs_of(table, t0 / kTab, t1 / kTab, nb);
        a = x.lo <= own.hi && own.lo <= x.hi;
        d = x.lo != x.hi || own.lo != own.hi || x.pad || own.pad;
      }
    }
    docs = __ballot(d);
    whole = whole0 = __ballot(a && all && !d);
    part = part0 = __ballot(a && (!all || d));
    if constexpr (TEAM) {
      const uint64_t below = (1ull << lane) - 1;
      const int rank = (whole >> lane) & 1 ? __popcll(whole & below) : __popcll(whole) + __popcll(part & below);
      const uint64_t mine = __ballot(((rank + seen) & 3) == (int)(threadIdx.x >> 6));
      seen += __popcll(whole | part);
      whole &= mine, part &= mine;
    }
    return true;
  }
  __device__ __forceinline__ int next(const Band& band, const i32x4* table, int nb, int lane) {
    while (rare((whole | part) == 0)) {
      if (!load(band, table, nb, lane)) return -1;
    }
    cut = whole == 0;
    const int i = __builtin_ctzll(cut ? part : whole);
    if (cut)
      part &= part - 1;
    else
      whole &= whole - 1;
    mixed = (docs >> i) & 1;
    return base + i;
  }
};

// Replaces the elements of a result block whose pair does not take part.  The owned row is query
// `own` against keys o + otx_row(r, h), or key `own` against queries.  ok: it is a token of a document;
// id: which, lid: those of the 32 rows (padding, below 0, equals none that is ok).
template <bool OWN_QUERIES, typename F>
__device__ __forceinline__ void mask_block(const Band& band, bool mixed, const int* lid, int o, int own, bool ok,
                                           int id, int h, F drop) {
  // relative to the first row of this half-wave: lo < row <= hi, or (a key in the prefix) row < pre
  const int base = o + 4 * h, w = band.window ? band.window : 0x20000000, none = -0x40000000;
  const int end = band.S - base;
  const int hi = ok ? OWN_QUERIES ? own - base : min(own + w - base, end) - 1 : none;
  const int lo = OWN_QUERIES ? own - w - base : own - 1 - base;
  if (band.prefix) {
    const int pre = !ok ? none : OWN_QUERIES ? band.prefix - base : own < band.prefix ? end : none;
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int row = otx_row(r, 0);
      drop(r, !(((row <= hi) & (row > lo)) | (row < pre)));
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; r++) drop(r, otx_row(r, 0) > hi);
    if (!OWN_QUERIES || band.window) {
#pragma unroll
      for (int r = 0; r < 16; r++) drop(r, otx_row(r, 0) <= lo);
    }
  }
  if (mixed) {
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const i32x4 ids = *(const i32x4*)(lid + 8 * g + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; i++) drop(4 * g + i, ids[i] != id);
    }
  }
}

// x of this lane and of the one 32 away, joined.
template <typename F>
__device__ __forceinline__ float join_halves(float x, F f) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(otx_f2u(x), otx_f2u(x), false, false));
  return f(otx_u2f(v[0]), otx_u2f(v[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  return join_halves(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float max_halves(float x) {
  return join_halves(x, [](float a, float b) { return fmaxf(a, b); });
}

// tanh-capped score in units of log 2, from a raw dot product; for the backward t / cap is kept.
template <typename T>
__device__ __forceinline__ float cap_tanh(float s, float sigma_over_cap) {
  if constexpr (sizeof(T) == 4) {
    return tanhf(s * sigma_over_cap);
  } else {  // 1 - 2 / (e^2x + 1): absolute error of a few 2^-24, far below a bf16 score's own
    const float e = __builtin_amdgcn_exp2f(s * (2.0f * kLog2e * sigma_over_cap));
    return __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
  }
}

// Copies of 16 or 4 bytes a lane straight into LDS, from `from` + off (off: bytes, of each lane) to `to` +
// 16 (4) * lane.  Written out so that the compiler does not count them: it cannot tell the buffer that
// is being filled from the one that is being read, and would wait for the copies before every read of
// LDS.  The kernels wait for them in arrived(), before the barrier that hands a buffer over.
template <int BYTES>
__device__ __forceinline__ void copy_lanes(const void* from, int off, uint32_t to) {
  const uint64_t f = (uint64_t)from;  // the same in every lane, as is `to`: told to the compiler
  const uint64_t base = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(f >> 32)) << 32 |
                        (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)f);
  const uint32_t lds = __builtin_amdgcn_readfirstlane(to);
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base)
                 : "m0", "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base)
                 : "m0", "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// ---- staging -------------------------------------------------------------------------------------
// BT rows of a tensor, copied straight into LDS (16 bytes a lane, no registers); rows past the end
// repeat the last one.  A wave's copy fills consecutive LDS, so the swizzle is applied to the chunk
// that a lane fetches.
template <typename T, int D, int BT, bool TEAM>  // TEAM: the lanes of one wave; otherwise the whole workgroup
struct Stage {
  using L = Tile<T, D>;
  static constexpr int NTH = TEAM ? 64 : kThreads;
  static constexpr int N = BT * L::NC / NTH, RS = NTH / L::NC;  // steps, rows a step
  static_assert(BT * L::NC % NTH == 0, "whole steps");
  const char* base;
  int stride, off, row, col;  // bytes, but for row
  __device__ __forceinline__ void init(const T* p, long s) {
    const int r = threadIdx.x % NTH / L::NC;
    row = r, col = ((threadIdx.x % L::NC) ^ L::swizzle(r)) * 16;
    base = (const char*)p, stride = (int)s * (int)sizeof(T), off = r * stride + col;
  }
  // From the chunk that this lane fetches in the first step to that of step i: the swizzle's bits are
  // exclusive-ors of the row's, so that of row r + i RS is that of r with that of i RS.
  __device__ __forceinline__ int turn(int i) const { return (col ^ (L::swizzle(i * RS) << 4)) - col; }
  __device__ __forceinline__ void copy(char* lds, int row0, int S) const {
    const char* p = base + (long)row0 * stride;
    const uint32_t to = lds_address(lds) + (TEAM ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024);
    const int last = S - 1 - row0;
    if (!rare(last < BT - 1)) {
#pragma unroll
      for (int i = 0; i < N; i++) copy_lanes<16>(p + (long)i * RS * stride, off + turn(i), to + i * NTH * 16);
    } else {
      const int r = here(row);
#pragma unroll
      for (int i = 0; i < N; i++)
        copy_lanes<16>(p, off + (min(r + i * RS, last) - r) * stride + turn(i), to + i * NTH * 16);
    }
  }
  // This thread's share of a tile in LDS.
  __device__ __forceinline__ static void look(const char* lds, Largest<T>& largest) {
    const char* at = lds + here(threadIdx.x) % NTH * 16;
#pragma unroll
    for (int i = 0; i < N; i++) largest.take(*(const u32x4*)(at + i * NTH * 16));
    fence_schedule();
  }
};

// This wave's copies have arrived; with the barrier after it, everybody's.
__device__ __forceinline__ void arrived() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70);  // the same for the compiler, which has its own loads counted as done
  __syncthreads();
}
// The same for a wave with tiles of its own, which has also read what the next copies overwrite.
__device__ __forceinline__ void arrived_here() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);
}

template <typename T, int D>
__device__ __forceinline__ void load_own(u32x4 (&f)[D * sizeof(T) / 32], const T* base, long stride, int row, int lane) {
#pragma unroll
  for (int ks = 0; ks < Tile<T, D>::KS; ks++)
    f[ks] = *(const u32x4*)(base + (long)row * stride + (2 * ks + (lane >> 5)) * (16 / (int)sizeof(T)));
}

// The eight bits of x after those that its bf16 rounding keeps, signed and rounded, in bits 8 to 15.
__device__ __forceinline__ int low_bits(float x) {
  const uint32_t high = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)x) << 16;
  return min((int)(__float_as_uint(x) + 128 - high), 0x7fff);
}
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  const uint32_t ab = __builtin_amdgcn_perm(low_bits(b), low_bits(a), 0x0c0c0501);
  const uint32_t cd = __builtin_amdgcn_perm(low_bits(d), low_bits(c), 0x05010c0c);
  return ab | cd;
}
__device__ __forceinline__ float with_low(float high, int low) { return __uint_as_float(__float_as_uint(high) + ((uint32_t)low << 8)); }

// Writes the 32 rows of a wave: acc^T (column n: row n) times f, to row * stride.  The results pass
// through this wave's share of LDS, so that 16 bytes a lane go to whole rows: stored as the lanes hold
// them, 8 bytes to each of 32 rows, they took 3 us of a workgroup's time.
template <typename T, int D, typename O>
__device__ __forceinline__ void store_rows(O* out, long stride, int row0, int S, char* lds, const f32x16 (&acc)[D / 32],
                                           float f, signed char* low = nullptr) {
  const int lane = here(threadIdx.x) & 63;
  constexpr int E = 16 / (int)sizeof(O), C = D / E;  // elements of a chunk, chunks of a row
  const int n = lane & 31, h = lane >> 5;
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int d = 32 * dt + 8 * g + 4 * h;
      char* at = lds + n * D * (int)sizeof(O) + (((d / E) ^ (n & (C - 1) & 15)) << 4) + d % E * (int)sizeof(O);
      if constexpr (sizeof(O) == 2) {
        bf16x4 o;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = (__bf16)(acc[dt][4 * g + i] * f);
        *(bf16x4*)at = o;
      } else {
        f32x4 o;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = acc[dt][4 * g + i] * f;
        *(f32x4*)at = o;
      }
    }
#pragma unroll
  for (int i = 0; i < C / 2; i++) {
    const int r = (i * 64 + lane) / C, c = (i * 64 + lane) % C;
    const u32x4 v = *(const u32x4*)(lds + r * D * (int)sizeof(O) + ((c ^ (r & (C - 1) & 15)) << 4));
    if (row0 + r < S) *(u32x4*)(out + (row0 + r) * stride + c * E) = v;
  }
  if (sizeof(O) == 2 && low) {
    constexpr int CL = D / 16;
#pragma unroll
    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        *(uint32_t*)(lds + n * D + (((2 * dt + g / 2) ^ (n & (CL - 1))) << 4) + 8 * (g & 1) + 4 * h) =
            low_bytes(acc[dt][4 * g] * f, acc[dt][4 * g + 1] * f, acc[dt][4 * g + 2] * f, acc[dt][4 * g + 3] * f);
      }
#pragma unroll
    for (int i = 0; i < CL / 2; i++) {
      const int r = (i * 64 + lane) / CL, c = (i * 64 + lane) % CL;
      const u32x4 v = *(const u32x4*)(lds + r * D + ((c ^ (r & (CL - 1))) << 4));
      if (row0 + r < S) *(u32x4*)(low + (long)(row0 + r) * D + c * 16) = v;
    }
  }
}

// The same for a team, whose four waves hold summands of the same 32 rows: added in the waves' order.
template <typename T, int D, typename O>
__device__ __forceinline__ void join_rows(O* out, long stride, int row0, int S, char* lds, const f32x16 (&acc)[D / 32],
                                          float f, signed char* low = nullptr) {
  constexpr int C = D / 4, PART = 32 * D * 4;  // chunks of four columns in a row, bytes of a wave's summand
  const int tid = here(threadIdx.x), lane = tid & 63, n = lane & 31, h = lane >> 5;
  char* mine = lds + (tid >> 6) * PART;
  __syncthreads();  // LDS is read no more
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int c = (32 * dt + 8 * g + 4 * h) / 4;
      f32x4 o;
#pragma unroll
      for (int i = 0; i < 4; i++) o[i] = acc[dt][4 * g + i] * f;
      *(f32x4*)(mine + n * D * 4 + ((c ^ (n & 15)) << 4)) = o;
    }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32 * C / kThreads; i++) {
    const int r = (i * kThreads + tid) / C, c = (i * kThreads + tid) % C;
    const char* at = lds + r * D * 4 + ((c ^ (r & 15)) << 4);
    f32x4 o = *(const f32x4*)at;
#pragma unroll
    for (int w = 1; w < 4; w++) o += *(const f32x4*)(at + w * PART);
    if (row0 + r < S) {
      O* to = out + (row0 + r) * stride + c * 4;
      if constexpr (sizeof(O) == 2) {
        bf16x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (__bf16)o[e];
        *(bf16x4*)to = v;
        if (low) *(uint32_t*)(low + (long)(row0 + r) * D + c * 4) = low_bytes(o[0], o[1], o[2], o[3]);
      } else {
        *(f32x4*)to = o;
      }
    }
  }
}

// The head that the i-th of n = B * H work items of a row of the grid takes.  Workgroups go round
// the 8 XCDs; where n allows, each XCD gets a run of neighbouring heads, whose keys its L2 then holds.
__device__ __forceinline__ int spread(int i, int n) { return n % 8 == 0 ? (i % 8) * (n / 8) + i / 8 : i; }

template <typename T> constexpr int tile_rows() { return sizeof(T) == 2 ? 64 : 32; }

// ---- block table ---------------------------------------------------------------------------------
// A wave reduces the 64 tokens of an entry: 5 us over 4 x 4096 tokens, a launch's time.
__global__ void __launch_bounds__(256) mask_table_kernel(const int* doc, i32x4* table, int B, int S, int nb) {
  const int lane = threadIdx.x & 63;
  const long n = (long)B * nb;
  for (long w = (long)blockIdx.x * 4 + (threadIdx.x >> 6); w < n; w += (long)gridDim.x * 4) {
    const long b = w / nb;
    const int i = (int)(w % nb) * kTab + lane;
    const int d = i < S ? doc[b * S + i] : 0;
    int lo = i < S && d >= 0 ? d : 0x7fffffff, hi = i < S && d >= 0 ? d : -1;
    for (int m = 32; m; m >>= 1) {
      lo = min(lo, __shfl_xor(lo, m));
      hi = max(hi, __shfl_xor(hi, m));
    }
    const int pad = __ballot(i < S && d < 0) != 0;
    if (lane == 0) table[w] = i32x4{lo, hi, pad, 0};
  }
}

// ---- backward: the weight and its gradient of one pair ------------------------------------------------
// What a score goes through: nothing; the distance bias; the cap (and the bias, of slope 0 where none is
// given: two of some twenty instructions a pair).  Of the kernel's type, so that no pair has a branch.
enum { kPlain, kBiased, kCapped };

struct Score {
  float cs, soc, cl, slope;  // sigma log2 e, sigma / cap, cap log2 e, slope log2 e
  __device__ __forceinline__ Score(const MaskAttnArgs& a, int head)
      : cs(a.sigma * kLog2e), soc(a.sigma / a.cap), cl(a.cap * kLog2e), slope(a.slopes ? a.slopes[head] * kLog2e : 0.0f) {}
};

// Element r of sv holds the raw dot product q.k, of dpv the product dO.v; on return p and dS (without
// sigma).  distance: i - j, exact up to 2^24.
template <typename T, int KIND>
__device__ __forceinline__ void weight(const Score& c, f32x16& sv, f32x16& dpv, int r, float lse, float dsum,
                                       float distance) {
  const float s = sv[r];
  float u, g = 1.0f;
  if constexpr (KIND == kCapped) {
    const float t = cap_tanh<T>(s, c.soc);
    u = __builtin_fmaf(t, c.cl, -lse);
    g = __builtin_fmaf(-t, t, 1.0f);
  } else {
    u = __builtin_fmaf(s, c.cs, -lse);
  }
  if constexpr (KIND != kPlain) u = __builtin_fmaf(-c.slope, fabsf(distance), u);
  sv[r] = __builtin_amdgcn_exp2f(u);
  dpv[r] = sv[r] * (dpv[r] - dsum);
  if constexpr (KIND == kCapped) dpv[r] *= g;
}

// ---- rows next to non-finite values ------------------------------------------------------------------
enum { kForward, kDQ, kDKDV, kDKDVPart };

__device__ __forceinline__ float wave_sum(float x) {
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
  return x;
}

template <typename T, int D>
__device__ __forceinline__ float dot(const T* x, const T* y) {
  float s = 0.0f;
#pragma unroll 1
  for (int c = 0; c < D; c += 16 / (int)sizeof(T)) {
    const u32x4 u = *(const u32x4*)(x + c), v = *(const u32x4*)(y + c);
#pragma unroll
    for (int e = 0; e < Elem<T>::VEC; e++) s = __builtin_fmaf(element<T>(u, e), element<T>(v, e), s);
  }
  return s;
}

// One row of the result by one wave, in binary32 throughout: lanes take 64 rows of the other side for
// the scores, then columns for the sums over those of them that the row sees, and only those.  For the
// rows of a workgroup that met a non-finite value; slow (some 16 instructions a pair and wave).
template <typename T, int D, int WHAT>
__device__ __forceinline__ void careful_row(const MaskAttnArgs& a, int b, int head, int hk, int own) {
  constexpr bool KEYS = WHAT == kDKDV || WHAT == kDKDVPart;  // the row is a key
  constexpr int C = D / 64;
  const int lane = here(threadIdx.x) & 63, S = a.S;
  const int* doc = a.doc ? a.doc + (long)b * S : nullptr;
  const int prefix = a.prefix ? min(max(a.prefix[b], 0), S) : 0, w = a.window ? a.window : S;
  const T* k = (const T*)a.k + b * a.sk[0] + hk * a.sk[1];
  const T* v = (const T*)a.v + b * a.sv[0] + hk * a.sv[1];
  float m = -INFINITY, l = 0.0f, x[C] = {}, y[C] = {};  // sums: O; dQ; dK and dV
  const int heads = WHAT == kDKDV ? a.H / a.Hkv : 1;
  for (int hq = head; hq < head + heads; hq++) {
    const T* q = (const T*)a.q + b * a.sq[0] + hq * a.sq[1];
    const T* g = (const T*)a.dout + b * a.sdo[0] + hq * a.sdo[1];
    const long row0 = ((long)b * a.H + hq) * S;
    const float slope = a.slopes ? a.slopes[hq] * kLog2e : 0.0f;
    for (int base = 0; base < S; base += 64) {
      const int other = min(base + lane, S - 1), i = KEYS ? other : own, j = KEYS ? own : other;
      const int id = doc ? doc[own] : 0;
      const bool see = base + lane < S && id >= 0 && (!doc || doc[other] == id) && ((j <= i && i - j < w) || j < prefix);
      uint64_t todo = __ballot(see);
      if (todo == 0) continue;
      const float s = dot<T, D>(q + i * a.sq[2], k + j * a.sk[2]);
      float u = s * (a.sigma * kLog2e), slope_of_cap = 1.0f;
      if (a.cap > 0.0f) {
        const float t = cap_tanh<T>(s, a.sigma / a.cap);
        u = a.cap * kLog2e * t;
        slope_of_cap = __builtin_fmaf(-t, t, 1.0f);
      }
      u = __builtin_fmaf(-slope, fabsf((float)(i - j)), u);
      float p, ds = 0.0f;
      if constexpr (WHAT == kForward) {
        float top = see ? u : -INFINITY;
        for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        p = see ? __builtin_amdgcn_exp2f(u - (m == -INFINITY ? 0.0f : m)) : 0.0f;
        l = l * f + wave_sum(p);
#pragma unroll
        for (int c = 0; c < C; c++) x[c] *= f;
      } else {
        p = __builtin_amdgcn_exp2f(u - a.lse[row0 + i]);
        ds = p * (dot<T, D>(g + i * a.sdo[2], v + j * a.sv[2]) - a.dsum[row0 + i]) * slope_of_cap;
      }
      for (; todo; todo &= todo - 1) {
        const int from = __builtin_ctzll(todo), r = base + from;
        const float pr = __shfl(p, from), dr = __shfl(ds, from);
#pragma unroll
        for (int c = 0; c < C; c++) {
          const int d = lane + 64 * c;
          if constexpr (WHAT == kForward) {
            x[c] = __builtin_fmaf(pr, Elem<T>::ld(v + r * a.sv[2] + d), x[c]);
          } else if constexpr (WHAT == kDQ) {
            x[c] = __builtin_fmaf(dr, Elem<T>::ld(k + r * a.sk[2] + d), x[c]);
          } else {
            x[c] = __builtin_fmaf(dr, Elem<T>::ld(q + r * a.sq[2] + d), x[c]);
            y[c] = __builtin_fmaf(pr, Elem<T>::ld(g + r * a.sdo[2] + d), y[c]);
          }
        }
      }
    }
  }
  const long row = ((long)b * a.H + head) * S + own;
#pragma unroll
  for (int c = 0; c < C; c++) {
    const int d = lane + 64 * c;
    if constexpr (WHAT == kForward) {
      const float o = l == 0.0f ? 0.0f : x[c] / l;
      ((T*)a.out)[b * a.so[0] + head * a.so[1] + own * a.so[2] + d] = Elem<T>::put(o);
      if (a.low) a.low[row * D + d] = (signed char)(low_bits(o) >> 8);
    } else if constexpr (WHAT == kDQ) {
      ((T*)a.dq)[b * a.sdq[0] + head * a.sdq[1] + own * a.sdq[2] + d] = Elem<T>::put(x[c] * a.sigma);
    } else if constexpr (WHAT == kDKDVPart) {
      a.part[row * D + d] = x[c] * a.sigma;
      a.part[(row + (long)a.B * a.H * S) * D + d] = y[c];
    } else {
      ((T*)a.dk)[b * a.sdk[0] + hk * a.sdk[1] + own * a.sdk[2] + d] = Elem<T>::put(x[c] * a.sigma);
      ((T*)a.dv)[b * a.sdv[0] + hk * a.sdv[1] + own * a.sdv[2] + d] = Elem<T>::put(y[c]);
    }
  }
  if (WHAT == kForward && lane == 0) a.lse[row] = l == 0.0f ? 0.0f : m + __builtin_log2f(l);
}

// Whether some thread of the workgroup met a non-finite value in the item `seq`.
template <typename T>
__device__ __forceinline__ bool met_nonfinite(const Largest<T>& largest, int& lbad, int seq) {
  if (largest.nonfinite()) lbad = seq;
  __syncthreads();
  return lbad == seq;
}

// ---- forward -------------------------------------------------------------------------------------
// Tiles of 64 keys (binary32: 32) are copied one ahead into the other of two buffers, with one barrier a
// tile; two workgroups of 128 queries share a unit, so that one's softmax fills the other's products.
// Bound by the vector instructions of the softmax beside the products (a wave hides five under a matrix
// instruction): the matrix pipe is busy 0.42 of the time over 16 heads x 8192 with a bias, 0.31 over packed
// documents.  4 x 16 heads over 4 x 4096 tokens, 128 columns, bf16: 319 us, 862 TFLOP/s of visible pairs
// (a large product reaches 1209); packed in documents of 900, 152 us, 430.  TEAM: see team_of.
template <typename T, int D, int KIND, bool TEAM>
__global__ void __launch_bounds__(kThreads, TEAM || sizeof(T) * D == 512 ? 1 : 2) mask_attn_fwd_kernel(const MaskAttnArgs a) {
  using L = Tile<T, D>;
  constexpr int BN = TEAM ? 32 : tile_rows<T>(), NT = BN / 32, BM = TEAM ? 32 : 128, BYTES = BN * L::RB;
  constexpr int NB = TEAM && L::RB == 512 ? 1 : 2, SETS = TEAM ? 4 : 1;  // buffers, and sets of them
  __shared__ __align__(1024) char tiles[SETS * 2 * NB * BYTES];
  __shared__ __align__(16) int lids[SETS][2][64];
  __shared__ int lbad;
  __shared__ float lml[SETS][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int set = TEAM ? wave : 0;
  char (*lk_)[BYTES] = (char (*)[BYTES])tiles + set * 2 * NB, (*lv_)[BYTES] = lk_ + NB;
  const int S = a.S, nq = (S + BM - 1) / BM, nk = (S + BN - 1) / BN, nb = (S + kTab - 1) / kTab;
  const long total = (long)a.B * a.H * nq;
  const uint32_t row_k = L::row_base(lds_address(lk_), lane), col_v = L::col_base(lds_address(lv_), lane);
  if (threadIdx.x == 0) lbad = -1;
  int seq = 0;  // items so far: lbad names the last one that met a non-finite value

  for (long w = blockIdx.x; w < total; w += gridDim.x) {
    const int bh = spread((int)(w % (a.B * a.H)), a.B * a.H), b = bh / a.H, hq = bh % a.H, hk = hq / (a.H / a.Hkv);
    const int q0 = (nq - 1 - (int)(w / (a.B * a.H))) * BM, q1 = min(q0 + BM, S) - 1;
    const int qw0 = q0 + (TEAM ? 0 : 32 * wave), qw1 = min(qw0 + 31, S - 1), qi = qw0 + (lane & 31);
    const int* doc = a.doc ? a.doc + (long)b * S : nullptr;
    const i32x4* table = a.doc ? (const i32x4*)a.table + (long)b * nb : nullptr;
    const Band band = {S, a.window, a.prefix ? min(max(a.prefix[b], 0), S) : 0};
    const Score sc(a, hq);
    Stage<T, D, BN, TEAM> gk, gv;
    gk.init((const T*)a.k + b * a.sk[0] + hk * a.sk[1], a.sk[2]);
    gv.init((const T*)a.v + b * a.sv[0] + hk * a.sv[1], a.sv[2]);

    const Docs own = docs_of(table, q0 / kTab, q1 / kTab, nb);
    // False, with nothing written, where a tile holds a non-finite value that some row does not see.
    auto item = [&]() {
      TileIter<BN, true, TEAM> it;
      it.init(q0, q1, own, nk);
      int kb = it.next(band, table, nb, lane), buf = 0;
      Largest<T> largest;  // of cut tiles: with an infinity among them, what is formed here is not used
      auto stage = [&]() {
        gk.copy(lk_[buf], kb * BN, S);
        gv.copy(lv_[buf], kb * BN, S);
        if (doc && (TEAM || wave == 0)) copy_lanes<4>(doc, min(kb * BN + lane, S - 1) * 4, lds_address(lids[set][buf]));
      };
      arrived();  // the last item's tiles have been read, and no copy is on its way
      if (kb >= 0) stage();
      u32x4 qf[L::KS];
      load_own<T, D>(qf, (const T*)a.q + b * a.sq[0] + hq * a.sq[1], a.sq[2], min(qi, S - 1), lane);
      const int qid = doc ? doc[min(qi, S - 1)] : 0;
      f32x16 acc[L::DT] = {};
      float m = -INFINITY, l = 0.0f;

      auto advance = [&]() {
        kb = it.next(band, table, nb, lane);
        buf ^= NB - 1;
        if (kb >= 0) stage();
      };
      auto tile = [&]() {
        const char* lv = lv_[buf];
        const uint32_t ak = row_k + buf * BYTES, av = col_v + buf * BYTES;
        const int k0 = kb * BN, k1 = k0 + BN - 1;
        const bool cut = it.cut, ids = it.mixed;
        const int* lid = lids[set][buf];
        if constexpr (TEAM) arrived_here(); else arrived();
        if (NB == 2) advance();
        if (rare(cut)) gv.look(lv, largest);
        f32x16 s[NT] = {};
        Rows<T, D> kr;
        Cols<T, D> vc;
        kr.read(ak);
        fence_schedule();
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int ks = 0; ks < L::KS; ks++) {
            s[t] = mma_rows<T>(kr.f[ks], qf[ks], s[t]);
            if (t + 1 < NT)
              kr.read(ak + (t + 1) * L::SUB, ks);
            else
              read_step(vc, av, ks);
            fence_schedule();
          }
        if constexpr (KIND != kPlain) {  // to scores in units of log 2
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) s[t][r] = KIND == kCapped ? sc.cl * cap_tanh<T>(s[t][r], sc.soc) : sc.cs * s[t][r];
          if (KIND == kBiased || a.slopes) {
            const float d0 = (float)(qi - k0 - 4 * h);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
              for (int r = 0; r < 16; r++)
                s[t][r] = __builtin_fmaf(-sc.slope, fabsf(d0 - (float)(32 * t + otx_row(r, 0))), s[t][r]);
          }
        }
        if (rare(cut)) {
#pragma unroll
          for (int t = 0; t < NT; t++)
            mask_block<true>(band, ids, lid + 32 * t, k0 + 32 * t, qi, qid >= 0, qid, h,
                             [&](int r, bool drop) { s[t][r] = drop ? -INFINITY : s[t][r]; });
        }
        float top = s[0][0];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int r = 0; r < 16; r++) top = fmaxf(top, s[t][r]);
        top = max_halves(top);
        if constexpr (KIND == kPlain) top *= sc.cs;
        // The statistics move only where a maximum grows by more than 2^8: weights stay below 2^8 and
        // the sums, in binary32, lose nothing; most tiles then leave the accumulator as it is.
        if (__ballot(top > m + 8.0f)) {
          const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= f;
#pragma unroll
          for (int dt = 0; dt < L::DT; dt++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[dt][r] *= f;
        }
        const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
          for (int r = 0; r < 16; r++) {
            // binary32: the maximum's own weight is 1 to the bit (bf16 rounds it to that)
            const float u = KIND != kPlain ? s[t][r] - mu
                            : sizeof(T) == 4 ? s[t][r] * sc.cs - mu : __builtin_fmaf(s[t][r], sc.cs, -mu);
            s[t][r] = __builtin_amdgcn_exp2f(u);
            l += s[t][r];
          }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
          if (t + 1 < NT) {
            fence_schedule();
#pragma unroll
            for (int half = 0; half < 2; half++) {
              const auto b = vc.weights(s[t], half);
#pragma unroll
              for (int dt = 0; dt < L::DT; dt++) {
                vc.mma(acc, b, half, dt);
                vc.read(av + (t + 1) * L::SUB, half, dt);
                fence_schedule();
              }
            }
          } else {
            vc.mma(acc, s[t]);
          }
        }
        if constexpr (NB == 1) {
          arrived_here();
          advance();
        }
      };
      while (kb >= 0) tile();
      if (rare(met_nonfinite(largest, lbad, seq++))) return false;
      l = sum_halves(l);
      float f = 1.0f;
      if constexpr (TEAM) {
        if (h == 0) lml[wave][lane] = m, lml[wave][32 + lane] = l;
        __syncthreads();
        const int n = lane & 31;
        const float own_m = m;
        m = fmaxf(fmaxf(lml[0][n], lml[1][n]), fmaxf(lml[2][n], lml[3][n]));
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++)
          l = __builtin_fmaf(lml[i][32 + n], m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lml[i][n] - m), l);
        f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(own_m - m);
      }
      f = l == 0.0f ? 0.0f : f / l;
      if (qi < S && h == 0 && (!TEAM || wave == 0))
        a.lse[((long)b * a.H + hq) * S + qi] = l == 0.0f ? 0.0f : m + __builtin_log2f(l);
      T* out = (T*)a.out + b * a.so[0] + hq * a.so[1];
      signed char* low = a.low ? a.low + ((long)b * a.H + hq) * S * D : nullptr;
      if constexpr (TEAM)
        join_rows<T, D>(out, a.so[2], qw0, S, tiles, acc, f, low);
      else
        store_rows<T, D>(out, a.so[2], qw0, S, tiles + wave * 32 * L::RB, acc, f, low);
      return true;
    };
    if (rare(!item())) {
      for (int i = qw0 + set; i <= qw1; i += SETS) careful_row<T, D, kForward>(a, b, hq, hk, i);
    }
  }
}

// ---- backward: dQ, and D_i on the way ---------------------------------------------------------------
// As the forward, with S and dP formed from the same tiles: 4 x 16 heads over 4 x 4096 tokens 425 us, 970
// TFLOP/s; packed in documents of 900, 193 us, 500 (the matrix pipe 0.35 busy: tiles that documents cut, and
// each workgroup's own rows and results, 3 us and 2 of its 12).
template <typename T, int D, int KIND, bool TEAM>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 && !TEAM ? 2 : 1) mask_attn_dq_kernel(const MaskAttnArgs a) {
  using L = Tile<T, D>;
  constexpr int BN = TEAM ? 32 : tile_rows<T>(), NT = BN / 32, BM = TEAM ? 32 : 128, BYTES = BN * L::RB;
  constexpr int NB = TEAM && L::RB == 512 ? 1 : 2, SETS = TEAM ? 4 : 1;  // buffers, and sets of them
  __shared__ __align__(1024) char tiles[SETS * 2 * NB * BYTES];
  __shared__ __align__(16) int lids[SETS][2][64];
  __shared__ int lbad;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int set = TEAM ? wave : 0;
  char (*lk_)[BYTES] = (char (*)[BYTES])tiles + set * 2 * NB, (*lv_)[BYTES] = lk_ + NB;
  const int S = a.S, nq = (S + BM - 1) / BM, nk = (S + BN - 1) / BN, nb = (S + kTab - 1) / kTab;
  const long total = (long)a.B * a.H * nq;
  const uint32_t row_k = L::row_base(lds_address(lk_), lane), col_k = L::col_base(lds_address(lk_), lane);
  const uint32_t row_v = L::row_base(lds_address(lv_), lane);
  if (threadIdx.x == 0) lbad = -1;
  int seq = 0;

  for (long w = blockIdx.x; w < total; w += gridDim.x) {
    const int bh = spread((int)(w % (a.B * a.H)), a.B * a.H), b = bh / a.H, hq = bh % a.H, hk = hq / (a.H / a.Hkv);
    const int q0 = (nq - 1 - (int)(w / (a.B * a.H))) * BM, q1 = min(q0 + BM, S) - 1;
    const int qw0 = q0 + (TEAM ? 0 : 32 * wave), qw1 = min(qw0 + 31, S - 1), qi = qw0 + (lane & 31), qr = min(qi, S - 1);
    const int* doc = a.doc ? a.doc + (long)b * S : nullptr;
    const i32x4* table = a.doc ? (const i32x4*)a.table + (long)b * nb : nullptr;
    const Band band = {S, a.window, a.prefix ? min(max(a.prefix[b], 0), S) : 0};
    const Score sc(a, hq);
    Stage<T, D, BN, TEAM> gk, gv;
    gk.init((const T*)a.k + b * a.sk[0] + hk * a.sk[1], a.sk[2]);
    gv.init((const T*)a.v + b * a.sv[0] + hk * a.sv[1], a.sv[2]);

    const Docs own = docs_of(table, q0 / kTab, q1 / kTab, nb);
    auto item = [&]() {
      TileIter<BN, true, TEAM> it;
      it.init(q0, q1, own, nk);
      int kb = it.next(band, table, nb, lane), buf = 0;
      Largest<T> largest;  // of cut tiles: with an infinity among them, what is formed here is not used
      auto stage = [&]() {
        gk.copy(lk_[buf], kb * BN, S);
        gv.copy(lv_[buf], kb * BN, S);
        if (doc && (TEAM || wave == 0)) copy_lanes<4>(doc, min(kb * BN + lane, S - 1) * 4, lds_address(lids[set][buf]));
      };
      __syncthreads();  // the last item is done with LDS
      if (kb >= 0) stage();
      u32x4 qf[L::KS], gf[L::KS];
      load_own<T, D>(qf, (const T*)a.q + b * a.sq[0] + hq * a.sq[1], a.sq[2], qr, lane);
      load_own<T, D>(gf, (const T*)a.dout + b * a.sdo[0] + hq * a.sdo[1], a.sdo[2], qr, lane);
      const long row = ((long)b * a.H + hq) * S + qr;
      // D_i by the matrix unit, in the order of dP's own products: where a row sees one key, O_i is its v
      // and dP - D_i is 0.  The products of 32 rows with 32 rows hold it on the diagonal.
      float dsum = 0.0f;
      {
        u32x4 of[L::KS];
        load_own<T, D>(of, (const T*)a.o + b * a.so[0] + hq * a.so[1], a.so[2], qr, lane);
        f32x16 dd = {};
#pragma unroll
        for (int ks = 0; ks < L::KS; ks++) dd = mma_rows<T>(of[ks], gf[ks], dd);
        if (sizeof(T) == 2 && a.low) {
#pragma unroll
          for (int ks = 0; ks < L::KS; ks++) {
            const uint2 low = *(const uint2*)(a.low + row * D + (2 * ks + h) * 8);
            bf16x8 x;
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const float high = element<T>(of[ks], e % Elem<T>::VEC);
              x[e] = (__bf16)(with_low(high, (int)((e < 4 ? low.x : low.y) << (24 - 8 * (e & 3))) >> 24) - high);
            }
            dd = mma_rows<T>(__builtin_bit_cast(u32x4, x), gf[ks], dd);
          }
        }
#pragma unroll
        for (int r = 0; r < 16; r++) dsum = otx_row(r, 0) + 4 * h == (lane & 31) ? dd[r] : dsum;
        dsum = sum_halves(dsum);
      }
      if (qi < S && h == 0 && (!TEAM || wave == 0)) a.dsum[row] = dsum;
      const float lse = a.lse[row];
      const int qid = doc ? doc[min(qi, S - 1)] : 0;
      f32x16 acc[L::DT] = {};

      auto advance = [&]() {
        kb = it.next(band, table, nb, lane);
        buf ^= NB - 1;
        if (kb >= 0) stage();
      };
      auto tile = [&]() {
        const char* lk = lk_[buf];
        const uint32_t ak = row_k + buf * BYTES, ac = col_k + buf * BYTES, av = row_v + buf * BYTES;
        const int k0 = kb * BN, k1 = k0 + BN - 1;
        const bool cut = it.cut, ids = it.mixed;
        const int* lid = lids[set][buf];
        if constexpr (TEAM) arrived_here(); else arrived();
        if (NB == 2) advance();
        const float d0 = (float)(qi - k0 - 4 * h);
        if (rare(cut)) gk.look(lk, largest);
#pragma unroll
        for (int t = 0; t < NT; t++) {
          f32x16 s = {}, dp = {};
          Rows<T, D> kr, vr;
          Cols<T, D> kc;
          kr.read(ak + t * L::SUB);
          fence_schedule();
#pragma unroll
          for (int ks = 0; ks < L::KS; ks++) {
            s = mma_rows<T>(kr.f[ks], qf[ks], s);
            vr.read(av + t * L::SUB, ks);
          }
          fence_schedule();
#pragma unroll
          for (int ks = 0; ks < L::KS; ks++) {
            dp = mma_rows<T>(vr.f[ks], gf[ks], dp);
            read_step(kc, ac + t * L::SUB, ks);
          }
          fence_schedule();
#pragma unroll
          for (int r = 0; r < 16; r++)
            weight<T, KIND>(sc, s, dp, r, lse, dsum, d0 - (float)(32 * t + otx_row(r, 0)));
          if (rare(cut)) {
            mask_block<true>(band, ids, lid + 32 * t, k0 + 32 * t, qi, qid >= 0, qid, h,
                             [&](int r, bool drop) { dp[r] = drop ? 0.0f : dp[r]; });
          }
          kc.mma(acc, dp);
        }
        if constexpr (NB == 1) {
          arrived_here();
          advance();
        }
      };
      while (kb >= 0) tile();
      if (rare(met_nonfinite(largest, lbad, seq++))) return false;
      T* out = (T*)a.dq + b * a.sdq[0] + hq * a.sdq[1];
      if constexpr (TEAM)
        join_rows<T, D>(out, a.sdq[2], qw0, S, tiles, acc, a.sigma);
      else
        store_rows<T, D>(out, a.sdq[2], qw0, S, tiles + wave * 32 * L::RB, acc, a.sigma);
      return true;
    };
    if (rare(!item())) {
      for (int i = qw0 + set; i <= qw1; i += SETS) careful_row<T, D, kDQ>(a, b, hq, hk, i);
    }
  }
}

// ---- backward: dK and dV ----------------------------------------------------------------------------
// SPLIT: a workgroup takes one query head and writes binary32 sums to a.part, which
// mask_attn_join_kernel adds over the group; otherwise it takes the group's heads one after the other.
// A wave holds its 32 keys' k, v, dK and dV, 384 registers at 128 columns, so one wave stays on a SIMD, and
// the weights of one block of queries are formed beside the products of the other (below).  4 x 16 heads
// over 4 x 4096 tokens 690 us, 795 TFLOP/s; packed in documents of 900, split, 326 us and 49 for the join, 345
// (the matrix pipe 0.25 busy, vector instructions 0.34, waits for LDS and barriers 0.29).  Measured and not
// kept: four buffers in place of two (754 us against 704), the same interleaving for cut tiles (its masks
// spill), workgroups that stay and take sorted blocks in turn (443 us against 420 on documents).
template <typename T, int D, int KIND, bool SPLIT, bool TEAM>
__global__ void __launch_bounds__(kThreads, sizeof(T) * D == 128 && !TEAM ? 2 : 1) mask_attn_dkdv_kernel(const MaskAttnArgs a) {
  using L = Tile<T, D>;
  constexpr int BN = TEAM ? 32 : tile_rows<T>(), NT = BN / 32, BM = TEAM ? 32 : 128, BYTES = BN * L::RB;
  constexpr int NB = TEAM && L::RB == 512 ? 1 : 2, SETS = TEAM ? 4 : 1;  // buffers, and sets of them  // BM keys owned, BN queries a tile
  constexpr bool PIPELINED = NT == 2 && L::KS == 8 && L::DT == 4;
  __shared__ __align__(1024) char tiles[SETS * 2 * NB * BYTES];
  __shared__ __align__(16) float lls[SETS][2][64], lds_[SETS][2][64];
  __shared__ __align__(16) int lids[SETS][2][64];
  __shared__ int lbad;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int set = TEAM ? wave : 0;
  char (*lq_)[BYTES] = (char (*)[BYTES])tiles + set * 2 * NB, (*lg_)[BYTES] = lq_ + NB;
  const int S = a.S, nkb = (S + BM - 1) / BM, nq = (S + BN - 1) / BN, nb = (S + kTab - 1) / kTab;
  const int group = a.H / a.Hkv, heads = SPLIT ? a.H : a.Hkv;
  const long total = (long)a.B * heads * nkb;
  const uint32_t row_q = L::row_base(lds_address(lq_), lane), col_q = L::col_base(lds_address(lq_), lane);
  const uint32_t row_g = L::row_base(lds_address(lg_), lane), col_g = L::col_base(lds_address(lg_), lane);
  if (threadIdx.x == 0) lbad = -1;
  int seq = 0;

  for (long w = blockIdx.x; w < total; w += gridDim.x) {
    // the first keys have the most queries, so they come first
    const int bh = (int)(w % ((long)a.B * heads)), b = bh / heads, head = bh % heads, hk = SPLIT ? head / group : head;
    const int k0 = (int)(w / ((long)a.B * heads)) * BM, k1 = min(k0 + BM, S) - 1;
    const int kw0 = k0 + (TEAM ? 0 : 32 * wave), kw1 = min(kw0 + 31, S - 1), kj = kw0 + (lane & 31), kr = min(kj, S - 1);
    const int* doc = a.doc ? a.doc + (long)b * S : nullptr;
    const i32x4* table = a.doc ? (const i32x4*)a.table + (long)b * nb : nullptr;
    const Band band = {S, a.window, a.prefix ? min(max(a.prefix[b], 0), S) : 0};
    const Docs own = docs_of(table, k0 / kTab, k1 / kTab, nb);
    const int first = SPLIT ? head : hk * group, last = SPLIT ? first + 1 : first + group;

    auto item = [&]() {
      f32x16 dk[L::DT] = {}, dv[L::DT] = {};
      Largest<T> largest;
      int hq = first, buf = 0;  // the head whose queries are copied next
      Stage<T, D, BN, TEAM> gq, gg;
      auto take_head = [&]() {
        gq.init((const T*)a.q + b * a.sq[0] + hq * a.sq[1], a.sq[2]);
        gg.init((const T*)a.dout + b * a.sdo[0] + hq * a.sdo[1], a.sdo[2]);
      };
      TileIter<BN, false, TEAM> it;
      it.init(k0, k1, own, nq);
      int qb;
      auto seek = [&]() {  // the next tile, of this head or of the one after it
        qb = it.next(band, table, nb, lane);
        if (qb < 0 && hq + 1 < last) {  // a team has one head
          hq++;
          take_head();
          it.again();
          qb = it.next(band, table, nb, lane);
        }
      };
      auto stage = [&]() {
        gq.copy(lq_[buf], qb * BN, S);
        gg.copy(lg_[buf], qb * BN, S);
        const int i = min(qb * BN + lane, S - 1) * 4;  // 64 rows, BN of them read
        const long row0 = ((long)b * a.H + hq) * S;
        if (TEAM || wave == 0) copy_lanes<4>(a.lse + row0, i, lds_address(lls[set][buf]));
        if (TEAM || wave == 1) copy_lanes<4>(a.dsum + row0, i, lds_address(lds_[set][buf]));
        if (doc && (TEAM || wave == 2)) copy_lanes<4>(doc, i, lds_address(lids[set][buf]));
      };
      __syncthreads();  // the last item is done with LDS
      take_head();
      seek();
      if (qb >= 0) stage();
      u32x4 kf[L::KS], vf[L::KS];
      load_own<T, D>(kf, (const T*)a.k + b * a.sk[0] + hk * a.sk[1], a.sk[2], kr, lane);
      load_own<T, D>(vf, (const T*)a.v + b * a.sv[0] + hk * a.sv[1], a.sv[2], kr, lane);
      const int kid = doc ? doc[kr] : 0;

      auto advance = [&]() {
        seek();
        buf ^= NB - 1;
        if (qb >= 0) stage();
      };
      auto tile = [&](auto masks) {
      constexpr bool MASKED = decltype(masks)::value;
        const char *lq = lq_[buf], *lg = lg_[buf];
        const float *ll = lls[set][buf], *ld = lds_[set][buf];
        const uint32_t off = buf * BYTES;
        const int q0 = qb * BN, q1 = q0 + BN - 1;
        const bool cut = it.cut, ids = it.mixed;
        const int* lid = lids[set][buf];
        const Score sc(a, hq);
        const float d0 = (float)(q0 + 4 * h - kj);
        if constexpr (TEAM) arrived_here(); else arrived();
        if (NB == 2) advance();
        if (MASKED && rare(cut)) {
          gq.look(lq, largest);
          gg.look(lg, largest);
        }
        f32x16 s[NT] = {}, dp[NT] = {};
        Rows<T, D> qr, gr;
        Cols<T, D> gc, qc;
        f32x4 x[4], y[4];  // lse and D_i of a block's queries
        auto stats = [&](int t) {
#pragma unroll
          for (int g = 0; g < 4; g++) {
            x[g] = *(const f32x4*)(ll + 32 * t + 8 * g + 4 * h);
            y[g] = *(const f32x4*)(ld + 32 * t + 8 * g + 4 * h);
          }
        };
        auto scores = [&](int t, int ks) {
          s[t] = mma_rows<T>(qr.f[ks], kf[ks], s[t]);
          dp[t] = mma_rows<T>(gr.f[ks], vf[ks], dp[t]);
        };
        auto soft = [&](int t, int r) {
          weight<T, KIND>(sc, s[t], dp[t], r, x[r >> 2][r & 3], y[r >> 2][r & 3], d0 + (float)(32 * t + otx_row(r, 0)));
        };
        const uint32_t rq = row_q + off, rg = row_g + off, cq = col_q + off, cg = col_g + off;
        qr.read(rq);
        gr.read(rg);
        stats(0);
        if constexpr (!MASKED && PIPELINED) {
          // One wave per SIMD: the weights of one block are formed beside the products of the other,
          // two elements to two products, and fragments are read where others have just been used.
          fence_schedule();
#pragma unroll
          for (int i = 0; i < 8; i++) {
            scores(0, i % L::KS);
            qr.read(rq + (NT - 1) * L::SUB, i % L::KS);
            gr.read(rg + (NT - 1) * L::SUB, i % L::KS);
            fence_schedule();
          }
#pragma unroll
          for (int i = 0; i < 8; i++) {
            scores(NT - 1, i % L::KS);
            gc.read(cg, i / 4 % 2, i % L::DT);
            qc.read(cq, i / 4 % 2, i % L::DT);
            soft(0, 2 * i);
            soft(0, 2 * i + 1);
            fence_schedule();
          }
          stats(NT - 1);
          typename Cols<T, D>::W p[2] = {gc.weights(s[0], 0), gc.weights(s[0], 1)};
          typename Cols<T, D>::W d[2] = {qc.weights(dp[0], 0), qc.weights(dp[0], 1)};
          fence_schedule();
#pragma unroll
          for (int i = 0; i < 8; i++) {
            gc.mma(dv, p[i / 4 % 2], i / 4 % 2, i % L::DT);
            qc.mma(dk, d[i / 4 % 2], i / 4 % 2, i % L::DT);
            gc.read(cg + (NT - 1) * L::SUB, i / 4 % 2, i % L::DT);
            qc.read(cq + (NT - 1) * L::SUB, i / 4 % 2, i % L::DT);
            soft(NT - 1, 2 * i);
            soft(NT - 1, 2 * i + 1);
            fence_schedule();
          }
          gc.mma(dv, s[NT - 1]);
          qc.mma(dk, dp[NT - 1]);
        } else {
#pragma unroll
          for (int t = 0; t < NT; t++) {
            if (t) {
              qr.read(rq + t * L::SUB);
              gr.read(rg + t * L::SUB);
              stats(t);
            }
            fence_schedule();
#pragma unroll
            for (int ks = 0; ks < L::KS; ks++) {
              scores(t, ks);
              read_step(gc, cg + t * L::SUB, ks);
              read_step(qc, cq + t * L::SUB, ks);
            }
            fence_schedule();
#pragma unroll
            for (int r = 0; r < 16; r++) soft(t, r);
            if (MASKED && rare(cut))
              mask_block<false>(band, ids, lid + 32 * t, q0 + 32 * t, kj, kid >= 0, kid, h, [&](int r, bool drop) {
                s[t][r] = drop ? 0.0f : s[t][r];
                dp[t][r] = drop ? 0.0f : dp[t][r];
              });
            fence_schedule();
            gc.mma(dv, s[t]);
            qc.mma(dk, dp[t]);
          }
        }
        if constexpr (NB == 1) {
          arrived_here();
          advance();
        }
      };
      while (qb >= 0) {
        if constexpr (PIPELINED)
          while (qb >= 0 && !it.cut) tile(std::false_type());
        while (qb >= 0 && (it.cut || !PIPELINED)) tile(std::true_type());
      }
      if (rare(met_nonfinite(largest, lbad, seq++))) return false;
      auto put = [&](auto* dk_at, long dk_stride, auto* dv_at, long dv_stride) {
        if constexpr (TEAM) {
          join_rows<T, D>(dk_at, dk_stride, kw0, S, tiles, dk, a.sigma);
          join_rows<T, D>(dv_at, dv_stride, kw0, S, tiles, dv, 1.0f);
        } else {
          char* lds = tiles + wave * 32 * D * (int)sizeof(*dk_at);
          store_rows<T, D>(dk_at, dk_stride, kw0, S, lds, dk, a.sigma);
          store_rows<T, D>(dv_at, dv_stride, kw0, S, lds, dv, 1.0f);
        }
      };
      if constexpr (SPLIT) {
        float* p = a.part + ((long)b * a.H + first) * S * D;
        put(p, D, p + (long)a.B * a.H * S * D, D);
      } else {
        put((T*)a.dk + b * a.sdk[0] + hk * a.sdk[1], a.sdk[2], (T*)a.dv + b * a.sdv[0] + hk * a.sdv[1], a.sdv[2]);
      }
      return true;
    };
    if (rare(!item())) {
      for (int j = kw0 + set; j <= kw1; j += SETS) careful_row<T, D, SPLIT ? kDKDVPart : kDKDV>(a, b, first, hk, j);
    }
  }
}

// The sum of a group's partial dK and dV, heads ascending, four columns a thread.  Bound by memory: 4 x 16
// heads x 4096 x 128, 302 MB, 49 us, 6.2 TB/s (part of it from the last-level cache).
template <typename T, int D>
__global__ void __launch_bounds__(256) mask_attn_join_kernel(const MaskAttnArgs a) {
  const int group = a.H / a.Hkv;
  const long n = (long)a.B * a.Hkv * a.S * (D / 4), half = (long)a.B * a.H * a.S * D;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < 2 * n; i += (long)gridDim.x * 256) {
    const bool isv = i >= n;
    long e = isv ? i - n : i;
    const int d = (int)(e % (D / 4)) * 4;
    e /= D / 4;
    const int s = (int)(e % a.S);
    e /= a.S;
    const int hk = (int)(e % a.Hkv), b = (int)(e / a.Hkv);
    const float* p = a.part + (isv ? half : 0) + (((long)b * a.H + hk * group) * a.S + s) * D + d;
    float4 sum = *(const float4*)p;
    for (int g = 1; g < group; g++) {
      const float4 x = *(const float4*)(p + (long)g * a.S * D);
      sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
    }
    T* o = isv ? (T*)a.dv + b * a.sdv[0] + hk * a.sdv[1] + s * a.sdv[2] + d
               : (T*)a.dk + b * a.sdk[0] + hk * a.sdk[1] + s * a.sdk[2] + d;
    o[0] = Elem<T>::put(sum.x), o[1] = Elem<T>::put(sum.y), o[2] = Elem<T>::put(sum.z), o[3] = Elem<T>::put(sum.w);
  }
}

int grid_of(long work) { return (int)(work < (1 << 20) ? work : (1 << 20)); }

}  // namespace

// Whether dK/dV splits a group of query heads over workgroups: that evens out what the compute units get,
// which counts with few blocks, with long sequences (the first keys have the most queries) and with
// documents (of unequal lengths), and costs the partial sums.  Groups of four heads of 128 bf16 columns,
// whole and split, in us: 128 blocks of 1024 tokens 232 and 79, 256 of 1024 152 and 156, 256 of 4096 563
// and 374, 512 of 1024 201 and 327, of 4096 660 and 731; with documents of 500 tokens 541 and 385
// (in two parts, half the sums: 4 x 4096 tokens in documents of 900, 688 us a pass where four take 665 to 680).
bool mask_attn_splits(int B, int H, int Hkv, int S, bool documents) {
  const long blocks = (long)B * Hkv * ((S + 127) / 128);
  return H > Hkv && blocks < (documents ? 3 : S >= 2048 ? 2 : 1) * otx_cu_count();
}

hipError_t launch_mask_table(const int* doc, void* table, int B, int S, hipStream_t st) {
  const int nb = (S + kTab - 1) / kTab;
  mask_table_kernel<<<grid_of(((long)B * nb + 3) / 4), 256, 0, st>>>(doc, (i32x4*)table, B, S, nb);
  return hipGetLastError();
}

// Whether the work is too little for the device in blocks of 128 rows: then a team of four waves takes 32
// rows, with tiles and sums of its own in each wave.  The waves share no tile, so this moves four times
// the data a row, and pays while compute units would stand idle, and from the third tile on.  Forward, dQ
// and dK/dV in us, blocks and teams: 2 x 4 heads x 197 binary32 28, 38, 49 and 14, 19, 21; 16 heads x 512
// bf16 (64 blocks) 18, 25, 28 and 14, 18, 18; 2 heads x 8192 (128 blocks) 123, 158, 214 and 64, 76, 108;
// 16 x 2048 (256 blocks) 49, 66, 80 and 70, 85, 95; 4 x 8 x 1000 binary32 (256) 86, 125, 165 and 75, 101, 120;
// 8 heads x 64 bf16, one tile, 8, 11, 11 and 9, 11, 11.
template <typename T>
static bool team_of(int B, int heads, int S) {
  const long blocks = (long)B * heads * ((S + 127) / 128);
  return S > 2 * tile_rows<T>() && blocks * (sizeof(T) == 2 ? 2 : 1) <= otx_cu_count();
}

template <typename T, int D, int KIND>
static hipError_t fwd_of(const MaskAttnArgs& a, hipStream_t st) {
  if (team_of<T>(a.B, a.H, a.S))
    mask_attn_fwd_kernel<T, D, KIND, true><<<grid_of((long)a.B * a.H * ((a.S + 31) / 32)), kThreads, 0, st>>>(a);
  else
    mask_attn_fwd_kernel<T, D, KIND, false><<<grid_of((long)a.B * a.H * ((a.S + 127) / 128)), kThreads, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T, int D, int KIND, bool SPLIT>
static void dkdv_of(const MaskAttnArgs& a, int heads, hipStream_t st) {
  if (team_of<T>(a.B, heads, a.S))
    mask_attn_dkdv_kernel<T, D, KIND, SPLIT, true><<<grid_of((long)a.B * heads * ((a.S + 31) / 32)), kThreads, 0, st>>>(a);
  else
    mask_attn_dkdv_kernel<T, D, KIND, SPLIT, false><<<grid_of((long)a.B * heads * ((a.S + 127) / 128)), kThreads, 0, st>>>(a);
}

template <typename T, int D, int KIND>
static hipError_t bwd_of(const MaskAttnArgs& a, hipStream_t st) {
  if (team_of<T>(a.B, a.H, a.S))
    mask_attn_dq_kernel<T, D, KIND, true><<<grid_of((long)a.B * a.H * ((a.S + 31) / 32)), kThreads, 0, st>>>(a);
  else
    mask_attn_dq_kernel<T, D, KIND, false><<<grid_of((long)a.B * a.H * ((a.S + 127) / 128)), kThreads, 0, st>>>(a);
  if (a.part) {
    dkdv_of<T, D, KIND, true>(a, a.H, st);
    mask_attn_join_kernel<T, D><<<grid_of(((long)a.B * a.Hkv * a.S * (D / 2) + 255) / 256), 256, 0, st>>>(a);
  } else {
    dkdv_of<T, D, KIND, false>(a, a.Hkv, st);
  }
  return hipGetLastError();
}

hipError_t launch_mask_attn(int dtype, int D, bool backward, const MaskAttnArgs& a, hipStream_t st) {
  const int kind = a.cap > 0.0f ? kCapped : a.slopes ? kBiased : kPlain;
#define OTX_MA(T, DD, KIND) \
  if (dtype == (sizeof(T) == 2) && D == DD && kind == KIND) return backward ? bwd_of<T, DD, KIND>(a, st) : fwd_of<T, DD, KIND>(a, st);
#define OTX_MA3(T, DD) OTX_MA(T, DD, kPlain) OTX_MA(T, DD, kBiased) OTX_MA(T, DD, kCapped)
  OTX_MA3(uint16_t, 64) OTX_MA3(uint16_t, 128) OTX_MA3(float, 64) OTX_MA3(float, 128)
#undef OTX_MA3
#undef OTX_MA
  return hipErrorInvalidValue;
}

}  // namespace otx
