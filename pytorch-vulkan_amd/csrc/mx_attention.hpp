// Products of attention on gfx950 matrix instructions, shared by mx_attention.hip
// (packed sequences) and mx_attention_paged.hip (a cache).
//
// FP32 operands are taken as three bf16 pieces and multiplied as six piece products
// (mfma_core.hpp's split), so FP32's range is there without a scale, but for the numbers from
// 2^128 (1 - 2^-9) on: their first piece would be infinite, and they count as infinite.  What is
// multiplied are tiles of 32 rows (queries or keys).  v_mfma_f32_32x32x16_bf16 leaves
// lane half h of the wave with rows 8 b + 4 h + 0 .. 3 of a 32 x 32 result; row r of an
// operand therefore stands for tile_row(r), so that a lane ends with the 16 consecutive
// rows 16 h .. 16 h + 15 of one column.  Scores are computed transposed where the next
// product runs along keys (and straight where it runs along queries): a lane then holds
// 16 of what the next product runs along, two operand fragments of 8, and the
// probabilities go from accumulator to operand without leaving the lane.
#pragma once

#include <type_traits>

#include "mfma_core.hpp"
#include "mx_internal.hpp"
#include "mx_pieces.hpp"
#include "mx_sequences.hpp"

namespace mx {
namespace attn {

using mfma::bf16x8;
using mfma::f32x16;
using mfma::f32x4;
using mfma::Frag3;
using mfma::split8;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kTile = 32;
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The row of a tile that row (or column) r of a matrix operand stands for.
__device__ __forceinline__ int tile_row(int r) { return (r >> 2 & 1) << 4 | r >> 3 << 2 | (r & 3); }

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// The five small piece products, and the large one.
__device__ __forceinline__ f32x16 mma_small(const Frag3& a, const Frag3& b, f32x16 c) {
  c = mma(a.lo, b.hi, c);
  c = mma(a.hi, b.lo, c);
  c = mma(a.mid, b.mid, c);
  c = mma(a.mid, b.hi, c);
  return mma(a.hi, b.mid, c);
}
__device__ __forceinline__ f32x16 mma_large(const Frag3& a, const Frag3& b, f32x16 c) { return mma(a.hi, b.hi, c); }
__device__ __forceinline__ f32x16 mma_small(bf16x8 a, const Frag3& b, f32x16 c) { return mma(a, b.mid, mma(a, b.lo, c)); }
__device__ __forceinline__ f32x16 mma_large(bf16x8 a, const Frag3& b, f32x16 c) { return mma(a, b.hi, c); }

// Pieces of values 8 t .. 8 t + 7 of a lane's 16.
__device__ __forceinline__ Frag3 split_half(const f32x16& v, int t) {
  return t ? split8(f32x4{v[8], v[9], v[10], v[11]}, f32x4{v[12], v[13], v[14], v[15]})
           : split8(f32x4{v[0], v[1], v[2], v[3]}, f32x4{v[4], v[5], v[6], v[7]});
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// a b, 0 where either is 0: what a probability of 0 meets may be anything.
extern "C" __device__ float mx_mul_legacy(float a, float b) __asm("llvm.amdgcn.fmul.legacy");
__device__ __forceinline__ float times(float a, float b) { return mx_mul_legacy(a, b); }

// Whether the query at position i sees the key at position j.
struct Mask {
  int window, sinks;  // window 0: every earlier key
  __device__ __forceinline__ bool sees(int i, int j) const {
    return j <= i && (window == 0 || i - j < window || j < sinks);
  }
  // Every one of queries i0 .. i1 sees every one of keys j0 .. j1; none sees any of them.
  __device__ __forceinline__ bool all(int i0, int i1, int j0, int j1) const {
    return j1 <= i0 && (window == 0 || i1 - j0 < window || j1 < sinks);
  }
  __device__ __forceinline__ bool none(int i0, int i1, int j0, int j1) const {
    return j0 > i1 || (window != 0 && i0 - j1 >= window && j0 >= sinks);
  }
};

// The tiles of U keys that queries i0 .. i1 see, first those of the first tokens.
template <int U = kTile>
struct KeyTiles {
  int sinks, from, count;  // tiles 0 .. sinks - 1, then from ..; `count` in all
  __device__ __forceinline__ KeyTiles(const Mask& m, int i0, int i1) {
    from = m.window ? max(0, i0 - m.window + 1) / U : 0;
    const int end = i1 < 0 ? 0 : i1 / U + 1;
    sinks = m.window ? min((m.sinks + U - 1) / U, min(from, end)) : 0;
    count = sinks + max(0, end - from);
  }
  __device__ __forceinline__ int tile(int n) const { return n < sinks ? n : from + n - sinks; }
};

// Whether workgroups of eight waves, which share a tile between twice as many rows, are enough of
// them to even out what they have to do (else four waves).
inline bool wide_blocks(int64_t blocks) { return blocks >= cu_count() * 4; }

struct Strided {
  const float* at;
  int64_t token, head;
};

// A packed tile: [step][piece][lane], DP / 16 steps, P pieces an element (three of FP32, one of
// what is a bf16 number).
template <int DP, int P = 3>
constexpr int kTileBytes = DP / 16 * P * 1024;
// Lane l's place in a fragment: the halves' lines are exchanged in fours, so that a
// transposing read's 16 lanes, 8 bytes of four rows from both halves, meet every bank once.
__device__ __forceinline__ int slot(int lane) { return lane ^ (lane >> 5 << 2); }

// Whether all pieces of x are finite: bf16's largest number and half a step rounds up.
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < 0x1.FFp127f; }

// Elements e .. e + 7 of a row, zero from `dim` on.
__device__ __forceinline__ void load8(const float* row, int e, int dim, f32x4 (&v)[2]) {
  v[0] = v[1] = f32x4{};
  if (e + 8 <= dim) {
    v[0] = *reinterpret_cast<const f32x4u*>(row + e);
    v[1] = *reinterpret_cast<const f32x4u*>(row + e + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i < dim) v[i >> 2][i & 3] = row[e + i];
  }
}

// ------------------------------------------------- tiles in LDS, and products
__device__ __forceinline__ uint32_t lds_address(char* p) {
  return uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)p));
}

// Two tensors' tiles (and STATS times 256 bytes of statistics) in LDS, two stages.
template <int DP, int P, int WAVES, int STATS>
struct Stages {
  static constexpr int kBytes = 2 * kTileBytes<DP, P> + (STATS ? 1024 : 0);
  static constexpr int kSecond = kTileBytes<DP, P>, kStats = 2 * kTileBytes<DP, P>;
  uint32_t lds;
  __device__ __forceinline__ void load(int stage, const char* a, const char* b, const char* stats, int wave, int lane) const {
    const uint32_t to = lds + stage * kBytes;
    const char *const pa = pieces::uniform(a), *const pb = pieces::uniform(b);
    constexpr int F = DP / 16 * P;
#pragma unroll
    for (int i = 0; i < (2 * F + WAVES - 1) / WAVES; ++i) {
      const int f = wave + WAVES * i;  // a's fragments, then b's
      if (2 * F % WAVES == 0 || f < 2 * F) pieces::load_lds16(f < F ? pa + f * 1024 : pb + (f - F) * 1024, lane * 16, to + f * 1024);
    }
    load_stats(to + kStats, stats, wave, lane);
  }
  // One tensor's tile alone.
  static __device__ __forceinline__ void load_one(uint32_t to, const char* from, int wave, int lane) {
    const char* const p = pieces::uniform(from);
    constexpr int F = DP / 16 * P;
#pragma unroll
    for (int i = 0; i < (F + WAVES - 1) / WAVES; ++i) {
      const int f = wave + WAVES * i;
      if (F % WAVES == 0 || f < F) pieces::load_lds16(p + f * 1024, lane * 16, to + f * 1024);
    }
  }
  static __device__ __forceinline__ void load_stats(uint32_t to, const char* stats, int wave, int lane) {
    if (wave < STATS) load_lds4(pieces::uniform(stats) + wave * 256, lane * 4, to + wave * 256);
  }
  // 4 bytes a lane from memory to LDS (as pieces::load_lds16).
  static __device__ __forceinline__ void load_lds4(const char* base, uint32_t lane_off, uint32_t at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(at), "v"(lane_off), "s"(base) : "memory");
  }
};

// A fragment of step `step`.
template <int P>
using Frag = std::conditional_t<P == 3, Frag3, bf16x8>;
template <int P>
__device__ __forceinline__ Frag<P> frag(uint32_t tile, int step, int lane) {
  const uint32_t at = tile + step * P * 1024 + slot(lane) * 16;
  if constexpr (P == 1) return *pieces::lds_at<const bf16x8>(at);
  else return {*pieces::lds_at<const bf16x8>(at), *pieces::lds_at<const bf16x8>(at + 1024), *pieces::lds_at<const bf16x8>(at + 2048)};
}

// Rows 16 h + 8 t + 0 .. 7 (h: the lane's half) of element 32 b + l % 32, by transposing reads: 16
// lanes name 4 elements of one of 4 rows each, and get 4 rows of one element.
__device__ __forceinline__ uint32_t column_base(int lane) {
  const int c = lane & 15, g = lane >> 4 & 1, h = lane >> 5, other = c >> 1 & 1;
  return uint32_t(g * 3072 + other * 512 + (((h ^ other) << 2) + (c >> 2)) * 16 + (c & 1) * 8);
}
__device__ __forceinline__ Frag3 frag_columns(uint32_t tile_and_base, int b, int t) {
  bf16x8 f[3];
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    mfma::s16x4 q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      q[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          pieces::lds_at<mfma::s16x4>(tile_and_base + b * 6144 + p * 1024 + (2 * t + i) * 128));
    f[p] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(q[0], q[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
  return {f[0], f[1], f[2]};
}

// Exponents of scores that are not seen (a NaN among them) have no probability.  The branch is the same for a wave; the
// barrier keeps the compiler from comparing in every tile, seen as a whole or not.
template <class F>
__device__ __forceinline__ void hide(f32x16& x, F&& sees) {
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (!sees(r)) x[r] = -__builtin_inff();
}

// a b along the head's elements: a's tile in LDS, b's fragments in registers.  (One accumulator:
// over so few terms the matrix instruction's rounding towards minus infinity does not add up.)
// low(s): the smallest pieces of b's step s.
template <int P, int N, class L>
__device__ __forceinline__ f32x16 product(uint32_t a, const Frag3 (&b)[N], int lane, L&& low) {
  f32x16 acc{};
#pragma unroll
  for (int s = 0; s < N; ++s) {
    const Frag<P> f = frag<P>(a, s, lane);
    const Frag3 o{b[s].hi, b[s].mid, low(s)};
    acc = mma_large(f, o, mma_small(f, o, acc));
  }
  return acc;
}
template <int P, int N>
__device__ __forceinline__ f32x16 product(uint32_t a, const Frag3 (&b)[N], int lane) {
  return product<P>(a, b, lane, [&](int s) { return b[s].lo; });
}

// f0 and f1's products with a tile's probabilities (or their like), added up among themselves: the
// sums over tiles are taken in FP32's rounding.
template <class F>
__device__ __forceinline__ f32x16 product_halves(const F& f0, const F& f1, const Frag3 (&p)[2]) {
  f32x16 acc{};
  acc = mma_small(f0, p[0], acc);
  acc = mma_small(f1, p[1], acc);
  acc = mma_large(f0, p[0], acc);
  return mma_large(f1, p[1], acc);
}
// Block b of a p along the tile's rows: a's tile in LDS (and the lane's column_base), p's pieces.
__device__ __forceinline__ f32x16 product_columns(uint32_t a, int b, const Frag3 (&p)[2]) {
  return product_halves(frag_columns(a, b, 0), frag_columns(a, b, 1), p);
}

// Own rows as fragments in registers, straight from memory.
template <int N>
__device__ __forceinline__ void own_rows(Frag3 (&f)[N], const Strided& t, int head, int64_t row, bool live, int dim, int h,
                                         float scale) {
  const float* const at = t.at + row * t.token + head * t.head;
#pragma unroll
  for (int s = 0; s < N; ++s) {
    f32x4 v[2] = {};
    if (live) load8(at, s * 16 + h * 8, dim, v);
    f[s] = split8(v[0] * scale, v[1] * scale);
  }
}
// Stores a lane's 16 elements of block b of one row: 8 k + 4 h + 0 .. 3.
__device__ __forceinline__ void store_block(float* row, const f32x16& v, int b, int h, int dim) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e = b * 32 + 8 * k + 4 * h;
    const f32x4 four{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
    if (e + 4 <= dim) *reinterpret_cast<f32x4u*>(row + e) = four;
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e + i < dim) row[e + i] = four[i];
  }
}

}  // namespace attn
}  // namespace mx
