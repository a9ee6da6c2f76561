// Products of attention on gfx950 matrix instructions, shared by mx_attention.hip
// (packed sequences) and mx_attention_paged.hip (a cache).
//
// FP32 operands are taken as three bf16 pieces and multiplied as six piece products
// (mfma_core.hpp's split), so the whole range of FP32 is there without a scale.  What is
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
#include "mx_sequences.hpp"

namespace mx {
namespace attn {

using mfma::bf16x8;
using mfma::f32x16;
using mfma::f32x4;
using mfma::Frag3;
using mfma::split8;

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

}  // namespace attn
}  // namespace mx
