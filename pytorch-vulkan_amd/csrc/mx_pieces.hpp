// Products of FP32 matrices held as two fp16 pieces, on gfx950 matrix
// instructions.
//
// A value x is kept as s x = hi + lo, hi the nearest fp16 of s x, lo the
// nearest fp16 of what hi leaves, s a power of two chosen by the caller so that
// no entry of the matrix passes fp16's largest.  hi + lo is off by at most
// 2^-23 of x (one FP32 place) while x is within 2^-17 of the largest entry that
// s allows for, and by at most 2^-40 of that entry below it.  A product is
// hi hi + hi lo + lo hi in FP32 accumulators; lo lo is below 2^-22 of a term.
// Against six products of three bf16 pieces this halves the matrix
// instructions and two thirds of the operands' bytes, and it needs what those
// do not: a bound on the entries.
//
// In memory a matrix of R rows and C columns (padded with zeros to whole tiles)
// is two planes, hi then lo, each [C / 8][R][8]: eight consecutive columns of a
// row are the 16 bytes that a lane feeds to a matrix instruction, and
// consecutive rows lie side by side, so a tile goes from memory to LDS in
// whole lines, without passing through registers, and is read there without
// bank conflicts.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mx {
namespace pieces {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kBK = 32;  // columns of a slab

// Planes of a matrix: hi at `at`, lo `plane` elements behind.
struct Planes {
  _Float16* at;
  int64_t plane;  // elements of one plane: rows * columns, both padded
  int rows;       // padded
};

__device__ __forceinline__ void split4(const float (&v)[4], half4& hi, half4& lo) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    hi[e] = _Float16(v[e]);
    lo[e] = _Float16(v[e] - float(hi[e]));
  }
}

template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int OCC_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_, OCC = OCC_;
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int FM = BM / WM / 32, FN = BN / WN / 32;
  static constexpr int A_BYTES = 2 * BM * kBK * 2, B_BYTES = 2 * BN * kBK * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int SMEM = STAGES * STAGE;
  static constexpr int LA = A_BYTES / 1024 / WAVES, LB = B_BYTES / 1024 / WAVES;  // wave-wide loads of a slab
  static_assert(LA * WAVES * 1024 == A_BYTES && LB * WAVES * 1024 == B_BYTES, "whole loads");
};

typedef const __attribute__((address_space(1))) void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

// 16 bytes a lane from memory to LDS, at `lds` + 16 * lane (lds wave-uniform).
__device__ __forceinline__ void load_lds16(const char* src, char* lds) {
  __builtin_amdgcn_global_load_lds((gvoid*)src, (lvoid*)lds, 16, 0, 0);
}

// An operand's slabs.  ROWS: T rows of the matrix, the product running along
// its columns; LDS [plane][k / 8][T][8].  COLS: T columns, the product running
// along its rows; LDS [plane][T / 8][32][8], the rows of a group rearranged so
// that the transposing reads of 16 lanes meet every bank once.
template <int T, int LOADS, int WAVES, bool COLS>
struct Operand {
  const char* src[LOADS];  // this lane's bytes of the next slab
  int64_t step;
  __device__ __forceinline__ void init(const Planes& p, int first, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int c = wave + i * WAVES;
      const _Float16* at;
      if constexpr (COLS) {
        constexpr int PER = T / 16;  // loads of a plane: two groups of eight columns each
        const int pl = c / PER, g = 2 * (c % PER) + (lane >> 5), r = (lane & 31) ^ ((g & 3) << 2);
        at = p.at + pl * p.plane + (int64_t(first / 8 + g) * p.rows + r) * 8;
      } else {
        constexpr int PER = 4 * T / 64;  // 64 rows of a group of eight columns each
        const int pl = c / PER, kg = c % PER / (T / 64), r = c % (T / 64) * 64 + lane;
        at = p.at + pl * p.plane + (int64_t(kg) * p.rows + first + r) * 8;
      }
      src[i] = reinterpret_cast<const char*>(at);
    }
    step = COLS ? int64_t(kBK) * 16 : int64_t(kBK / 8) * p.rows * 16;
  }
  __device__ __forceinline__ void load(char* lds, int wave) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      load_lds16(src[i], lds + (wave + i * WAVES) * 1024);
      src[i] += step;
    }
  }
  // Rows (columns) first .. first + 31 at k 16 s .. 16 s + 15 of plane pl.
  static __device__ __forceinline__ half8 frag(const char* lds, int pl, int first, int s, int lane) {
    if constexpr (COLS) {
      const int c = lane & 15, g = first / 8 + ((lane & 16) >> 3) + ((c & 3) >> 1);
      s16x4 q[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = 16 * s + 8 * (lane >> 5) + (c >> 2) + 4 * h;
        const char* at = lds + pl * T * kBK * 2 + (g * 32 + (k ^ ((g & 3) << 2))) * 16 + 8 * (c & 1);
        q[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
      }
      return __builtin_bit_cast(half8, __builtin_shufflevector(q[0], q[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      return *reinterpret_cast<const half8*>(lds + pl * T * kBK * 2 + ((2 * s + (lane >> 5)) * T + first + (lane & 31)) * 16);
    }
  }
};

template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);  // vmcnt(N) alone
}

// acc[i][j] += rows m0 + 32 i.. of A with rows (COLS: columns) n0 + 32 j.. of B
// over nk slabs.  The matrix instruction's row operand is B: a lane ends with
// four consecutive columns n of one row m, 8 bytes of a plane.
template <class T, bool COLS>
__device__ __forceinline__ void product(f32x16 (&acc)[T::FM][T::FN], const Planes& a, const Planes& b, int m0, int n0,
                                        int nk, char* smem) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WN * (T::BM / T::WM), wn = wave % T::WN * (T::BN / T::WN);
  Operand<T::BM, T::LA, T::WAVES, false> oa;
  Operand<T::BN, T::LB, T::WAVES, COLS> ob;
  oa.init(a, m0, wave, lane);
  ob.init(b, n0, wave, lane);
#pragma unroll
  for (int i = 0; i < T::FM; ++i)
#pragma unroll
    for (int j = 0; j < T::FN; ++j) acc[i][j] = 0.f;
  const auto issue = [&](int t) {
    char* const st = smem + (t % T::STAGES) * T::STAGE;
    oa.load(st, wave);
    ob.load(st + T::A_BYTES, wave);
  };
#pragma unroll
  for (int t = 0; t < T::STAGES - 1; ++t)
    if (t < nk) issue(t);
  for (int t = 0; t < nk; ++t) {
    // Slab t has landed for every wave, and every wave has left slab t - 1,
    // whose stage takes slab t + STAGES - 1.
    if (t + T::STAGES - 2 < nk)
      wait_loads<(T::STAGES - 2) * (T::LA + T::LB)>();
    else
      wait_loads<0>();
    __syncthreads();
    if (t + T::STAGES - 1 < nk) issue(t + T::STAGES - 1);
    const char* const sa = smem + (t % T::STAGES) * T::STAGE;
    const char* const sb = sa + T::A_BYTES;
#pragma unroll
    for (int s = 0; s < kBK / 16; ++s) {
      half8 fa[2][T::FM], fb[2][T::FN];
#pragma unroll
      for (int j = 0; j < T::FN; ++j)
#pragma unroll
        for (int pl = 0; pl < 2; ++pl)
          fb[pl][j] = Operand<T::BN, T::LB, T::WAVES, COLS>::frag(sb, pl, wn + 32 * j, s, lane);
#pragma unroll
      for (int i = 0; i < T::FM; ++i)
#pragma unroll
        for (int pl = 0; pl < 2; ++pl)
          fa[pl][i] = Operand<T::BM, T::LA, T::WAVES, false>::frag(sa, pl, wm + 32 * i, s, lane);
#pragma unroll
      for (int i = 0; i < T::FM; ++i) {
#pragma unroll
        for (int j = 0; j < T::FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fb[1][j], fa[0][i], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < T::FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fb[0][j], fa[1][i], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < T::FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fb[0][j], fa[0][i], acc[i][j], 0, 0, 0);
      }
    }
  }
}

// Walk of a tile's results: f(m, n, v) with four consecutive columns n.. of row
// m (tile-relative).
template <class T, class F>
__device__ __forceinline__ void for_each4(const f32x16 (&acc)[T::FM][T::FN], F&& f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / T::WN * (T::BM / T::WM), wn = wave % T::WN * (T::BN / T::WN);
#pragma unroll
  for (int i = 0; i < T::FM; ++i)
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float v[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        f(wm + 32 * i + (lane & 31), wn + 32 * j + 8 * g + 4 * (lane >> 5), v);
      }
}

// Element (row, col .. col + 3) of a plane, col % 4 == 0.
__device__ __forceinline__ int64_t elem(const Planes& p, int row, int col) {
  return (int64_t(col >> 3) * p.rows + row) * 8 + (col & 7);
}

}  // namespace pieces
}  // namespace mx
