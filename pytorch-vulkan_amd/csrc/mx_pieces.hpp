// Products of FP32 matrices held as two fp16 pieces, on gfx950 matrix
// instructions.
//
// A value x is kept as s x = hi + 2^-r lo, hi the nearest fp16 of s x, lo the
// nearest fp16 of 2^r times what hi leaves, s a power of two chosen by the caller
// so that no entry of the matrix passes fp16's largest.  hi + lo is off by at most
// 2^-23 of x (one FP32 place) while x is within 2^-17 of the largest entry that
// s allows for, and by at most 2^-40 of that entry below it; with r = 12
// (kRaised), which keeps lo from fp16's subnormals for as long as hi, within 2^-28
// and by 2^-51.  A product is hi hi + hi lo + lo hi in FP32 accumulators, the last
// two in one of their own where lo is raised; lo lo is below 2^-22 of a term.
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
#include <type_traits>

#include "mfma_core.hpp"

namespace mx {
namespace pieces {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kBK = 16;  // columns of a slab: one step of the matrix instruction
// r of raised lo pieces: what hi leaves of entries below 2^15 is at most 2^3.
constexpr int kRaised = 12;

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

// STAGES: slabs in LDS, four or eight.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int OCC_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_, OCC = OCC_;
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int FM = BM / WM / 32, FN = BN / WN / 32;
  static constexpr int A_BYTES = 2 * BM * kBK * 2, B_BYTES = 2 * BN * kBK * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int SMEM = STAGES * STAGE;
  static constexpr int BASES = (SMEM + 65535) / 65536, PER_BASE = STAGES / BASES;  // LDS addresses, slabs that one reaches
  static constexpr int LA = A_BYTES / 1024 / WAVES, LB = B_BYTES / 1024 / WAVES;  // wave-wide loads of a slab
  static constexpr bool DUAL = FM * FN <= 4;  // hi lo and lo hi in accumulators of their own
  static_assert(LA * WAVES * 1024 == A_BYTES && LB * WAVES * 1024 == B_BYTES, "whole loads");
};

// An LDS address as the pointer that reads take.
template <class V>
__device__ __forceinline__ __attribute__((address_space(3))) V* lds_at(uint32_t at) {
  return (__attribute__((address_space(3))) V*)(uintptr_t)at;
}

// 16 bytes a lane from memory (a wave's base and each lane's offset) to LDS, at
// lds + 16 * lane.  Written out because the compiler, which cannot tell the
// slabs of a stage apart, waits for loads like these before any transposing
// read; wait_loads() and barrier() are what orders them here.  No register of
// the wave receives anything.
__device__ __forceinline__ void load_lds16(const char* base, uint32_t lane_off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(lane_off), "s"(base)
               : "memory");
}

// A pointer that is the same for a wave, in scalar registers.
__device__ __forceinline__ const char* uniform(const void* p) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(int(uint32_t(a)));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(int(uint32_t(a >> 32)));
  return reinterpret_cast<const char*>(uint64_t(hi) << 32 | lo);
}

// An operand's slabs.  ROWS: T rows of the matrix, the product running along
// its columns; LDS [plane][k / 8][T][8].  COLS: T columns, the product running
// along its rows; LDS [plane][T / 8][16][8], the rows of a group rearranged so
// that the transposing reads of 16 lanes meet every bank once.
template <int T, int LOADS, int WAVES, bool COLS>
struct Operand {
  static constexpr int PARTS = COLS ? 2 : 1;  // LDS reads of a fragment
  const char* src[LOADS];  // the wave's part of the next slab
  uint32_t lane_off;
  int64_t step;
  __device__ __forceinline__ void init(const Planes& p, int first, int slab0, int wave, int lane) {
    step = COLS ? int64_t(kBK) * 16 : int64_t(kBK / 8) * p.rows * 16;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int c = wave + i * WAVES;
      const _Float16* at;
      if constexpr (COLS) {
        constexpr int PER = T / 32;  // loads of a plane: four groups of eight columns each
        at = p.at + c / PER * p.plane + int64_t(first / 8 + 4 * (c % PER)) * p.rows * 8;
      } else {
        constexpr int PER = 2 * T / 64;  // 64 rows of a group of eight columns each
        at = p.at + c / PER * p.plane + (int64_t(c % PER / (T / 64)) * p.rows + first + c % (T / 64) * 64) * 8;
      }
      src[i] = uniform(at) + slab0 * step;
    }
    lane_off = COLS ? (uint32_t(lane >> 4) * uint32_t(p.rows) + uint32_t((lane & 15) ^ (lane >> 4 << 2))) * 16u : uint32_t(lane) * 16u;
  }
  __device__ __forceinline__ void load(uint32_t lds, int wave) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      load_lds16(src[i], lane_off, lds + uint32_t(wave + i * WAVES) * 1024u);
      src[i] += step;
    }
  }
  // Bytes from a slab's start to this lane's part of the fragment of rows
  // (columns) first .. first + 31, first a multiple of 32; COLS: half h of it.
  static __device__ __forceinline__ uint32_t lane_offset(int first, int lane, int h) {
    if constexpr (COLS) {
      const int c = lane & 15, g = first / 8 + ((lane & 16) >> 3) + ((c & 3) >> 1);
      const int k = 8 * (lane >> 5) + (c >> 2) + 4 * h;
      return uint32_t((g * 16 + (k ^ ((g & 3) << 2))) * 16 + 8 * (c & 1));
    } else {
      return uint32_t(((lane >> 5) * T + first + (lane & 31)) * 16);
    }
  }
  // The fragment of plane pl, 32 j rows (columns) on, from the LDS address of
  // this lane's parts; `off` is the slab's.
  static __device__ __forceinline__ half8 frag(const uint32_t (&at)[PARTS], int off, int pl, int j) {
    const int to = off + pl * T * kBK * 2 + j * 32 * (COLS ? 32 : 16);
    if constexpr (COLS) {
      s16x4 q[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        q[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<s16x4>(at[h] + to));
      return __builtin_bit_cast(half8, __builtin_shufflevector(q[0], q[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      return *lds_at<const half8>(at[0] + to);
    }
  }
};

template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);  // vmcnt(N) alone
}

// A barrier that orders LDS accesses without waiting for loads on their way
// there (__syncthreads waits for all of them).
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// acc[i][j] = rows (A_COLS: columns) m0 + 32 i.. of A with rows (B_COLS:
// columns) n0 + 32 j.. of B over nk slabs from slab0 (nk a multiple of four, at least four).  The matrix instruction's
// row operand is B, so that a lane ends with four consecutive columns n of one
// row m, 8 bytes of a plane (ROW_LANES: A, and it ends with four rows of one
// column, neighbours beside it).  RAISE: r of both operands' lo.
//
// Slab t's products run from registers while slab t + 1's fragments are read
// from LDS and slabs t + 2 and t + 3 come from memory, one barrier a slab.
template <class T, bool A_COLS, bool B_COLS, bool ROW_LANES = false, int RAISE = 0>
__device__ __forceinline__ void product(f32x16 (&acc)[T::FM][T::FN], const Planes& a, const Planes& b, int m0, int n0,
                                        int slab0, int nk, char* smem) {
  static_assert(RAISE == 0 || T::DUAL, "raised products need accumulators of their own");
  using OpA = Operand<T::BM, T::LA, T::WAVES, A_COLS>;
  using OpB = Operand<T::BN, T::LB, T::WAVES, B_COLS>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WN * (T::BM / T::WM), wn = wave % T::WN * (T::BN / T::WN);
  OpA oa;
  OpB ob;
  oa.init(a, m0, slab0, wave, lane);
  ob.init(b, n0, slab0, wave, lane);
#pragma unroll
  for (int i = 0; i < T::FM; ++i)
#pragma unroll
    for (int j = 0; j < T::FN; ++j) acc[i][j] = 0.f;
  f32x16 low[T::DUAL ? T::FM : 1][T::DUAL ? T::FN : 1] = {};
  const uint32_t lds = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem));
  const auto issue = [&](int stage) {
    oa.load(lds + stage * T::STAGE, wave);
    ob.load(lds + stage * T::STAGE + T::A_BYTES, wave);
  };
  half8 fa[2][2][T::FM], fb[2][2][T::FN];  // [set][plane]
  // LDS addresses of this lane's parts, one for each 64 KiB (what an
  // instruction's own offset reaches).  Opaque to the compiler, which would keep
  // an address register for every read otherwise.
  uint32_t pa[T::BASES][OpA::PARTS], pb[T::BASES][OpB::PARTS];
#pragma unroll
  for (int half = 0; half < T::BASES; ++half) {
#pragma unroll
    for (int h = 0; h < OpA::PARTS; ++h) {
      pa[half][h] = lds + half * T::PER_BASE * T::STAGE + OpA::lane_offset(wm, lane, h);
      asm volatile("" : "+v"(pa[half][h]));
    }
#pragma unroll
    for (int h = 0; h < OpB::PARTS; ++h) {
      pb[half][h] = lds + half * T::PER_BASE * T::STAGE + T::A_BYTES + OpB::lane_offset(wn, lane, h);
      asm volatile("" : "+v"(pb[half][h]));
    }
  }
  const auto read = [&](int set, int stage) {
    const int half = stage / T::PER_BASE, off = stage % T::PER_BASE * T::STAGE;
#pragma unroll
    for (int pl = 1; pl >= 0; --pl) {
#pragma unroll
      for (int j = 0; j < T::FN; ++j) fb[set][pl][j] = OpB::frag(pb[half], off, pl, j);
#pragma unroll
      for (int i = 0; i < T::FM; ++i) fa[set][pl][i] = OpA::frag(pa[half], off, pl, i);
    }
  };
  constexpr int S = T::STAGES, NL = T::LA + T::LB;
  // Slab t of stage u: its products, the next slab's reads among the first of
  // them, slab t + S - 1 on its way into the stage that slab t - 1 has left.
  const auto slab = [&](auto u_, bool more) {
    constexpr int u = decltype(u_)::value, set = u & 1;
    barrier();
    if (more) issue((u + S - 1) % S);
    read(set ^ 1, (u + 1) % S);
#pragma unroll
    for (int q = 0; q < 3; ++q)  // lo hi, hi lo, hi hi
#pragma unroll
      for (int i = 0; i < T::FM; ++i)
#pragma unroll
        for (int j = 0; j < T::FN; ++j) {
          f32x16& c = T::DUAL && q < 2 ? low[T::DUAL ? i : 0][T::DUAL ? j : 0] : acc[i][j];
          c = ROW_LANES ? __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[set][q == 1][i], fb[set][q == 0][j], c, 0, 0, 0)
                        : __builtin_amdgcn_mfma_f32_32x32x16_f16(fb[set][q == 0][j], fa[set][q == 1][i], c, 0, 0, 0);
        }
    constexpr int READS = 2 * T::FM * OpA::PARTS + 2 * T::FN * OpB::PARTS, PRODUCTS = 3 * T::FM * T::FN;
#pragma unroll
    for (int r = 0; r < (READS < PRODUCTS ? READS : PRODUCTS); ++r) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, READS < PRODUCTS ? 1 : (READS + PRODUCTS - 1) / PRODUCTS, 0);
    }
  };
  using std::integral_constant;
  // Before slab t's barrier a wave waits until its part of slab t + 1 has landed:
  // after the barrier everyone's has.
#pragma unroll
  for (int t = 0; t < S - 1; ++t)
    if (t < 4 || t < nk) issue(t);
  if (nk >= S)
    wait_loads<(S - 2) * NL>();
  else
    wait_loads<0>();
  barrier();
  read(0, 0);
  const auto four = [&](auto u_, int t) {
    constexpr int u = decltype(u_)::value;
    const auto one = [&](auto v_) {
      constexpr int v = decltype(v_)::value;
      if (t + v + S - 1 < nk) {
        wait_loads<(S - 3) * NL>();
        slab(integral_constant<int, u + v>{}, true);
      } else {
        wait_loads<0>();
        slab(integral_constant<int, u + v>{}, false);
      }
    };
    one(integral_constant<int, 0>{});
    one(integral_constant<int, 1>{});
    one(integral_constant<int, 2>{});
    one(integral_constant<int, 3>{});
  };
  if constexpr (S == 4) {
    using N1 = integral_constant<int, 1>;
    const auto all = [&](auto wait_, auto u_, bool more) {
      wait_loads<decltype(wait_)::value>();
      slab(u_, more);
    };
    using A = integral_constant<int, NL>;
    using Z = integral_constant<int, 0>;
    for (int t = 4; t < nk; t += 4) {
      all(A{}, Z{}, true);
      all(A{}, N1{}, true);
      all(A{}, integral_constant<int, 2>{}, true);
      all(A{}, integral_constant<int, 3>{}, true);
    }
    all(A{}, Z{}, true);
    all(A{}, N1{}, false);
    all(Z{}, integral_constant<int, 2>{}, false);
    all(Z{}, integral_constant<int, 3>{}, false);
  } else {
    for (int t = 0; t < nk; t += S) {
      four(integral_constant<int, 0>{}, t);
      if (t + 4 < nk) four(integral_constant<int, S - 4>{}, t + 4);
    }
  }
  if constexpr (T::DUAL) {
#pragma unroll
    for (int i = 0; i < T::FM; ++i)
#pragma unroll
      for (int j = 0; j < T::FN; ++j) acc[i][j] += RAISE ? low[i][j] * (1.f / float(1 << RAISE)) : low[i][j];
  }
}

// Lanes 4 i .. 4 i + 3 hold four values each, a 4 x 4 block by columns; returns
// it by rows.
__device__ __forceinline__ half4 transpose4(half4 v) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  const auto dpp = [](uint32_t x, auto ctrl) {
    return uint32_t(__builtin_amdgcn_mov_dpp(int(x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  using Near = std::integral_constant<int, 0xB1>;  // lane ^ 1
  using Far = std::integral_constant<int, 0x4E>;   // lane ^ 2
  const uint32_t sel = threadIdx.x & 1 ? 0x03020706u : 0x05040100u;
  const uint32_t a = __builtin_amdgcn_perm(dpp(w[0], Near{}), w[0], sel);
  const uint32_t b = __builtin_amdgcn_perm(dpp(w[1], Near{}), w[1], sel);
  const bool upper = threadIdx.x & 2;
  const uint32_t got = dpp(upper ? a : b, Far{});
  return __builtin_bit_cast(half4, upper ? u32x2{got, b} : u32x2{a, got});
}

// Element (row, col .. col + 3) of a plane, col % 4 == 0.
__device__ __forceinline__ int64_t elem(const Planes& p, int row, int col) {
  return (int64_t(col >> 3) * p.rows + row) * 8 + (col & 7);
}

// ------------------------------------------------------------- tiles to CUs
// Workgroups take whole tiles, `whole` of them; the tiles after those are taken
// by `parts` workgroups each, which leave their sums of a share of the slabs in
// `sums` for a second launch to join.
struct Shares {
  int whole, parts;
  float* sums;
};

// Tile, part and slabs [k0, k1) of a workgroup.
struct Unit {
  int tile, part, k0, k1;
};
__device__ __forceinline__ Unit unit_of(const Shares& p, int id, int nk) {
  if (id < p.whole) return {mfma::xcd_remap(id, p.whole), 0, 0, nk};
  const int part = (id - p.whole) % p.parts;
  return {p.whole + (id - p.whole) / p.parts, part, part * (nk / 4) / p.parts * 4, (part + 1) * (nk / 4) / p.parts * 4};
}

template <class T>
__device__ __forceinline__ void store_sums(const f32x16 (&acc)[T::FM][T::FN], const Shares& p, const Unit& u) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  f32x4* const to = reinterpret_cast<f32x4*>(p.sums) +
                    ((int64_t(u.tile - p.whole) * p.parts + u.part) * T::WAVES + wave) * (T::FM * T::FN * 256) + lane;
#pragma unroll
  for (int i = 0; i < T::FM; ++i)
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        to[((i * T::FN + j) * 4 + q) * 64] =
            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
}

// Fragment `id` of the joined tiles (32 x 32, workgroups of one wave): the parts in
// their order.  m and n are its place in the tile.
template <class T>
__device__ __forceinline__ f32x16 join_sums(const Shares& p, int id, int& tile, int& m, int& n) {
  constexpr int FRAGS = T::FM * T::FN, PER = T::WAVES * FRAGS;
  const int at = id / PER, wave = id % PER / FRAGS, f = id % FRAGS;
  const f32x4* from = reinterpret_cast<const f32x4*>(p.sums) +
                      ((int64_t(at) * p.parts * T::WAVES + wave) * FRAGS + f) * 256 + threadIdx.x;
  f32x4 s[4] = {};
#pragma unroll 4
  for (int q = 0; q < p.parts; ++q) {
#pragma unroll
    for (int g = 0; g < 4; ++g) s[g] += from[int64_t(q) * PER * 256 + g * 64];
  }
  f32x16 v;
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = s[e >> 2][e & 3];
  tile = p.whole + at;
  m = wave / T::WN * (T::BM / T::WM) + f / T::FN * 32;
  n = wave % T::WN * (T::BN / T::WN) + f % T::FN * 32;
  return v;
}

// 64 x 64: 4 waves of 32 x 32.  A slab is 96 cycles of a wave's products, a load
// some 1500: with one workgroup to a CU eight slabs in LDS shorten it (one
// product of 1024^3 0.18 -> 0.13 us a slab), with four of them four do as well and
// leave them room.
using Tile64Deep = Tile<64, 64, 2, 2, 8, 2>;
using Tile64 = Tile<64, 64, 2, 2, 4, 4>;
using Tile128 = Tile<128, 128, 2, 2, 4, 2>;  // 4 waves of 64 x 64
using Tile256 = Tile<256, 256, 2, 4, 4, 2>;  // 8 waves of 128 x 64

// A CU's time per slab with n workgroups of a tile on it, and how many it
// holds; microseconds, fitted to products of 16 x 1024^3 and of 4096^3.
struct TileCost {
  int tile, per_cu;
  double fixed, each;
  double slab(double n) const { return fixed + each * n; }
};
enum TileIndex { kTile64Deep, kTile64, kTile128, kTile256, kTileCount };
constexpr TileCost kTiles[kTileCount] = {{64, 2, -0.062, 0.19}, {64, 4, 0.11, 0.077}, {128, 2, 0.05, 0.285}, {256, 1, 0.0, 1.15}};

// How a product's tiles are dealt: whole rounds of the chip, then what is left
// over in parts along K where a join (a launch and a pass over the sums) costs
// less than the round that it shortens.
struct Deal {
  int64_t tiles, whole;
  int parts;
  double time;  // microseconds
  int64_t sum_bytes(int tile) const { return (tiles - whole) * parts * tile * tile * 4; }
};
inline Deal deal(const TileCost& c, int64_t tiles, int64_t nk, int64_t cu) {
  Deal d{tiles, tiles, 1, 3.0};
  const int64_t slots = cu * c.per_cu, full = tiles / slots, rest = tiles - full * slots;
  d.time += double(full * nk) * c.slab(c.per_cu);
  if (!rest) return d;
  double least = double(nk) * c.slab(double((rest + cu - 1) / cu));
  for (int64_t parts = 2; parts <= 16 && parts * rest <= slots && parts * 8 <= nk; ++parts) {
    const double share = double((nk / 4 + parts - 1) / parts * 4);
    const double split = share * c.slab(double((rest * parts + cu - 1) / cu)) + 6.0 +
                         double(rest * parts) * c.tile * c.tile * 8.0 / 3e6;
    if (split >= least) continue;
    least = split;
    d.whole = full * slots;
    d.parts = int(parts);
  }
  d.time += least;
  return d;
}

}  // namespace pieces
}  // namespace mx
