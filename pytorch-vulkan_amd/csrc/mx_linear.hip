// Linear layer with its bias, activation and residual in the product's
// epilogue, and its backward (FP32, contiguous).
//
//   z = x w^T + bias,  y = act(z) + residual
//   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = sum_m dz
//
// The forward is one product whose stores apply the rest.  The backward makes
// dz in one pass that sums its columns on the way (the products would otherwise
// evaluate the slope once for every tile that reads the element), then takes the
// two products of it.
//
// Four forms of the products (form_of).  Large ones run on operands packed as two
// fp16 pieces (mx_pieces.hpp): a pass over each operand finds its largest and its
// least element on the way, a second one writes the pieces, scaled by a power of two
// for the whole operand, and the products take half the matrix instructions of
// three bf16 pieces.  Where the two passes cost more than they save, the products
// are mx_gemm.hip's, or small ones without staging, or for a few tokens sums of
// vector instructions.
//
// What one scale holds: an element is off by at most 2^-23 of itself or, with raised
// lo pieces, 2^-51 of the operand's largest (both as powers of two).  An element d
// powers below that largest is therefore off by 2^(d - 51) of itself, and while no
// nonzero one of either operand is deeper than 23 + log2 k, a sum over k is off by at
// most (k / 8) 2^-24 of its terms' magnitudes by that, whatever the operands are.
// Of normal random operands with 2^24 elements and k = 1024 one in 160 has a deeper
// one.
//
// Deeper ones (the tails of GELU and SiLU have them) are lost only in sums without
// larger terms, so the second pass counts, for every row and column that a product
// takes, the elements that are within 2^-14 of the largest.  Where any two rows
// of the operands have k + 64 of them together, 64 terms at least have both, which
// is 64 2^-28 of the largest product, against at most 4 k 2^-51 that the deep
// elements are off by: (k / 8) 2^-24 of the terms again.  Rows of zeros need none.
//
// The products leave operands that neither holds for, that are not finite or whose
// largest is below 2^-100, to mx_gemm.hip's kernels, which follow on the stream and
// end at once otherwise.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "mx_activation.hpp"
#include "mx_internal.hpp"
#include "mx_pieces.hpp"

namespace mx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// What the second pass tells of an operand: its largest element's power, and by
// how many powers its least nonzero one lies below that.
struct About {
  int exponent, depth;
};
constexpr int kMisfit = 1 << 20;          // depth of an operand that no scale holds
constexpr int kLargeDepth = 14, kShared = 64;  // of the counted elements, and how many any two rows share
// A call's operands, and for each product whether it is left to mx_gemm.hip's
// kernels.
struct Head {
  About a, b, c;
  int left[2];
};

// Large elements of a row or a column: for each group of its elements (as many as a
// workgroup of the second pass holds) theirs and 1.  A row's groups of zeros add
// nothing, which tells rows of zeros (masked tokens) from others.
typedef uint32_t Large;

// Those of an operand's rows, or columns.  Each is the sum of `reps` words `len`
// apart, to which its groups add in turn, up to kAdds of them to a word (a packed
// backward of 200000 x 129 -> 129, deep operands: 747 us, all to one 817; 100000 x 256
// -> 512 561 and 592; 64 or 256 to a word the same as 128).  A list of more than kListed
// words is gone over by a launch of its own, which leaves the products kListEnds of
// them (by every workgroup of the products: 844 and 600 us).
struct Counts {
  Large* at;  // null where no product asks
  int len, reps, groups;
  Large* ends;  // of a long list
};
constexpr int kAdds = 128, kListed = 65536, kListEnds = 64;

// One operand's first pass: where `z` is not null src is dy and the values are
// dz = dy act'(z), written to dz.  Column sums to sums[part][n] where that is
// not null; with ENDS the largest magnitude (as bits: NaN counts above infinity)
// and the least one's negative (0: all are zero) of the workgroup's block to
// ends[workgroup], and the counts cleared for the second pass.
struct ScanOp {
  const float* src;
  const float* z;
  float* dz;
  float* sums;
  uint2* ends;
  Counts rows, columns;
  int64_t m;
  int n;
  int64_t rows_per;
  int col_blocks, parts;
  int first;  // first workgroup
};
struct ScanArgs {
  ScanOp op[3];
  int count, act;
};

// Largest over a wave, in lane 63, by moves within the vector unit (a shuffle
// goes through LDS).
__device__ __forceinline__ uint32_t wave_top(uint32_t v) {
  const auto with = [&](auto ctrl) {
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), decltype(ctrl)::value, 0xF, 0xF, false)));
  };
  with(std::integral_constant<int, 0x111>{});  // row_shr:1, 2, 4, 8 within 16 lanes
  with(std::integral_constant<int, 0x112>{});
  with(std::integral_constant<int, 0x114>{});
  with(std::integral_constant<int, 0x118>{});
  with(std::integral_constant<int, 0x142>{});  // row_bcast:15, 31 across them
  with(std::integral_constant<int, 0x143>{});
  return v;
}

// Sum over a wave, in lane 63, the same way.
__device__ __forceinline__ float wave_sum(float v) {
  const auto with = [&](auto ctrl) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  with(std::integral_constant<int, 0x111>{});
  with(std::integral_constant<int, 0x112>{});
  with(std::integral_constant<int, 0x114>{});
  with(std::integral_constant<int, 0x118>{});
  with(std::integral_constant<int, 0x142>{});
  with(std::integral_constant<int, 0x143>{});
  return v;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// A thread holds W columns; 64 threads lie along a row and the workgroup's four
// waves take a row each.  W == 4 for n >= 4: the last thread of a row takes its
// last four elements (it and its neighbour write the same values).  ENDS: the
// second pass follows.
template <int W, bool ENDS>
__global__ __launch_bounds__(256) void scan_kernel(ScanArgs p) {
  typedef float vec __attribute__((ext_vector_type(W)));
  typedef float vecu __attribute__((ext_vector_type(W), aligned(4)));
  __shared__ vec sums[256];
  __shared__ uint2 ends[4];
  int k = 0;
  while (k + 1 < p.count && int(blockIdx.x) >= p.op[k + 1].first) ++k;
  const ScanOp& o = p.op[k];
  const int id = blockIdx.x - o.first, bx = id % o.col_blocks, by = id / o.col_blocks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = o.n;
  const int64_t col = (int64_t(bx) * 64 + lane) * W;
  const bool in = col < n;
  const int64_t at = min(col, int64_t(n - W));
  const int64_t r0 = by * o.rows_per, r1 = min(o.m, r0 + o.rows_per);
  const float* const src = o.src;
  const float* const z = o.z;
  vec s = 0.f;
  uint32_t top = 0, low = 0;
  constexpr int ROWS = 4;  // of a wave, on their way together
  for (int64_t r = r0 + wave; r < r1; r += 4 * ROWS) {
    vec d[ROWS], t[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const bool ok = in && r + 4 * u < r1;
      d[u] = t[u] = 0.f;
      if (ok) d[u] = *reinterpret_cast<const vecu*>(src + (r + 4 * u) * n + at);
      if (ok && z) t[u] = *reinterpret_cast<const vecu*>(z + (r + 4 * u) * n + at);
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      if (z) {
#pragma unroll
        for (int e = 0; e < W; ++e) d[u][e] *= activate_slope(p.act, t[u][e]);
        if (o.dz && in && r + 4 * u < r1) *reinterpret_cast<vecu*>(o.dz + (r + 4 * u) * n + at) = d[u];
      }
      s += d[u];
      if constexpr (ENDS) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const uint32_t v = magnitude(d[u][e]);
          top = max(top, v);
          low = max(low, 0u - v);
        }
      }
    }
  }
  if constexpr (ENDS) {
    const auto clear = [](const Counts& c, int64_t i) {
      for (int rep = 0; rep < c.reps; ++rep) c.at[int64_t(rep) * c.len + i] = 0;
    };
    if (o.rows.at && bx == 0)
      for (int64_t r = r0 + threadIdx.x; r < r1; r += 256) clear(o.rows, r);
    if (o.columns.at && by == 0 && threadIdx.x < 64 * W && int64_t(bx) * 64 * W + threadIdx.x < n)
      clear(o.columns, int64_t(bx) * 64 * W + threadIdx.x);
  }
  if (!o.sums && !ENDS) return;
  sums[threadIdx.x] = s;
  if constexpr (ENDS) {
    top = wave_top(top);
    low = wave_top(low);
    if (lane == 63) ends[wave] = {top, low};
  }
  __syncthreads();
  if (wave != 0) return;
  if (o.sums && in) {
    s += sums[64 + lane];
    s += sums[128 + lane];
    s += sums[192 + lane];
    *reinterpret_cast<vecu*>(o.sums + int64_t(by) * n + at) = s;
  }
  if constexpr (ENDS) {
    if (lane == 0)
      o.ends[id] = {max(max(ends[0].x, ends[1].x), max(ends[2].x, ends[3].x)),
                    max(max(ends[0].y, ends[1].y), max(ends[2].y, ends[3].y))};
  }
}

// Second pass: the pieces of an operand [m][n], padded with zeros to
// [planes.rows] x 64 columns_of_64, times 2^(14 - e) where 2^e is its largest
// element's power.  What the products need to know of it goes to *about, and its
// large elements (of at least 1 then) are counted.
struct PackOp {
  const float* src;
  int m, n;
  pieces::Planes to;
  const uint2* ends;
  int blocks;  // of the first pass
  Counts rows, columns;
  About* about;
  int wide;   // workgroups along a row
  int first;  // first workgroup
};
struct PackArgs {
  PackOp op[3];
  int count;
  // Column sums of the first pass, by workgroups from first_sum on: 32 columns to
  // each, in column_sum_kernel's order, so that they are the same bits asked alone.
  const float* part;
  int parts, n, first_sum;
  float* out;
};

__global__ __launch_bounds__(256) void pack_kernel(PackArgs p) {
  __shared__ uint2 ends[4];
  __shared__ int found[4][32];
  if (int(blockIdx.x) >= p.first_sum) {
    __shared__ float sums[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = (int(blockIdx.x) - p.first_sum) * 32 + tx;
    float s[4] = {};
    if (c < p.n) {
#pragma unroll 4
      for (int i = ty; i < p.parts; i += 32)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (i + 8 * g < p.parts) s[g] += p.part[int64_t(i + 8 * g) * p.n + c];
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) sums[ty + 8 * g][tx] = s[g];
    __syncthreads();
    if (ty == 0 && c < p.n) {
#pragma unroll
      for (int g = 1; g < 32; ++g) s[0] += sums[g][tx];
      p.out[c] = s[0];
    }
    return;
  }
  int k = 0;
  while (k + 1 < p.count && int(blockIdx.x) >= p.op[k + 1].first) ++k;
  const PackOp& o = p.op[k];
  const int id = blockIdx.x - o.first, bx = id % o.wide, by = id / o.wide, tid = threadIdx.x;
  const int row = by * 32 + (tid & 31), col = bx * 64 + (tid >> 5) * 8;
  // This thread's eight columns of a row, on their way while the largest is found.
  float v[8] = {};
  if (row < o.m && col < o.n) {
    const float* const from = o.src + int64_t(row) * o.n + col;
    if (col + 8 <= o.n) {
      const f32x4 a = *reinterpret_cast<const f32x4u*>(from), b = *reinterpret_cast<const f32x4u*>(from + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = col + e < o.n ? from[e] : 0.f;
    }
  }
  uint32_t top = 0, low = 0;
  for (int i = tid; i < o.blocks; i += 256) {
    const uint2 e = o.ends[i];
    top = max(top, e.x);
    low = max(low, e.y);
  }
  top = wave_top(top);
  low = wave_top(low);
  if ((tid & 63) == 63) ends[tid >> 6] = {top, low};
  __syncthreads();
  top = max(max(ends[0].x, ends[1].x), max(ends[2].x, ends[3].x));
  const bool fits = top == 0 || (top < 0x7F800000u && __uint_as_float(top) >= 0x1p-100f);
  const int e = top == 0 || !fits ? 0 : int(top >> 23) - 127;
  if (id == 0 && tid == 0) {
    const uint32_t least = 0u - max(max(ends[0].y, ends[1].y), max(ends[2].y, ends[3].y));
    // A subnormal's own power is not in its bits: as the least there is.
    const int power = least < 0x00800000u ? -149 : int(least >> 23) - 127;
    *o.about = {e, top == 0 ? 0 : fits ? e - power : kMisfit};
  }
  pieces::half8 hi, lo;
  int large = 0, column = 0;
  bool some = false;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float f = ldexpf(v[q], 14 - e);
    hi[q] = _Float16(f);
    lo[q] = _Float16((f - float(hi[q])) * float(1 << pieces::kRaised));
    static_assert(kLargeDepth == 14);
    const bool is = fabsf(f) >= 1.f;
    large += is;
    some |= v[q] != 0.f;
    if (o.columns.at) {
      // Half a wave holds 32 rows of a column: their count to the half's lane q.
      const uint64_t which = __ballot(is);
      asm("v_writelane_b32 %0, %1, %2" : "+v"(column) : "s"(__popc(uint32_t(which))), "i"(q));
      asm("v_writelane_b32 %0, %1, %2" : "+v"(column) : "s"(__popc(uint32_t(which >> 32))), "i"(32 + q));
    }
  }
  const int at = col + (tid & 31);
  if (o.columns.at && (tid & 31) < 8 && at < o.n)
    atomicAdd(o.columns.at + int64_t(by % o.columns.reps) * o.n + at, Large(column) + 1);
  if (o.rows.at) {
    // The row's eight groups of eight: two to a wave.
    large |= int(some) << 16;
    large += __shfl_xor(large, 32, 64);
    if ((tid & 63) < 32) found[tid >> 6][tid & 31] = large;
    __syncthreads();
    if (tid < 32 && row < o.m) {
      large = (found[0][tid] + found[1][tid]) + (found[2][tid] + found[3][tid]);
      if (large) atomicAdd(o.rows.at + int64_t(bx % o.rows.reps) * o.m + row, Large(large & 0xFFFF) + 1);
    }
  }
  _Float16* const to = o.to.at + (int64_t(col >> 3) * o.to.rows + row) * 8;
  *reinterpret_cast<pieces::half8*>(to) = hi;
  *reinterpret_cast<pieces::half8*>(to + o.to.plane) = lo;
}

// A product of packed operands: out[m][n], whole 128-byte lines of a row to a
// half wave.  EPI: bias, activation and residual, z where it is not null.
struct PieceArgs {
  pieces::Planes a, b;
  int nk, tiles_m, tiles_n;
  pieces::Shares share;
  const About *ea, *eb;
  Counts large_a, large_b;  // of a's and b's rows (columns where the product runs along them)
  int* left;
  int m, n, k;
  float* out;
  const float *bias, *residual;
  float* z;
  int act;
};

template <bool EPI, bool WHOLE>
__device__ __forceinline__ void store_piece(const PieceArgs& p, int m, int n, const pieces::f32x16& acc, int up) {
  const int lane = threadIdx.x & 63, col = n + (lane & 31), row0 = m + 4 * (lane >> 5);
  const auto in = [&](int r) { return WHOLE || (col < p.n && row0 + r < p.m); };
  const int64_t at = int64_t(row0) * p.n + col;
  float bias = 0.f, res[16];
  if constexpr (EPI) {
    if (p.bias && (WHOLE || col < p.n)) bias = p.bias[col];
    if (p.residual) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 8 * (i >> 2) + (i & 3);
        res[i] = in(r) ? p.residual[at + int64_t(r) * p.n] : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = 8 * (i >> 2) + (i & 3);
    float v = ldexpf(acc[i], up);
    if constexpr (EPI) {
      v += bias;
      if (p.z && in(r)) p.z[at + int64_t(r) * p.n] = v;
      v = activate(p.act, v) + (p.residual ? res[i] : 0.f);
    }
    if (in(r)) p.out[at + int64_t(r) * p.n] = v;
  }
}

// A 32 x 32 fragment at row m, column n.
template <bool EPI>
__device__ __forceinline__ void finish_piece(const PieceArgs& p, int m, int n, const pieces::f32x16& acc, int up) {
  if (m + 32 <= p.m && n + 32 <= p.n)
    store_piece<EPI, true>(p, m, n, acc, up);
  else if (m < p.m && n < p.n)
    store_piece<EPI, false>(p, m, n, acc, up);
}

// Both products of a backward go in one launch: 256 tiles of each leave room for
// the other's on every CU.  The one with the longer K goes first, so that the
// launch does not end on a few long workgroups (a backward of 8192 x 4096 ->
// 512, whose dw has 128 tiles with K 8192: 375 us, in the other order 413, in two
// launches 418; of 4096 x 1024 -> 4096, both K 4096: 257, in two launches 266).
struct PieceLaunch {
  PieceArgs p[2];
  int second;    // first workgroup of the product that goes second
  bool swapped;  // p[1] goes first
};

// The least of words [first, first + step, ...) that are not zero, eight on their way
// together; negative, as in the first pass (0: there is none).
__device__ __forceinline__ uint32_t least_large(const Counts& of, int first, int step) {
  uint32_t low = 0;
  for (int i = first; i < of.len; i += 8 * step) {
    Large c[8] = {};
    for (int rep = 0; rep < of.reps; ++rep)
#pragma unroll
      for (int u = 0; u < 8; ++u) c[u] += of.at[int64_t(rep) * of.len + min(int64_t(i) + u * int64_t(step), int64_t(of.len - 1))];
#pragma unroll
    for (int u = 0; u < 8; ++u) low = max(low, 0u - c[u]);
  }
  return low;
}

// Long lists' least words, kListEnds workgroups to each.
struct ListArgs {
  Counts of[4];
};
__global__ __launch_bounds__(256) void list_kernel(ListArgs p) {
  __shared__ uint32_t low[4];
  const Counts& c = p.of[blockIdx.y];
  const uint32_t l = wave_top(least_large(c, blockIdx.x * 256 + threadIdx.x, kListEnds * 256));
  if ((threadIdx.x & 63) == 63) low[threadIdx.x >> 6] = l;
  __syncthreads();
  if (threadIdx.x == 0) c.ends[blockIdx.x] = 0u - max(max(low[0], low[1]), max(low[2], low[3]));
}

// Whether the product is left to mx_gemm.hip's kernels.
__device__ __forceinline__ bool left_out(const PieceArgs& p, const About& ea, const About& eb, char* smem) {
  const int deepest = max(ea.depth, eb.depth);
  if (deepest >= kMisfit) return true;
  if (deepest <= max(28, 23 + 31 - __clz(p.k))) return false;
  uint2* const lds = reinterpret_cast<uint2*>(smem);
  uint2 low = {least_large(p.large_a, threadIdx.x, blockDim.x), least_large(p.large_b, threadIdx.x, blockDim.x)};
  low = {wave_top(low.x), wave_top(low.y)};
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = low;
  __syncthreads();
  low = lds[0];
  for (int w = 1; w < int(blockDim.x >> 6); ++w) low = {max(low.x, lds[w].x), max(low.y, lds[w].y)};
  __syncthreads();
  // Without the groups' own; rows of zeros have nothing to cover.
  const auto count = [](uint32_t v, int groups) { return v ? max(int64_t(0u - v) - groups, int64_t(0)) : int64_t(1) << 32; };
  return count(low.x, p.large_a.groups) + count(low.y, p.large_b.groups) < int64_t(p.k) + kShared;
}

template <class T, bool A_COLS, bool B_COLS, bool EPI>
__device__ __forceinline__ void piece_tile(const PieceArgs& p, int id, char* smem) {
  const About ea = *p.ea, eb = *p.eb;
  const bool left = left_out(p, ea, eb, smem);
  if (id == 0 && threadIdx.x == 0) *p.left = left;
  if (left) return;
  const pieces::Unit unit = pieces::unit_of(p.share, id, p.nk);
  int tm, tn;
  mfma::tile_coords(unit.tile, p.tiles_m, p.tiles_n, tm, tn);
  pieces::f32x16 acc[T::FM][T::FN];
  pieces::product<T, A_COLS, B_COLS, true, pieces::kRaised>(acc, p.a, p.b, tm * T::BM, tn * T::BN, unit.k0, unit.k1 - unit.k0, smem);
  if (unit.tile >= p.share.whole) {
    pieces::store_sums<T>(acc, p.share, unit);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), up = ea.exponent + eb.exponent - 28;
  const int m0 = tm * T::BM + wave / T::WN * (T::BM / T::WM), n0 = tn * T::BN + wave % T::WN * (T::BN / T::WN);
#pragma unroll
  for (int i = 0; i < T::FM; ++i)
#pragma unroll
    for (int j = 0; j < T::FN; ++j) finish_piece<EPI>(p, m0 + 32 * i, n0 + 32 * j, acc[i][j], up);
}

template <class T>
__global__ __launch_bounds__(T::THREADS) __attribute__((amdgpu_waves_per_eu(T::OCC, T::OCC))) void piece_forward_kernel(PieceArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[T::SMEM];
  piece_tile<T, false, false, true>(p, blockIdx.x, smem);
}

// p[0]: dx = dz w, p[1]: dw = dz^T x.
template <class T>
__global__ __launch_bounds__(T::THREADS) __attribute__((amdgpu_waves_per_eu(T::OCC, T::OCC))) void piece_backward_kernel(PieceLaunch l) {
  __shared__ __attribute__((aligned(1024))) char smem[T::SMEM];
  const bool second = int(blockIdx.x) >= l.second;
  const int id = int(blockIdx.x) - (second ? l.second : 0);
  if (second == l.swapped)
    piece_tile<T, false, true, false>(l.p[0], id, smem);
  else
    piece_tile<T, true, true, false>(l.p[1], id, smem);
}

template <class T, bool EPI>
__global__ __launch_bounds__(64) void piece_join_kernel(PieceLaunch l) {
  const bool second = int(blockIdx.x) >= l.second;
  const PieceArgs& p = l.p[second ? 1 : 0];
  if (*p.left) return;
  int tile, m, n, tm, tn;
  const pieces::f32x16 v = pieces::join_sums<T>(p.share, int(blockIdx.x) - (second ? l.second : 0), tile, m, n);
  mfma::tile_coords(tile, p.tiles_m, p.tiles_n, tm, tn);
  finish_piece<EPI>(p, tm * T::BM + m, tn * T::BN + n, v, p.ea->exponent + p.eb->exponent - 28);
}

constexpr int kFewRows = 4, kFewTokens = 4;  // of w to a workgroup, of x at most

// A few tokens, `groups` of M.  A workgroup takes a group and R rows of w and splits
// k between its four waves, lane after lane along it; a wave's partial sums meet in
// LDS.  A weight is 16 bytes to a lane, all rows of a stretch on their way together.
// One group is bound by reading the weights (4 x 1024 -> 4096: 4.2 us, 4096 -> 16384
// for one token 44 us, 6.0 TB/s).  More groups take the same rows on the same XCD
// one after another, so that all but the first find them in its L2: 16 x 4096 ->
// 1024 8.3 us, where all tokens to a workgroup took 14.1 (M = 8: 7.6, but 5.9
// against 5.8 for 8 x 1024 -> 4096 and 9.0 against 7.5 for 12).
template <int M>
__global__ __launch_bounds__(256) void few_kernel(const float* x, const float* w, const float* bias, const float* residual,
                                                  int tokens, int groups, int64_t k, int n, int act, float* y, float* z) {
  constexpr int R = kFewRows;
  __shared__ float sums[4][M * R];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int turn = int(blockIdx.x) / 8, group = turn % groups, first = group * M, m = min(M, tokens - first);
  const int64_t n0 = (int64_t(turn / groups) * 8 + int(blockIdx.x) % 8) * R;
  if (n0 >= n) return;
  x += int64_t(first) * k;
  float acc[M][R] = {};
  for (int64_t k0 = wave * 256; k0 < k; k0 += 1024) {
    // The lane that k ends in takes its last four elements and leaves out those
    // that its neighbour has.
    const int64_t kk = k0 + lane * 4, at = min(kk, k - 4);
    const int skip = kk < k ? int(kk - at) : 4;
    f32x4 wv[R], xv[M];
#pragma unroll
    for (int r = 0; r < R; ++r) wv[r] = *reinterpret_cast<const f32x4u*>(w + min(n0 + r, int64_t(n - 1)) * k + at);
#pragma unroll
    for (int i = 0; i < M; ++i) xv[i] = *reinterpret_cast<const f32x4u*>(x + int64_t(min(i, m - 1)) * k + at);
    if (skip) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e >= skip) continue;
#pragma unroll
        for (int r = 0; r < R; ++r) wv[r][e] = 0.f;
#pragma unroll
        for (int i = 0; i < M; ++i) xv[i][e] = 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < M; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[i][r] = fmaf(xv[i][e], wv[r][e], acc[i][r]);
  }
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float s = wave_sum(acc[i][r]);
      if (lane == 63) sums[wave][i * R + r] = s;
    }
  __syncthreads();
  const int t = threadIdx.x;
  if (t >= M * R) return;
  const int i = t / R;
  const int64_t col = n0 + t % R;
  if (i >= m || col >= n) return;
  float v = ((sums[0][t] + sums[1][t]) + (sums[2][t] + sums[3][t])) + (bias ? bias[col] : 0.f);
  const int64_t to = int64_t(first + i) * n + col;
  if (z) z[to] = v;
  v = activate(act, v);
  y[to] = v + (residual ? residual[to] : 0.f);
}

// ------------------------------------------------------------ small products
// out[M][N] = sum_k a[m][k] b[n][k] for products whose time is latency: 32 x 32
// outputs to a wave, whose lanes read their eight k of a row straight from memory
// into registers, four steps of 16 k ahead, and split them there into three bf16
// pieces (the arithmetic of mx_gemm.hip's tiles).  No LDS and no barrier until the
// WK waves of a workgroup, which share K where it is long enough, join their sums
// (WK == 1: a tile to each of its four waves).  Values past tiles' edges are read
// twice and not stored.
//
// A backward's two products go in one launch, and the tiles of dw's first column
// sum their rows of dz into db.  (With dz evaluated from dy and z as it is read,
// every tile of a row over again, a step took three times as long.)
struct DirectProduct {
  const float *a, *b;
  float *out, *row_sums;
  int m, n, k;
  int64_t a_stride, b_stride;  // of a row where k is contiguous, else of k
  bool a_along;                // a's k is contiguous (b's too in a forward)
  int tiles_n, first;          // first tile
};
struct DirectArgs {
  DirectProduct p[2];
  int count, tiles, act;
  const float *bias, *residual;
  float* z;
};

constexpr int kAhead = 4;

// A lane's row of an operand.  ALONG: k contiguous.
template <bool ALONG>
struct DirectRow {
  const float* p;
  int64_t stride;
  int k;
  __device__ __forceinline__ DirectRow(const float* base, int64_t stride_, int row, int k_)
      : p(base + (ALONG ? row * stride_ : int64_t(row))), stride(stride_), k(k_) {}
  // Eight k from k0, zeros past K; whole: none of the wave's 16 is past it.
  __device__ __forceinline__ void read(float (&v)[8], int k0, bool whole) const {
    if constexpr (ALONG) {
      if (whole) {
        const f32x4 a = *reinterpret_cast<const f32x4u*>(p + k0), b = *reinterpret_cast<const f32x4u*>(p + k0 + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = a[e];
          v[4 + e] = b[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k0 + e < k ? p[k0 + e] : 0.f;
      }
    } else {
      const float* const at = p + int64_t(k0) * stride;
      if (whole) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = at[e * stride];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k0 + e < k ? at[e * stride] : 0.f;
      }
    }
  }
};

struct DirectRegs {
  float a[8], b[8];
};

// acc (times the returned factor) = steps [s0, s1) of a tile's product; sum: this
// lane's part of its row of a.
template <bool A_ALONG, bool B_ALONG>
__device__ __forceinline__ float direct_product(const DirectProduct& p, int row, int col, int s0, int s1,
                                                mfma::f32x16& acc, float& sum) {
  const int lane = threadIdx.x & 63, half = 8 * (lane >> 5);
  const DirectRow<A_ALONG> ra(p.a, p.a_stride, min(row + (lane & 31), p.m - 1), p.k);
  const DirectRow<B_ALONG> rb(p.b, p.b_stride, min(col + (lane & 31), p.n - 1), p.k);
  const auto load = [&](DirectRegs& g, int s) {
    if (s >= s1) return;
    const bool whole = 16 * s + 16 <= p.k;
    ra.read(g.a, 16 * s + half, whole);
    rb.read(g.b, 16 * s + half, whole);
  };
  DirectRegs g[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) load(g[u], s0 + u);
  acc = 0.f;
  sum = 0.f;
  const auto quads = [](const float (&v)[8]) {
    const float f = mfma::kPieceScale;
    return mfma::split8(mfma::f32x4{v[0] * f, v[1] * f, v[2] * f, v[3] * f}, mfma::f32x4{v[4] * f, v[5] * f, v[6] * f, v[7] * f});
  };
  for (int s = s0; s < s1; s += kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (s + u >= s1) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += g[u].a[e];
      const mfma::Frag3 a = quads(g[u].a), b = quads(g[u].b);
      load(g[u], s + u + kAhead);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.lo, b.hi, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.lo, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b.mid, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b.hi, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.mid, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.hi, acc, 0, 0, 0);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(acc[e]) << 1);
  if (!__any(top >= 0xFF000000u)) return mfma::kProductScale;
  // Pieces cannot hold an operand or a sum: again on the FP32 instruction.
  acc = 0.f;
  for (int s = s0; s < s1; ++s) {
    load(g[0], s);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(g[0].a[e], g[0].b[e], acc, 0, 0, 0);
  }
  return 1.f;
}

template <bool FORWARD, int WK>
__global__ __launch_bounds__(WK > 1 ? 64 * WK : 256) void direct_kernel(DirectArgs d) {
  __shared__ float sums[WK > 1 ? WK * 1024 : 1], rows[WK > 1 ? WK * 32 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tile = WK > 1 ? int(blockIdx.x) : int(blockIdx.x) * 4 + wave;
  if (tile >= d.tiles) return;  // whole workgroups where waves meet at barriers
  const DirectProduct& p = d.p[!FORWARD && d.count > 1 && tile >= d.p[1].first ? 1 : 0];
  tile -= p.first;
  const int row = tile / p.tiles_n * 32, col = tile % p.tiles_n * 32;
  const int steps = (p.k + 15) / 16, s0 = WK > 1 ? wave * steps / WK : 0, s1 = WK > 1 ? (wave + 1) * steps / WK : steps;
  mfma::f32x16 acc;
  float sum, scale;
  if constexpr (FORWARD)
    scale = direct_product<true, true>(p, row, col, s0, s1, acc, sum);
  else if (p.a_along)
    scale = direct_product<true, false>(p, row, col, s0, s1, acc, sum);
  else
    scale = direct_product<false, false>(p, row, col, s0, s1, acc, sum);
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] *= scale;
  // Both halves of a wave hold half of a row's k.
  const bool want_rows = !FORWARD && p.row_sums && col == 0;
  if (want_rows) sum += __shfl_xor(sum, 32, 64);
  constexpr int MINE = WK > 1 ? 16 / WK : 16;  // this wave's registers of the joined tile
  float v[MINE];
  const int e0 = WK > 1 ? MINE * wave : 0;
  if constexpr (WK > 1) {
#pragma unroll
    for (int e = 0; e < 16; ++e) sums[(wave * 16 + e) * 64 + lane] = acc[e];
    if (want_rows && lane < 32) rows[wave * 32 + lane] = sum;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < MINE; ++q) {
      const float* const at = sums + (e0 + q) * 64 + lane;
      v[q] = at[0];
#pragma unroll
      for (int w = 1; w < WK; ++w) v[q] += at[w * 1024];
    }
    if (want_rows && wave == 0 && lane < 32) {
      sum = rows[lane];
#pragma unroll
      for (int w = 1; w < WK; ++w) sum += rows[w * 32 + lane];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = acc[e];
  }
  if (want_rows && (WK == 1 || wave == 0) && lane < 32 && row + lane < p.m) p.row_sums[row + lane] = sum;
  const int c = col + (lane & 31);
  if (c >= p.n || !p.out) return;
  const float bias = FORWARD && d.bias ? d.bias[c] : 0.f;
#pragma unroll
  for (int q = 0; q < MINE; ++q) {
    const int e = e0 + q, r = row + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
    if (r >= p.m) continue;
    const int64_t to = int64_t(r) * p.n + c;
    float o = v[q];
    if constexpr (FORWARD) {
      o += bias;
      if (d.z) d.z[to] = o;
      o = activate(d.act, o) + (d.residual ? d.residual[to] : 0.f);
    }
    p.out[to] = o;
  }
}

// out[c] = sum of part[p][c]: 32 columns to a workgroup, and 32 groups of partials
// (every 32nd p), each summed in the order of p and then group after group.
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* part, int parts, int n, float* out) {
  __shared__ float sum[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t at = int64_t(blockIdx.x) * 32 + tx;
  float s = 0.f;
  if (at < n) {
#pragma unroll 8
    for (int p = ty; p < parts; p += 32) s += part[int64_t(p) * n + at];
  }
  sum[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && at < n) {
#pragma unroll
    for (int g = 1; g < 32; ++g) s += sum[g][tx];
    out[at] = s;
  }
}

__global__ void zero_kernel(float* out, int64_t n) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) out[i] = 0.f;
}

int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

// Row ranges of the first pass: enough workgroups to fill the chip without
// splitting a range below 16 rows.
struct ScanPlan {
  int64_t rows_per;
  int parts, col_blocks;
  int blocks() const { return parts * col_blocks; }
};
ScanPlan plan_scan(int64_t m, int64_t n) {
  ScanPlan p{};
  const int w = n >= 4 ? 4 : 1;
  p.col_blocks = int((n + 64 * w - 1) / (64 * w));
  const int64_t want = std::max<int64_t>(1, int64_t(cu_count()) * 8 / p.col_blocks);
  p.rows_per = std::max<int64_t>(16, (m + want - 1) / want);
  p.parts = int((m + p.rows_per - 1) / p.rows_per);
  return p;
}

mx_gemm_desc product(int64_t m, int64_t n, int64_t k, int64_t am, int64_t ak, int64_t bk, int64_t bn) {
  mx_gemm_desc d{};
  d.batch = 1;
  d.m = m;
  d.n = n;
  d.k = k;
  d.a_stride_m = am;
  d.a_stride_k = ak;
  d.b_stride_k = bk;
  d.b_stride_n = bn;
  d.ldc = n;
  d.alpha = 1.f;
  return d;
}

mx_gemm_desc forward_desc(int64_t m, int64_t k, int64_t n, bool bias) {
  mx_gemm_desc d = product(m, n, k, k, 1, 1, k);
  d.beta = 1.f;
  d.bias_kind = bias ? MX_BIAS_COL : MX_BIAS_NONE;
  d.bias_stride_n = 1;
  return d;
}
mx_gemm_desc dx_desc(int64_t m, int64_t k, int64_t n) { return product(m, k, n, n, 1, k, 1); }
mx_gemm_desc dw_desc(int64_t m, int64_t k, int64_t n) { return product(n, k, m, 1, n, k, 1); }

// Most scratch that the products' K splits may take.
constexpr int64_t kPartials = int64_t(64) << 20;

// Scratch of one product, whatever its operands' alignment.
int partials(const mx_gemm_desc& d, int64_t* bytes) {
  std::string name;
  int64_t a = 0, b = 0;
  MX_TRY(gemm_describe(&d, reinterpret_cast<const float*>(256), reinterpret_cast<const float*>(256), kPartials, &name, &a));
  MX_TRY(gemm_describe(&d, reinterpret_cast<const float*>(260), reinterpret_cast<const float*>(260), kPartials, &name, &b));
  *bytes = up256(std::max(a, b));
  return MX_OK;
}

int check(const char* who, int64_t m, int64_t k, int64_t n, int act) {
  MX_REQUIRE(m >= 0 && k >= 0 && n >= 0, MX_ERR_INVALID, who, ": negative size");
  MX_REQUIRE(m <= INT32_MAX && k <= INT32_MAX && n <= INT32_MAX, MX_ERR_INVALID, who, ": size exceeds int32");
  MX_REQUIRE(act >= MX_ACT_NONE && act <= MX_ACT_GELU_TANH, MX_ERR_INVALID, who, ": unknown activation ", act);
  return MX_OK;
}

// Carves a workspace (or, with a null base, adds up what it takes).
struct Carve {
  char* base;
  int64_t used = 0;
  explicit Carve(void* p) : base(static_cast<char*>(p)) {}
  template <class T>
  T* take(int64_t count) {
    T* const at = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += up256(count * int64_t(sizeof(T)));
    return at;
  }
};

// ------------------------------------------------------------ packed products
// Products of packed operands run on 128 x 128 tiles, two workgroups to a CU, so
// that one's stores and activations go on beside the other's products (4096 x
// 1024 -> 4096 with GELU: 113 us, on 256 x 256 tiles 103 to 116; a lone
// product without an epilogue 90 and 87: not worth kernels of their own).
using PieceTile = pieces::Tile128;
constexpr int kPad = PieceTile::BM;
int64_t padded(int64_t v) { return (v + kPad - 1) / kPad * kPad; }
double piece_work(int64_t m, int64_t n, int64_t k) { return double(padded(m) / kPad * (padded(n) / kPad)) * double(padded(k)); }
// share: the part of the chip that the product has, the rest beside it another's.
pieces::Deal plan_piece(int64_t m, int64_t n, int64_t k, double share) {
  return pieces::deal(pieces::kTiles[pieces::kTile128], padded(m) / kPad * (padded(n) / kPad), padded(k) / pieces::kBK,
                      std::max<int64_t>(1, int64_t(double(cu_count()) * share)));
}

// An operand [m][n] of packed products: what its passes write.
struct Packed {
  int64_t m, n;
  ScanPlan scan;
  ScanOp first;
  PackOp second;
};

Counts counts_of(int64_t len, int64_t groups, Carve* c) {
  Counts o{};
  o.len = int(len);
  o.groups = int(groups);
  o.reps = int(std::clamp<int64_t>(len > kListed ? 16 : kListed / len, 1, (groups + kAdds - 1) / kAdds));
  o.at = c->take<Large>(len * o.reps);
  if (len > kListed) o.ends = c->take<Large>(kListEnds);
  return o;
}

// by_rows, by_cols: products run along its rows, its columns.
Packed packed(int64_t m, int64_t n, bool by_rows, bool by_cols, Carve* c) {
  Packed o{};
  o.m = m;
  o.n = n;
  o.scan = plan_scan(m, n);
  const int64_t mp = padded(m), np = padded(n);
  o.first.m = m;
  o.first.n = int(n);
  o.first.rows_per = o.scan.rows_per;
  o.first.col_blocks = o.scan.col_blocks;
  o.first.parts = o.scan.parts;
  o.first.ends = c->take<uint2>(o.scan.blocks());
  if (by_rows) o.first.rows = counts_of(m, np / 64, c);
  if (by_cols) o.first.columns = counts_of(n, mp / 32, c);
  o.second.m = int(m);
  o.second.n = int(n);
  o.second.to = {c->take<_Float16>(2 * mp * np), mp * np, int(mp)};
  o.second.ends = o.first.ends;
  o.second.blocks = o.scan.blocks();
  o.second.rows = o.first.rows;
  o.second.columns = o.first.columns;
  o.second.wide = int(np / 64);
  return o;
}

// Most that a call's packed operands (and dz with them) may take: 3 % of the card's
// memory.
constexpr double kMostPacked = 8.0 * (int64_t(1) << 30);

// How a call's products run: as mx_gemm.hip's tiles, as small ones without
// staging, on packed operands, or (a forward) as a few tokens.
enum class Form { kTiles, kSmall, kPacked, kFew };

// The form whose time is least, each as fitted to measurements of 113 shapes from
// 17 to 8192 rows and 48 to 4096 columns (which take 1.6 % longer so than with the
// best form of each), packed ones on the sizes that they are padded to: of 37 backward
// shapes, tall and narrow ones among them, the choice takes 1.3 % longer than the
// best, 23 % at most (30000 x 384 -> 384 200 us packed, 162 in tiles); on their own
// sizes 6.8 %, and 200000 x 129 -> 129, padded to 256, ran for 747 us, in tiles for 405.
// Microseconds, tiles / small / packed, with GELU:
//   m x k -> n            forward              backward
//   17 x 512 -> 512       15 /   7 /  -         25 /  11 /  -
//   512 x 512 -> 512      16 /   8 /  -         36 /  16 /  -
//   700 x 700 -> 700      17 /  15 /  29        42 /  32 /  34
//   64 x 4096 -> 4096     27 /  38 /  80        60 /  79 /  88
//   8192 x 256 -> 1024    42 /  94 /  46       103 / 135 /  96
//   1024 x 1024 -> 1024   30 /  35 /  42        65 /  59 /  40
//   601 x 803 -> 1205     30 /  23 /  42        60 /  46 /  39   (rows not 16-byte aligned)
//   1000 x 701 -> 1999    39 /  62 /  46        96 /  88 /  52   (the same)
//   256 x 4096 -> 4096    62 / 118 /  97       123 / 201 / 117
//   2048 x 2048 -> 2048  114 / 229 /  82       228 / 370 / 133
//   8192 x 4096 -> 512   203 / 455 / 204       395 / 752 / 395
//   4096 x 1024 -> 4096  203 /   - / 128       438 /   - / 268
// and a forward of few tokens, best of the others / few:
//   m                     4           8           16          32          48
//   64 -> 2000            3.7 / 3.5   3.9 / 3.6   4.0 / 4.7   4.2 / 7.2   4.2 / 9.6
//   3000 -> 300           11 / 4.1    11 / 4.2    11 / 4.6    12 / 5.6    12 / 6.7
//   1024 -> 4096          9.7 / 4.2   10 / 5.8    11 / 9.1    12 / 15     12 / 22
//   4096 -> 1024          13 / 5.2    14 / 5.5    14 / 8.3    15 / 12     15 / 17
//   4096 -> 4096          23 / 12     24 / 14     24 / 21     25 / 38     26 / 58
// Tiles and small products pay for odd rows, small ones by a CU's share of
// workgroups (a step of 16 k takes four waves 0.45 us), packed ones for two
// passes over each operand, few tokens for every group's pass over the weights.
Form form_of(int64_t m, int64_t k, int64_t n, bool backward) {
  const auto up = [](int64_t v, int64_t to) { return double((v + to - 1) / to); };
  const double out = 1e-6 * double(m) * double(n), sides = 1e-6 * double(k) * double(m + n), cu = cu_count();
  const double gflop = (backward ? 4e-3 : 2e-3) * out * double(k);
  const bool odd = k % 4 || (backward && n % 4);
  // Packed operands are padded: 129 columns take 256.
  const double mp = double(padded(m)), kp = double(padded(k)), np = double(padded(n));
  const double out_p = 1e-6 * mp * np, sides_p = 1e-6 * kp * (mp + np), gflop_p = (backward ? 4e-3 : 2e-3) * out_p * kp;
  double tiles, small, packed;
  if (backward) {
    const double workgroups = up(m, 32) * up(k, 32) * up(n, 64) + up(n, 32) * up(k, 32) * up(m, 64);
    tiles = std::min(19.0 + 0.45 * up(std::min(m, n), 16), 32.0) + (odd ? 10.0 : 5.0) * gflop + 3.5 * out + 1.4 * sides;
    small = 9.5 + (odd ? 0.44 : 0.34) * std::max(up(std::max(m, n), 64), workgroups / cu) + 6.5 * out + 2.4 * sides;
    packed = 25.0 + 1.8 * gflop_p + 3.4 * sides_p + 5.0 * out_p;
  } else {
    tiles = std::min(6.0 + 0.23 * up(k, 16), 11.0) + (odd ? 10.8 : 5.7) * gflop + out + 0.7 * sides;
    small = 3.8 + (odd ? 0.165 : 0.11) * up(k, 16) * std::max(1.0, up(m, 32) * up(n, 32) / cu) + 3.4 * out;
    packed = 26.5 + 2.0 * gflop_p + 2.7 * sides_p + 1.6 * out_p;
  }
  const double scratch = 4e6 * (sides_p + (backward ? out_p + out : 0.0));
  if (std::min({m, k, n}) < 4 || scratch > kMostPacked) packed = INFINITY;
  double few = INFINITY;
  const double groups = up(m, kFewTokens), turns = groups * up(n, kFewRows);
  if (!backward && m <= 64 && k >= 4 && turns <= 1 << 20)  // as measured, and what a grid holds
    few = 2.7 + 3e-4 * double(k) + 0.05 * sides + 1e-3 * turns * (0.83 + 7.5e-4 * double(k));
  const double least = std::min({tiles, small, packed, few});
  return least == few ? Form::kFew : least == packed ? Form::kPacked : least == small ? Form::kSmall : Form::kTiles;
}

// out [m][n] over k: operands a (its rows, or where a_cols its columns, are m) and
// b, dealt as d.
void fill_piece(PieceArgs* p, const pieces::Deal& d, const Packed& a, bool a_cols, const Packed& b, bool b_cols,
                int* left, float* sums) {
  p->a = a.second.to;
  p->b = b.second.to;
  p->ea = a.second.about;
  p->eb = b.second.about;
  const auto listed = [](const Counts& c) { return c.ends ? Counts{c.ends, kListEnds, 1, c.groups, nullptr} : c; };
  p->large_a = listed(a_cols ? a.second.columns : a.second.rows);
  p->large_b = listed(b_cols ? b.second.columns : b.second.rows);
  p->left = left;
  p->m = int(a_cols ? a.n : a.m);
  p->n = int(b_cols ? b.n : b.m);
  p->k = int(a_cols ? a.m : a.n);
  p->nk = int(padded(p->k) / pieces::kBK);
  p->tiles_m = int(padded(p->m) / kPad);
  p->tiles_n = int(padded(p->n) / kPad);
  p->share = {int(d.whole), d.parts, sums};
}
int piece_blocks(const PieceArgs& p) {
  return p.share.whole + (p.tiles_m * p.tiles_n - p.share.whole) * p.share.parts;
}
template <bool EPI>
int run_joins(PieceLaunch l, hipStream_t s) {
  using T = PieceTile;
  constexpr int PER = T::WAVES * T::FM * T::FN;
  l.second = (l.p[0].tiles_m * l.p[0].tiles_n - l.p[0].share.whole) * PER;
  const int blocks = l.second + (l.p[1].tiles_m * l.p[1].tiles_n - l.p[1].share.whole) * PER;
  if (!blocks) return MX_OK;
  hipLaunchKernelGGL((piece_join_kernel<T, EPI>), dim3(unsigned(blocks)), dim3(64), 0, s, l);
  MX_LAUNCHED();
  return MX_OK;
}
int run_forward(const PieceArgs& p, hipStream_t s) {
  using T = PieceTile;
  hipLaunchKernelGGL(piece_forward_kernel<T>, dim3(unsigned(piece_blocks(p))), dim3(T::THREADS), 0, s, p);
  MX_LAUNCHED();
  PieceLaunch l{};
  l.p[0] = p;
  return run_joins<true>(l, s);
}
int run_backward(PieceLaunch l, hipStream_t s) {
  using T = PieceTile;
  const int blocks[2] = {piece_blocks(l.p[0]), piece_blocks(l.p[1])};
  l.swapped = l.p[1].nk > l.p[0].nk;
  l.second = blocks[l.swapped];
  hipLaunchKernelGGL(piece_backward_kernel<T>, dim3(unsigned(blocks[0] + blocks[1])), dim3(T::THREADS), 0, s, l);
  MX_LAUNCHED();
  return run_joins<false>(l, s);
}

// First and second pass of a call's operands.
template <bool ENDS>
int run_scan(ScanArgs* p, hipStream_t s) {
  int blocks = 0;
  for (int i = 0; i < p->count; ++i) {
    p->op[i].first = blocks;
    blocks += p->op[i].col_blocks * p->op[i].parts;
  }
  if (p->op[0].n >= 4)
    hipLaunchKernelGGL((scan_kernel<4, ENDS>), dim3(unsigned(blocks)), dim3(256), 0, s, *p);
  else
    hipLaunchKernelGGL((scan_kernel<1, ENDS>), dim3(unsigned(blocks)), dim3(256), 0, s, *p);
  MX_LAUNCHED();
  return MX_OK;
}
int run_pack(PackArgs* p, hipStream_t s) {
  int blocks = 0;
  for (int i = 0; i < p->count; ++i) {
    p->op[i].first = blocks;
    blocks += p->op[i].wide * (p->op[i].to.rows / 32);
  }
  p->first_sum = blocks;
  if (p->out) blocks += (p->n + 31) / 32;
  hipLaunchKernelGGL(pack_kernel, dim3(unsigned(blocks)), dim3(256), 0, s, *p);
  MX_LAUNCHED();
  ListArgs lists{};
  int count = 0;
  for (int i = 0; i < p->count; ++i)
    for (const Counts* c : {&p->op[i].rows, &p->op[i].columns})
      if (c->ends) lists.of[count++] = *c;
  if (!count) return MX_OK;
  hipLaunchKernelGGL(list_kernel, dim3(kListEnds, unsigned(count)), dim3(256), 0, s, lists);
  MX_LAUNCHED();
  return MX_OK;
}

// ----------------------------------------------------------------- the calls
// Workspace of a forward: the packed operands, or the product's K split.
struct Forward {
  bool packed;
  Packed x, w;
  Head* head = nullptr;
  pieces::Deal deal{};
  float* sums = nullptr;
  int64_t partial = 0;
  Forward(int64_t m, int64_t k, int64_t n, Carve* c) : packed(form_of(m, k, n, false) == Form::kPacked) {
    if (!packed) return;
    head = c->take<Head>(1);
    x = mx::packed(m, k, true, false, c);
    w = mx::packed(n, k, true, false, c);
    deal = plan_piece(m, n, k, 1.0);
    sums = c->take<float>(deal.sum_bytes(kPad) / 4);
  }
};

// Waves that share a tile's K, each with a step of it: eight for a forward's few
// tiles; four for a backward (of the layer's longer product, whichever gradients
// are asked for: their sums do not depend on it), most of whose tiles have short K.
int direct_waves(int64_t m, int64_t k, int64_t n, bool backward) {
  const int64_t steps = ((backward ? std::max(m, n) : k) + 15) / 16;
  return steps >= 8 && !backward ? 8 : steps >= 4 ? 4 : 1;
}

DirectProduct direct_product_of(const float* a, const float* b, float* out, int64_t m, int64_t n, int64_t k,
                                int64_t a_stride, int64_t b_stride, bool a_along) {
  DirectProduct p{};
  p.a = a;
  p.b = b;
  p.out = out;
  p.m = int(m);
  p.n = int(n);
  p.k = int(k);
  p.a_stride = a_stride;
  p.b_stride = b_stride;
  p.a_along = a_along;
  p.tiles_n = int((n + 31) / 32);
  return p;
}

template <bool FORWARD>
int run_direct(DirectArgs* d, int wk, hipStream_t s) {
  d->tiles = 0;
  for (int i = 0; i < d->count; ++i) {
    d->p[i].first = d->tiles;
    d->tiles += (d->p[i].m + 31) / 32 * d->p[i].tiles_n;
  }
  const dim3 grid(unsigned(wk == 1 ? (d->tiles + 3) / 4 : d->tiles)), block(unsigned(wk == 1 ? 256 : 64 * wk));
  if (wk == 8)
    hipLaunchKernelGGL((direct_kernel<FORWARD, 8>), grid, block, 0, s, *d);
  else if (wk == 4)
    hipLaunchKernelGGL((direct_kernel<FORWARD, 4>), grid, block, 0, s, *d);
  else
    hipLaunchKernelGGL((direct_kernel<FORWARD, 1>), grid, block, 0, s, *d);
  MX_LAUNCHED();
  return MX_OK;
}

template <int M>
int run_few(const float* x, const float* w, const float* bias, const float* residual, int64_t m, int64_t k, int64_t n, int act,
            float* y, float* z, hipStream_t s) {
  const int64_t groups = (m + M - 1) / M, blocks = (n + kFewRows - 1) / kFewRows;
  hipLaunchKernelGGL(few_kernel<M>, dim3(unsigned((blocks + 7) / 8 * 8 * groups)), dim3(256), 0, s, x, w, bias, residual,
                     int(m), int(groups), k, int(n), act, y, z);
  MX_LAUNCHED();
  return MX_OK;
}

int forward_bytes(int64_t m, int64_t k, int64_t n, int64_t* bytes) {
  *bytes = 0;
  if (m == 0 || n == 0 || k == 0) return MX_OK;
  const Form form = form_of(m, k, n, false);
  if (form == Form::kFew || form == Form::kSmall) return MX_OK;
  Carve c(nullptr);
  const Forward f(m, k, n, &c);
  *bytes = c.used;
  return f.packed ? MX_OK : partials(forward_desc(m, k, n, true), bytes);
}

// Workspace of small products' backward.
float* small_dz(int64_t m, int64_t n, bool slope, Carve* c) { return slope ? c->take<float>(m * n) : nullptr; }

// Workspace of a backward.
struct Backward {
  bool packed;
  ScanPlan scan;  // of dz
  float *dz = nullptr, *part = nullptr, *sums_x = nullptr, *sums_w = nullptr;
  Head* head = nullptr;
  Packed g, x, w;
  pieces::Deal to_x{}, to_w{};
  int64_t gemm = 0;
  void* split = nullptr;
  int status = MX_OK;
  Backward(int64_t m, int64_t k, int64_t n, bool slope, bool want_x, bool want_w, bool want_b, bool split_room,
           bool piece_room, Carve* c)
      : packed(piece_room && (want_x || want_w) && form_of(m, k, n, true) == Form::kPacked), scan(plan_scan(m, n)) {
    if (slope && (want_x || want_w)) dz = c->take<float>(m * n);
    if (want_b && scan.parts > 1) part = c->take<float>(int64_t(scan.parts) * n);
    if (packed) {
      head = c->take<Head>(1);
      g = mx::packed(m, n, want_x, want_w, c);
      if (want_w) x = mx::packed(m, k, false, true, c);
      if (want_x) w = mx::packed(n, k, false, true, c);
      // Dealt as if both were wanted: a gradient's sums do not depend on the other.
      const double wx = piece_work(m, k, n), ww = piece_work(n, k, m);
      to_x = plan_piece(m, k, n, wx / (wx + ww));
      to_w = plan_piece(n, k, m, ww / (wx + ww));
      sums_x = c->take<float>(want_x ? to_x.sum_bytes(kPad) / 4 : 0);
      sums_w = c->take<float>(want_w ? to_w.sum_bytes(kPad) / 4 : 0);
    } else if (split_room && k > 0) {
      int64_t a = 0, b = 0;
      if (want_x) status = partials(dx_desc(m, k, n), &a);
      if (want_w && status == MX_OK) status = partials(dw_desc(m, k, n), &b);
      gemm = std::max(a, b);
      split = c->take<char>(gemm);
    }
  }
};

}  // namespace
}  // namespace mx

using namespace mx;

extern "C" int mx_linear_workspace(int64_t m, int64_t k, int64_t n, int activation, int backward, int64_t* bytes) {
  MX_ABI_BEGIN
  MX_TRY(check("mx_linear_workspace", m, k, n, activation));
  MX_REQUIRE(bytes, MX_ERR_INVALID, "mx_linear_workspace: null result");
  *bytes = 0;
  if (m == 0 || n == 0) return MX_OK;
  if (!backward) return forward_bytes(m, k, n, bytes);
  Carve c(nullptr);
  if (k > 0 && form_of(m, k, n, true) == Form::kSmall) {
    (void)small_dz(m, n, activation != MX_ACT_NONE, &c);
    *bytes = c.used;
    return MX_OK;
  }
  const Backward b(m, k, n, activation != MX_ACT_NONE, k > 0, k > 0, true, true, true, &c);
  *bytes = c.used;
  return b.status;
  MX_ABI_END
}

extern "C" int mx_linear_variant(int64_t m, int64_t k, int64_t n, int backward, char* buf, size_t len) {
  MX_ABI_BEGIN
  MX_TRY(check("mx_linear_variant", m, k, n, MX_ACT_NONE));
  MX_REQUIRE(buf || !len, MX_ERR_INVALID, "mx_linear_variant: null buffer");
  std::string name = "none";
  if (m > 0 && n > 0 && k > 0) {
    switch (form_of(m, k, n, backward != 0)) {
      case Form::kFew: name = "few"; break;
      case Form::kSmall: name = cat("small<", direct_waves(m, k, n, backward != 0), ">"); break;
      case Form::kPacked: name = "packed"; break;
      default: {
        const float* const at = reinterpret_cast<const float*>(256);
        int64_t bytes;
        const mx_gemm_desc d = backward ? dx_desc(m, k, n) : forward_desc(m, k, n, true);
        MX_TRY(gemm_describe(&d, at, at, kPartials, &name, &bytes));
        if (backward) {
          std::string other;
          const mx_gemm_desc dw = dw_desc(m, k, n);
          MX_TRY(gemm_describe(&dw, at, at, kPartials, &other, &bytes));
          name += " " + other;
        }
      }
    }
  }
  copy_name(name, buf, len);
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_linear_forward(const float* x, const float* w, const float* bias, const float* residual, int64_t m,
                                 int64_t k, int64_t n, int activation, float* y, float* z, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  const char* const who = "mx_linear_forward";
  MX_TRY(check(who, m, k, n, activation));
  if (m == 0 || n == 0) return MX_OK;
  MX_REQUIRE(y && (k == 0 || (x && w)), MX_ERR_INVALID, who, ": null buffer");
  hipStream_t s = resolve_stream(stream);
  if (k > 0 && form_of(m, k, n, false) == Form::kFew) {
    static_assert(kFewTokens == 4);
    if (m == 1) return run_few<1>(x, w, bias, residual, m, k, n, activation, y, z, s);
    if (m == 2) return run_few<2>(x, w, bias, residual, m, k, n, activation, y, z, s);
    return run_few<kFewTokens>(x, w, bias, residual, m, k, n, activation, y, z, s);
  }
  if (k > 0 && form_of(m, k, n, false) == Form::kSmall) {
    DirectArgs a{};
    a.count = 1;
    a.act = activation;
    a.bias = bias;
    a.residual = residual;
    a.z = z;
    a.p[0] = direct_product_of(x, w, y, m, n, k, k, k, true);
    return run_direct<true>(&a, direct_waves(m, k, n, false), s);
  }
  const mx_gemm_desc d = forward_desc(m, k, n, bias != nullptr);
  const GemmEpilogue epi{activation, residual, z};
  int64_t need = 0;
  Workspace ws;
  if (form_of(m, k, n, false) != Form::kPacked) {
    // The product's own scratch is optional: without the caller's, it allocates
    // where it may.
    if (workspace) {
      MX_TRY(forward_bytes(m, k, n, &need));
      MX_TRY(ws.take(who, workspace, workspace_bytes, need, s));
    }
    return gemm_within(&d, x, w, bias, y, kPartials, s, &epi, ws.as<void>());
  }
  MX_TRY(forward_bytes(m, k, n, &need));
  const int room = ws.take(who, workspace, workspace_bytes, need, s);
  if (room == MX_ERR_OOM) {  // no room for pieces: tiles need none
    clear_error();
    return gemm_within(&d, x, w, bias, y, kPartials, s, &epi);
  }
  MX_TRY(room);
  Carve c(ws.as<void>());
  Forward f(m, k, n, &c);
  f.x.first.src = f.x.second.src = x;
  f.w.first.src = f.w.second.src = w;
  f.x.second.about = &f.head->a;
  f.w.second.about = &f.head->b;
  ScanArgs scan{{f.x.first, f.w.first}, 2, activation};
  MX_TRY(run_scan<true>(&scan, s));
  PackArgs pack{};
  pack.count = 2;
  pack.op[0] = f.x.second;
  pack.op[1] = f.w.second;
  MX_TRY(run_pack(&pack, s));
  PieceArgs p{};
  p.out = y;
  p.bias = bias;
  p.residual = residual;
  p.z = z;
  p.act = activation;
  fill_piece(&p, f.deal, f.x, false, f.w, false, f.head->left, f.sums);
  MX_TRY(run_forward(p, s));
  return gemm_within(&d, x, w, bias, y, 0, s, &epi, nullptr, f.head->left);
  MX_ABI_END
}

extern "C" int mx_linear_backward(const float* dy, const float* x, const float* w, const float* z, int64_t m, int64_t k,
                                  int64_t n, int activation, float* dx, float* dw, float* db, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  const char* const who = "mx_linear_backward";
  MX_TRY(check(who, m, k, n, activation));
  hipStream_t s = resolve_stream(stream);
  const auto zero = [&](float* p, int64_t count) -> int {
    if (!p || count == 0) return MX_OK;
    hipLaunchKernelGGL(zero_kernel, dim3(unsigned(std::min<int64_t>((count + 255) / 256, 65535))), dim3(256), 0, s, p, count);
    MX_LAUNCHED();
    return MX_OK;
  };
  if (m == 0 || n == 0) {  // empty sums
    MX_TRY(zero(dx, m * k));
    MX_TRY(zero(dw, n * k));
    return zero(db, n);
  }
  const bool slope = activation != MX_ACT_NONE;
  MX_REQUIRE(dy && (!slope || z) && (k == 0 || ((!dx || w) && (!dw || x))), MX_ERR_INVALID, who, ": null buffer");
  if (k == 0) dx = dw = nullptr;
  if (!dx && !dw && !db) return MX_OK;
  if (k > 0 && form_of(m, k, n, true) == Form::kSmall) {
    Carve size(nullptr);
    (void)small_dz(m, n, slope, &size);
    Workspace ws;
    MX_TRY(ws.take(who, workspace, workspace_bytes, size.used, s));
    Carve c(ws.as<void>());
    const float* g = dy;
    if (slope) {
      float* const dz = small_dz(m, n, slope, &c);
      const ScanPlan sp = plan_scan(m, n);
      ScanArgs scan{};
      scan.act = activation;
      scan.count = 1;
      ScanOp& o = scan.op[0];
      o.src = dy;
      o.z = z;
      o.dz = dz;
      o.m = m;
      o.n = int(n);
      o.rows_per = sp.rows_per;
      o.col_blocks = sp.col_blocks;
      o.parts = sp.parts;
      MX_TRY(run_scan<false>(&scan, s));
      g = dz;
    }
    DirectArgs a{};
    if (dx) a.p[a.count++] = direct_product_of(g, w, dx, m, k, n, n, k, true);
    if (dw || db) {  // db alone: the first column of dw's tiles, not stored
      DirectProduct& p = a.p[a.count++];
      p = direct_product_of(g, dw ? x : g, dw, n, dw ? k : 1, m, n, dw ? k : 0, false);
      p.row_sums = db;
    }
    return run_direct<false>(&a, direct_waves(m, k, n, true), s);
  }
  // Without the caller's workspace the K splits of products that are not packed
  // are left to them (captured calls take one pass each).
  Workspace ws;
  const auto take = [&](bool piece_room) -> int {
    Carve size(nullptr);
    const Backward want(m, k, n, slope, dx, dw, db, workspace != nullptr, piece_room, &size);
    MX_TRY(want.status);
    return ws.take(who, workspace, workspace_bytes, size.used, s);
  };
  int room_for = take(true);
  const bool piece_room = room_for != MX_ERR_OOM;
  if (!piece_room) {  // none for pieces: tiles need dz and its column sums alone
    clear_error();
    room_for = take(false);
  }
  MX_TRY(room_for);
  Carve c(ws.as<void>());
  Backward b(m, k, n, slope, dx, dw, db, workspace != nullptr, piece_room, &c);
  const float* const g = b.dz ? b.dz : dy;
  // First pass: dz, its column sums and, for packed products, everyone's largest.
  ScanArgs scan{};
  scan.act = activation;
  scan.count = 1;
  ScanOp& first = scan.op[0];
  if (b.packed) {
    first = b.g.first;
  } else {
    first.m = m;
    first.n = int(n);
    first.rows_per = b.scan.rows_per;
    first.col_blocks = b.scan.col_blocks;
    first.parts = b.scan.parts;
  }
  first.src = dy;
  first.z = slope ? z : nullptr;
  first.dz = b.dz;
  first.sums = !db ? nullptr : b.scan.parts > 1 ? b.part : db;
  if (b.packed) {
    b.g.second.src = g;
    b.g.second.about = &b.head->a;
    PackArgs pack{};
    pack.op[pack.count++] = b.g.second;
    if (dw) {
      b.x.first.src = b.x.second.src = x;
      b.x.second.about = &b.head->b;
      scan.op[scan.count++] = b.x.first;
      pack.op[pack.count++] = b.x.second;
    }
    if (dx) {
      b.w.first.src = b.w.second.src = w;
      b.w.second.about = &b.head->c;
      scan.op[scan.count++] = b.w.first;
      pack.op[pack.count++] = b.w.second;
    }
    MX_TRY(run_scan<true>(&scan, s));
    if (db && b.scan.parts > 1) {
      pack.part = b.part;
      pack.parts = b.scan.parts;
      pack.n = int(n);
      pack.out = db;
    }
    MX_TRY(run_pack(&pack, s));
  } else if (db || b.dz) {
    MX_TRY(run_scan<false>(&scan, s));
  }
  if (db && b.scan.parts > 1 && !b.packed) {
    hipLaunchKernelGGL(column_sum_kernel, dim3(unsigned((n + 31) / 32)), dim3(1024), 0, s, b.part, b.scan.parts, int(n), db);
    MX_LAUNCHED();
  }
  const int64_t room = b.packed ? 0 : kPartials;
  if (b.packed) {
    PieceLaunch l{};
    if (dx) {
      l.p[0].out = dx;
      fill_piece(&l.p[0], b.to_x, b.g, false, b.w, true, b.head->left, b.sums_x);
    }
    if (dw) {
      l.p[1].out = dw;
      fill_piece(&l.p[1], b.to_w, b.g, true, b.x, true, b.head->left + 1, b.sums_w);
    }
    MX_TRY(run_backward(l, s));
  }
  if (dx) {
    const mx_gemm_desc d = dx_desc(m, k, n);
    MX_TRY(gemm_within(&d, g, w, nullptr, dx, room, s, nullptr, b.split, b.packed ? b.head->left : nullptr));
  }
  if (dw) {
    const mx_gemm_desc d = dw_desc(m, k, n);
    MX_TRY(gemm_within(&d, g, x, nullptr, dw, room, s, nullptr, b.split, b.packed ? b.head->left + 1 : nullptr));
  }
  return MX_OK;
  MX_ABI_END
}
