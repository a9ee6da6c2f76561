// Orthogonalised momentum: Newton-Schulz iterations on the matrices of one
// shape side by side, and the optimizer step around them (FP32).
//
//   X = U / max(|U|_F, eps), U turned so that its shorter side is the rows
//   steps times:  G = X X^T,  P = b G + c G^2,  X = a X + P X
//   out = X, or  param = param (1 - lr wd) - lr r X
//
// a X is added to the finished product, once: as a I in P it would be in the
// sum from the first slab on, and every later rounding would be one of a X,
// while P X is small in the first iterations, whose errors the later ones
// multiply (4096 x 4096 against float64: 4.6e-6 so, 2.6e-6 added).  The last
// iteration, which nothing follows, has it in P and so reads X only once.
//
// The iterates are this file's own, so they are kept as two fp16 pieces
// (mx_pieces.hpp) from the first read of U to the last product, whose stores
// give FP32.  What bounds their entries is what the pieces' scale needs: an
// entry is at most the largest singular value, 1 for X (the norm divides it),
// and from there the polynomial's extremes (bounds(), on the host).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "mfma_core.hpp"
#include "mx_internal.hpp"
#include "mx_pieces.hpp"

namespace mx {
namespace {

using namespace pieces;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kBatch = 48;      // matrices of one set of launches
constexpr int kNormParts = 1024;  // most partial squares of one matrix
constexpr int64_t kMaxScratch = int64_t(1) << 30;  // of one set, unless one matrix takes more

// The matrices of one set of launches, all of one shape.
struct Table {
  const float* in[kBatch];  // U, or the gradient
  float* buf[kBatch];       // momentum (Muon)
  float* out[kBatch];       // the factor, or the parameter
};

// U of an element: itself, or Nesterov's or plain momentum.
struct Update {
  int muon, nesterov;
  float momentum, rest;  // mu, 1 - mu
  __device__ __forceinline__ float moved(float buf, float g) const { return buf + rest * (g - buf); }
  __device__ __forceinline__ float u(float buf, float g) const { return nesterov ? g + momentum * (buf - g) : buf; }
};

// Squares of U, in double (FP32 squares of a gradient overflow at 2^64 and
// vanish at 2^-75), and the new momentum.  16 bytes at a time where VEC (all
// tensors 16-byte aligned).
template <bool VEC>
__global__ __launch_bounds__(256) void norm_kernel(Table tab, Update up, int64_t numel, double* parts) {
  __shared__ double sum[4];
  const int b = blockIdx.y;
  const float* const in = tab.in[b];
  float* const buf = tab.buf[b];
  double s = 0;
  const int64_t first = int64_t(blockIdx.x) * 256 + threadIdx.x, step = int64_t(gridDim.x) * 256;
  const int64_t vecs = VEC ? numel / 4 : 0;
#pragma unroll 4
  for (int64_t i = first; i < vecs; i += step) {
    f32x4 u = reinterpret_cast<const f32x4*>(in)[i];
    if (up.muon) {
      f32x4 m = reinterpret_cast<const f32x4*>(buf)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[e] = up.moved(m[e], u[e]);
        u[e] = up.u(m[e], u[e]);
      }
      reinterpret_cast<f32x4*>(buf)[i] = m;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s += double(u[e]) * double(u[e]);
  }
#pragma unroll 4
  for (int64_t i = vecs * 4 + first; i < numel; i += step) {
    float u = in[i];
    if (up.muon) {
      const float m = up.moved(buf[i], u);
      buf[i] = m;
      u = up.u(m, u);
    }
    s += double(u) * double(u);
  }
  for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
  if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) parts[b * kNormParts + blockIdx.x] = sum[0] + sum[1] + sum[2] + sum[3];
}

// |U|_F from its partial squares, to every thread of a workgroup of 256.
__device__ __forceinline__ double norm_of(const double* parts, int nparts) {
  __shared__ double sum[4];
  double s = 0;
  for (int i = threadIdx.x; i < nparts; i += 256) s += parts[i];
  for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
  if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = s;
  __syncthreads();
  return sqrt(sum[0] + sum[1] + sum[2] + sum[3]);
}

struct Geometry {
  int rows, cols;     // of U
  int s, l;           // shorter and longer side
  int sp, lp;         // padded
  bool turned;        // X = U^T
  __host__ __device__ int64_t x_plane() const { return int64_t(sp) * lp; }
  __host__ __device__ int64_t g_plane() const { return int64_t(sp) * sp; }
};

// U's elements at X's row and eight columns from col, zeros past X's end.
__device__ __forceinline__ void take_u(const Table& tab, const Update& up, const Geometry& g, int b, int row, int col,
                                       float (&u)[8]) {
  const auto take = [&](const float* from, float (&to)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) to[e] = 0.f;
    if (row >= g.s || col >= g.l) return;
    if (g.turned) {  // neighbours along U's rows in neighbouring lanes
#pragma unroll
      for (int e = 0; e < 8; ++e) to[e] = col + e < g.l ? from[int64_t(col + e) * g.cols + row] : 0.f;
    } else if (col + 8 <= g.l) {
      const f32x4u* const at = reinterpret_cast<const f32x4u*>(from + int64_t(row) * g.cols + col);
      const f32x4 a = at[0], c = at[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        to[e] = a[e];
        to[4 + e] = c[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) to[e] = col + e < g.l ? from[int64_t(row) * g.cols + col + e] : 0.f;
    }
  };
  take(tab.in[b], u);
  if (!up.muon) return;
  float m[8];
  take(tab.buf[b], m);
#pragma unroll
  for (int e = 0; e < 8; ++e) u[e] = up.u(m[e], u[e]);
}

// What U's elements are multiplied by to become X's stored value.  |X|_F is 1,
// unless eps is what divides: then X is kept times 2^up2, which no iteration's
// growth takes past the bounds, so that fp16 holds it.
__device__ __forceinline__ double scale_of(const double* parts, int nparts, double eps, double growth, float scale,
                                           int& up2) {
  const double n = norm_of(parts, nparts), d = n < eps ? eps : n, small = n / d * growth;
  up2 = small > 0 && small < 1 ? int(floor(-log2(small))) : 0;
  return ldexp(double(scale), up2) / d;
}

// X's pieces: 32 rows of X and 64 of its columns to a workgroup, eight columns
// of a row to a thread.
__global__ __launch_bounds__(256) void pack_kernel(Table tab, Update up, Geometry g, const double* parts, int nparts,
                                                   double eps, float scale, double growth, _Float16* x,
                                                   float* lift) {
  const int b = blockIdx.z;
  const int row = blockIdx.y * 32 + (threadIdx.x & 31), col = blockIdx.x * 64 + (threadIdx.x >> 5) * 8;
  float u[8];
  take_u(tab, up, g, b, row, col, u);
  int up2;
  const double inv = scale_of(parts + b * kNormParts, nparts, eps, growth, scale, up2);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) lift[b] = float(ldexp(1.0, -up2));
  half8 hi, lo;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = float(double(u[e]) * inv);
    hi[e] = _Float16(v);
    lo[e] = _Float16(v - float(hi[e]));
  }
  const int64_t plane = g.x_plane();
  _Float16* const to = x + b * 2 * plane + (int64_t(col >> 3) * g.sp + row) * 8;
  *reinterpret_cast<half8*>(to) = hi;
  *reinterpret_cast<half8*>(to + plane) = lo;
}

// kLast: U's rows are X's columns; kLastRows: U's rows are X's.
enum Kind { kGram, kPoly, kNext, kLast, kLastRows };

struct StepArgs {
  const _Float16 *a, *b;  // operands (kPoly: both G)
  _Float16* out;          // pieces of the result
  int64_t a_plane, b_plane, out_plane;
  int a_rows, b_rows, out_rows;
  int nk;                 // slabs
  int tiles_m, tiles_n;
  Shares share;
  float alpha;            // product of pieces -> stored value
  float diag, lin, unit;  // kPoly: a (the last iteration's) and b times the stored scale, 1 / G's scale
  float keep;             // kNext: a times the stored scale over X's
  const float* lift;      // X's pieces hold X / lift[matrix]
  // kLast
  Table tab;
  Geometry g;
  int muon;
  float decay, step;      // 1 - lr wd, lr r
};

constexpr bool symmetric(int kind) { return kind == kGram || kind == kPoly; }

// Tile t of the lower triangle of n x n tiles, in bands of eight tile rows
// walked column by column: tiles that run together share rows of both operands
// (row by row, 64 neighbours read 65 panels; so, 16).
__device__ __forceinline__ void lower_tile(int t, int n, int& tm, int& tn) {
  // Band g begins at 32 g^2 + 4 g.
  int g = int((sqrtf(16.f + 128.f * float(t)) - 4.f) / 64.f);
  while (32 * g * g + 4 * g > t) --g;
  while (32 * (g + 1) * (g + 1) + 4 * (g + 1) <= t) ++g;
  const int first = 8 * g, rows = min(8, n - first);
  t -= 32 * g * g + 4 * g;
  if (t < first * rows) {
    tm = first + t % rows;
    tn = t / rows;
    return;
  }
  t -= first * rows;
  int r = 0;
  while (t > r) t -= ++r;
  tm = first + r;
  tn = first + t;
}

template <int KIND>
__device__ __forceinline__ void tile_of(const StepArgs& p, int id, int& b, int& tm, int& tn) {
  const int per = symmetric(KIND) ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * p.tiles_n;
  b = id / per;
  if constexpr (symmetric(KIND))
    lower_tile(id - b * per, p.tiles_m, tm, tn);
  else
    mfma::tile_coords(id - b * per, p.tiles_m, p.tiles_n, tm, tn);
}

// What a fragment adds to its product: pieces (kPoly: of G, kNext: of X) or, for
// the last product of a Muon step, the parameter.
template <int KIND>
struct Before {
  half4 hi[4], lo[4];
};
template <>
struct Before<kGram> {};
struct Parameter {
  float was[16];
};
template <>
struct Before<kLast> : Parameter {};
template <>
struct Before<kLastRows> : Parameter {};

// Reads that for the 32 x 32 fragment at row m, column n.
template <int KIND>
__device__ __forceinline__ void read_before(const StepArgs& p, int b, int m, int n, Before<KIND>& o) {
  const int lane = threadIdx.x & 63;
  if constexpr (KIND == kLast || KIND == kLastRows) {
    if (!p.muon) return;
    const int col = min((KIND == kLast ? m : n) + (lane & 31), p.g.cols - 1), row0 = (KIND == kLast ? n : m) + 4 * (lane >> 5);
    const float* const at = p.tab.out[b] + col;
#pragma unroll
    for (int i = 0; i < 16; ++i) o.was[i] = at[int64_t(min(row0 + 8 * (i >> 2) + (i & 3), p.g.rows - 1)) * p.g.cols];
  } else if constexpr (KIND != kGram) {
    const int r = m + (lane & 31), c0 = n + 4 * (lane >> 5);
    const int64_t plane = KIND == kPoly ? p.a_plane : p.b_plane;
    const Planes po{p.out, p.out_plane, p.out_rows};
    const _Float16* const was = (KIND == kPoly ? p.a : p.b) + b * 2 * plane;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      o.hi[q] = *reinterpret_cast<const half4*>(was + elem(po, r, c0 + 8 * q));
      o.lo[q] = *reinterpret_cast<const half4*>(was + plane + elem(po, r, c0 + 8 * q));
    }
  }
}

// Stores a 32 x 32 fragment of a product at row m, column n (of X for the last
// product).  mirror: its transpose too.
template <int KIND>
__device__ __forceinline__ void finish(const StepArgs& p, int b, bool mirror, int m, int n, const f32x16& v, const Before<KIND>& was) {
  const int lane = threadIdx.x & 63;
  if constexpr (KIND == kLast || KIND == kLastRows) {
    // A wave writes whole 128-byte lines of U's rows either way round.
    const float alpha = p.alpha * p.lift[b];
    const int col = (KIND == kLast ? m : n) + (lane & 31), row0 = (KIND == kLast ? n : m) + 4 * (lane >> 5);
    float* const to = p.tab.out[b] + int64_t(row0) * p.g.cols + col;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = 8 * (i >> 2) + (i & 3);
      const float x = v[i] * alpha;
      if (col < p.g.cols && row0 + r < p.g.rows) to[int64_t(r) * p.g.cols] = p.muon ? was.was[i] * p.decay - p.step * x : x;
    }
  } else {
    // G's pieces hold G itself: where X is tiny, all of it that b G and c G^2
    // add to a I lies below what G's scale can hold.
    const float alpha = KIND == kGram ? p.alpha * p.lift[b] * p.lift[b] : p.alpha;
    const Planes po{p.out + b * 2 * p.out_plane, p.out_plane, p.out_rows};
    const int r = m + (lane & 31), c0 = n + 4 * (lane >> 5);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = c0 + 8 * q;
      const int64_t at = elem(po, r, c);
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = alpha * v[4 * q + e];
        if constexpr (KIND == kPoly)
          o[e] = (r == c + e ? p.diag : 0.f) + p.lin * ((float(was.hi[q][e]) + float(was.lo[q][e])) * p.unit) + o[e];
        if constexpr (KIND == kNext) o[e] += p.keep * (float(was.hi[q][e]) + float(was.lo[q][e]));
      }
      half4 hi, lo;
      split4(o, hi, lo);
      *reinterpret_cast<half4*>(po.at + at) = hi;
      *reinterpret_cast<half4*>(po.at + po.plane + at) = lo;
      if constexpr (symmetric(KIND)) {
        if (mirror) {  // each lane takes a row of its four lanes' block
          const int64_t across = elem(po, c + (r & 3), r & ~3);
          *reinterpret_cast<half4*>(po.at + across) = transpose4(hi);
          *reinterpret_cast<half4*>(po.at + po.plane + across) = transpose4(lo);
        }
      }
    }
  }
}

// One product of the iteration.  G and P are symmetric: only the tiles on and
// below the diagonal are computed, and stored both ways.
template <class T, int KIND>
__global__ __launch_bounds__(T::THREADS) __attribute__((amdgpu_waves_per_eu(T::OCC, T::OCC))) void step_kernel(StepArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[T::SMEM];
  constexpr bool SYM = symmetric(KIND);
  const Unit unit = unit_of(p.share, blockIdx.x, p.nk);
  int b, tm, tn;
  tile_of<KIND>(p, unit.tile, b, tm, tn);
  const Planes pa{const_cast<_Float16*>(p.a) + b * 2 * p.a_plane, p.a_plane, p.a_rows};
  const Planes pb{const_cast<_Float16*>(p.b) + b * 2 * p.b_plane, p.b_plane, p.b_rows};
  f32x16 acc[T::FM][T::FN];
  product<T, false, !SYM, KIND == kLastRows>(acc, pa, pb, tm * T::BM, tn * T::BN, unit.k0, unit.k1 - unit.k0, smem);
  if (unit.tile >= p.share.whole) {
    store_sums<T>(acc, p.share, unit);
    return;
  }
  const int wave = threadIdx.x >> 6;
  const int m0 = tm * T::BM + wave / T::WN * (T::BM / T::WM), n0 = tn * T::BN + wave % T::WN * (T::BN / T::WN);
  // What fragments add is read that far ahead: behind the stores of the one
  // before, which might be to the same place, each would wait for memory anew (the
  // last product of a step over 16 x 1024^2 took 160 us so and takes 114, over 6 x 1000
  // x 513 32 and 20; the pieces that the others read are still in the caches).
  constexpr int F = T::FM * T::FN, AHEAD = F > 4 ? 2 : F;
  Before<KIND> was[AHEAD];
  const auto read = [&](int f) { read_before<KIND>(p, b, m0 + f / T::FN * 32, n0 + f % T::FN * 32, was[f % AHEAD]); };
#pragma unroll
  for (int f = 0; f < AHEAD; ++f) read(f);
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const Before<KIND> mine = was[f % AHEAD];
    if (f + AHEAD < F) read(f + AHEAD);
    finish<KIND>(p, b, tm != tn, m0 + f / T::FN * 32, n0 + f % T::FN * 32, acc[f / T::FN][f % T::FN], mine);
  }
}

// The tiles that were taken in parts.
template <class T, int KIND>
__global__ __launch_bounds__(64) void join_kernel(StepArgs p) {
  int tile, m, n, b, tm, tn;
  const f32x16 v = join_sums<T>(p.share, blockIdx.x, tile, m, n);
  tile_of<KIND>(p, tile, b, tm, tn);
  m += tm * T::BM;
  n += tn * T::BN;
  Before<KIND> was;
  read_before<KIND>(p, b, m, n, was);
  finish<KIND>(p, b, tm != tn, m, n, v, was);
}

// steps == 0: the scaled matrix itself.
__global__ __launch_bounds__(256) void scaled_kernel(Table tab, Update up, int64_t numel, const double* parts, int nparts,
                                                     double eps, float decay, float step) {
  const int b = blockIdx.y;
  const double n = norm_of(parts + b * kNormParts, nparts), inv = 1.0 / (n < eps ? eps : n);
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < numel; i += int64_t(gridDim.x) * 256) {
    float u = tab.in[b][i];
    if (up.muon) u = up.u(tab.buf[b][i], u);
    const float x = float(double(u) * inv);
    tab.out[b][i] = up.muon ? tab.out[b][i] * decay - step * x : x;
  }
}

// ------------------------------------------------------- one launch a step
// Matrices of at most 64 rows: an iteration is one launch.  Each workgroup sums
// the partial G's that the workgroups of the launch before it left, makes P of it
// for itself, moves its own columns of X by it, and leaves its part of the next
// G.  X stays where it is.  The first launch packs X; the last one stores the
// factor.  Bound by the launches and by the barriers within one (use_small()).
struct SmallArgs {
  Table tab;
  Update up;
  Geometry g;
  const double* norms;
  int nparts;
  double eps, growth;
  float scale;            // of X's first pieces
  float* lift;
  _Float16* x;
  const float* from;      // partial G's of the launch before, [matrix][workgroup][fragment][256][4]
  float* to;
  float gram;             // pieces of X, product -> G's stored value
  float alpha, diag, lin, unit;  // P
  float move, keep;       // X: product -> stored value, X's pieces -> stored value
  float decay, step;
};
enum SmallMode { kSmallFirst, kSmallNext, kSmallLast };
constexpr int kSmall = 64;       // X's rows, padded
constexpr int kSmallWide = 16;   // most workgroups of a matrix: each reads every other's part of G

template <int MODE>
__global__ __launch_bounds__(256) void small_kernel(SmallArgs p) {
  constexpr int SP = kSmall, F = SP / 32, NF = F * (F + 1) / 2;  // fragments of a side, of the triangle
  constexpr int ITEMS = SP * 8 / 256;                            // groups of eight columns of a thread
  __shared__ __attribute__((aligned(16))) char gp[MODE == kSmallFirst ? 16 : 2 * SP * SP * 2];
  __shared__ __attribute__((aligned(16))) char xs[2 * SP * 64 * 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = blockIdx.x, nw = gridDim.x, b = blockIdx.y;
  // Three waves hold the triangle's fragments (0, 0), (1, 0), (1, 1).
  const bool mine = wave < NF;
  const int fr = wave == 0 ? 0 : 1, fc = wave == 2 ? 1 : 0;
  // 16 bytes of G's or P's plane pl: eight columns from 8 kg of a row; of X's, rows
  // of a group rearranged so that transposing reads meet every bank once.
  const auto g_at = [&](int pl, int kg, int row) { return gp + ((pl * (SP / 8) + kg) * SP + row) * 16; };
  const auto x_at = [&](int pl, int kg, int row) { return xs + ((pl * 8 + kg) * SP + (row ^ ((kg & 3) << 2))) * 16; };
  const auto mul = [](f32x16& acc, const half8 (&fb)[2], const half8 (&fa)[2]) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fb[1], fa[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fb[0], fa[1], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fb[0], fa[0], acc, 0, 0, 0);
  };
  const auto store_g = [&](int m, int n, const float (&o)[16]) {
    const int r = m + (lane & 31);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = n + 8 * q + 4 * (lane >> 5);
      const float v[4] = {o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]};
      half4 h[2];
      split4(v, h[0], h[1]);
#pragma unroll
      for (int pl = 0; pl < 2; ++pl) {
        *reinterpret_cast<half4*>(g_at(pl, c >> 3, r) + (c & 7) * 2) = h[pl];
        if (m != n) *reinterpret_cast<half4*>(g_at(pl, r >> 3, c + (r & 3)) + (r & 4) * 2) = transpose4(h[pl]);
      }
    }
  };
  if constexpr (MODE != kSmallFirst) {
    float p_of[16];
    const float gram = p.gram * p.lift[b] * p.lift[b];
    if (mine) {
      f32x4 s[4] = {};
      const f32x4* at = reinterpret_cast<const f32x4*>(p.from) + (int64_t(b) * nw * NF + wave) * 256 + lane;
#pragma unroll 4
      for (int w = 0; w < nw; ++w) {
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] += at[int64_t(w) * NF * 256 + q * 64];
      }
      float o[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = s[e >> 2][e & 3] * gram;
      store_g(32 * fr, 32 * fc, o);
    }
    __syncthreads();
    if (mine) {
      f32x16 acc = 0.f;
#pragma unroll
      for (int ks = 0; ks < SP / 16; ++ks) {
        half8 fa[2], fb[2];
#pragma unroll
        for (int pl = 0; pl < 2; ++pl) {
          fa[pl] = *reinterpret_cast<const half8*>(g_at(pl, 2 * ks + (lane >> 5), 32 * fr + (lane & 31)));
          fb[pl] = *reinterpret_cast<const half8*>(g_at(pl, 2 * ks + (lane >> 5), 32 * fc + (lane & 31)));
        }
        mul(acc, fb, fa);
      }
      const int r = 32 * fr + (lane & 31);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = 32 * fc + 8 * q + 4 * (lane >> 5);
        const half4 h = *reinterpret_cast<const half4*>(g_at(0, c >> 3, r) + (c & 7) * 2);
        const half4 l = *reinterpret_cast<const half4*>(g_at(1, c >> 3, r) + (c & 7) * 2);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          p_of[4 * q + e] = (r == c + e ? p.diag : 0.f) + p.lin * ((float(h[e]) + float(l[e])) * p.unit) + p.alpha * acc[4 * q + e];
      }
    }
    __syncthreads();
    if (mine) store_g(32 * fr, 32 * fc, p_of);
  }
  const int64_t plane = p.g.x_plane();
  _Float16* const x = p.x + b * 2 * plane;
  const int blocks = p.g.lp / 64, first = j * blocks / nw, end = (j + 1) * blocks / nw;
  double inv = 0;
  if constexpr (MODE == kSmallFirst) {
    int up2;
    inv = scale_of(p.norms + b * kNormParts, p.nparts, p.eps, p.growth, p.scale, up2);
    if (j == 0 && tid == 0) p.lift[b] = float(ldexp(1.0, -up2));
  }
  f32x16 acc = 0.f;  // this wave's part of the next G
  half8 held[ITEMS][2];
  const auto fetch = [&](int cb) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int item = tid + 256 * i, row = item % SP, kg = item / SP;
      const _Float16* const at = x + (int64_t(cb * 8 + kg) * SP + row) * 8;
      held[i][0] = *reinterpret_cast<const half8*>(at);
      held[i][1] = *reinterpret_cast<const half8*>(at + plane);
    }
  };
  if (MODE != kSmallFirst && first < end) fetch(first);
  for (int cb = first; cb < end; ++cb) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int item = tid + 256 * i, row = item % SP, kg = item / SP;
      if constexpr (MODE == kSmallFirst) {
        float v[8];
        take_u(p.tab, p.up, p.g, b, row, cb * 64 + kg * 8, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = float(double(v[e]) * inv);
          held[i][0][e] = _Float16(f);
          held[i][1][e] = _Float16(f - float(held[i][0][e]));
        }
        _Float16* const at = x + (int64_t(cb * 8 + kg) * SP + row) * 8;
        *reinterpret_cast<half8*>(at) = held[i][0];
        *reinterpret_cast<half8*>(at + plane) = held[i][1];
      }
#pragma unroll
      for (int pl = 0; pl < 2; ++pl) *reinterpret_cast<half8*>(x_at(pl, kg, row)) = held[i][pl];
    }
    __syncthreads();
    if constexpr (MODE != kSmallFirst) {
      if (cb + 1 < end) fetch(cb + 1);
      half4 moved[4][2];
      const int m = wave / 2 * 32, n = wave % 2 * 32;
      {
        f32x16 v = 0.f;
#pragma unroll
        for (int ks = 0; ks < SP / 16; ++ks) {
          half8 fa[2], fb[2];
          const int c = lane & 15, kg = n / 8 + ((lane & 16) >> 3) + ((c & 3) >> 1);
#pragma unroll
          for (int pl = 0; pl < 2; ++pl) {
            fa[pl] = *reinterpret_cast<const half8*>(g_at(pl, 2 * ks + (lane >> 5), m + (lane & 31)));
            s16x4 q[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
              q[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (__attribute__((address_space(3))) s16x4*)(x_at(pl, kg, 16 * ks + 8 * (lane >> 5) + (c >> 2) + 4 * h) + 8 * (c & 1)));
            fb[pl] = __builtin_bit_cast(half8, __builtin_shufflevector(q[0], q[1], 0, 1, 2, 3, 4, 5, 6, 7));
          }
          mul(v, fb, fa);
        }
        const int r = m + (lane & 31);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = n + 8 * q + 4 * (lane >> 5);
          if constexpr (MODE == kSmallLast) {
            const float alpha = p.move * p.lift[b];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int col = cb * 64 + c + e;
              if (r >= p.g.s || col >= p.g.l) continue;
              float* const at = p.tab.out[b] + (p.g.turned ? int64_t(col) * p.g.cols + r : int64_t(r) * p.g.cols + col);
              const float f = v[4 * q + e] * alpha;
              *at = p.up.muon ? *at * p.decay - p.step * f : f;
            }
          } else {
            const half4 h = *reinterpret_cast<const half4*>(x_at(0, c >> 3, r) + (c & 7) * 2);
            const half4 l = *reinterpret_cast<const half4*>(x_at(1, c >> 3, r) + (c & 7) * 2);
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = p.move * v[4 * q + e] + p.keep * (float(h[e]) + float(l[e]));
            split4(o, moved[q][0], moved[q][1]);
          }
        }
      }
      if constexpr (MODE == kSmallNext) {
        __syncthreads();
        const int r = m + (lane & 31);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = n + 8 * q + 4 * (lane >> 5);
          _Float16* const at = x + (int64_t(cb * 8 + (c >> 3)) * SP + r) * 8 + (c & 7);
#pragma unroll
          for (int pl = 0; pl < 2; ++pl) {
            *reinterpret_cast<half4*>(x_at(pl, c >> 3, r) + (c & 7) * 2) = moved[q][pl];
            *reinterpret_cast<half4*>(at + pl * plane) = moved[q][pl];
          }
        }
        __syncthreads();
      }
    }
    if constexpr (MODE != kSmallLast) {
      if (mine) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          half8 fa[2], fb[2];
#pragma unroll
          for (int pl = 0; pl < 2; ++pl) {
            fa[pl] = *reinterpret_cast<const half8*>(x_at(pl, 2 * ks + (lane >> 5), 32 * fr + (lane & 31)));
            fb[pl] = *reinterpret_cast<const half8*>(x_at(pl, 2 * ks + (lane >> 5), 32 * fc + (lane & 31)));
          }
          mul(acc, fb, fa);
        }
      }
    }
    __syncthreads();
  }
  if constexpr (MODE != kSmallLast) {
    if (mine) {
      f32x4* const at = reinterpret_cast<f32x4*>(p.to) + ((int64_t(b) * nw + j) * NF + wave) * 256 + lane;
#pragma unroll
      for (int q = 0; q < 4; ++q) at[q * 64] = f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    }
  }
}

template <class T, int KIND>
int launch(const StepArgs& p, int tiles, hipStream_t s) {
  const int rest = tiles - p.share.whole;
  hipLaunchKernelGGL((step_kernel<T, KIND>), dim3(unsigned(p.share.whole + rest * p.share.parts)), dim3(T::THREADS), 0, s, p);
  MX_LAUNCHED();
  if (rest) {
    hipLaunchKernelGGL((join_kernel<T, KIND>), dim3(unsigned(rest * T::WAVES * T::FM * T::FN)), dim3(64), 0, s, p);
    MX_LAUNCHED();
  }
  return MX_OK;
}

template <class T>
int launch_kind(int kind, const StepArgs& p, int tiles, hipStream_t s) {
  switch (kind) {
    case kGram: return launch<T, kGram>(p, tiles, s);
    case kPoly: return launch<T, kPoly>(p, tiles, s);
    case kNext: return launch<T, kNext>(p, tiles, s);
    case kLast: return launch<T, kLast>(p, tiles, s);
    default: return launch<T, kLastRows>(p, tiles, s);
  }
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Tiles of a set's products (the symmetric ones and the others), what its sides
// are padded to, and how the tiles are dealt.
// Over 25 sets from one 64 x 100 to 16 x 1024^2 and 4096^2, all sixteen pairs of
// tiles timed, the choice takes 3.5% more than the best on average, 11% at most
// (one 1024 x 4096: 377 us, 339 with 128 x 128 tiles throughout).
struct Plan {
  Geometry g;
  int sym, next;  // indexes into kTiles
  Deal gram, poly, update;
  int64_t sums;   // bytes of partial sums
  int wide;       // one launch a step, this many workgroups a matrix; 0: by products
};

// Sets of one launch a step, microseconds by products / so: one 32 x 32 61 / 35,
// one 64 x 100 61 / 39, one 64 x 4096 97 / 85, sixteen 64 x 4096 132 / 112, forty
// 64 x 2048 142 / 156.  (128 rows in one workgroup's LDS the same way: one 100 x
// 128 68 / 84, one 128 x 4096 103 / 291.)
bool use_small(int64_t s, int64_t l, int64_t batch) { return s <= kSmall && l * batch <= 65536; }

Plan plan_set(int64_t rows, int64_t cols, int64_t batch) {
  Plan best{};
  double least = -1;
  const int64_t cu = cu_count(), s = std::min(rows, cols), l = std::max(rows, cols);
  if (use_small(s, l, batch)) {
    Geometry& g = best.g;
    g.rows = int(rows);
    g.cols = int(cols);
    g.turned = rows > cols;
    g.s = int(s);
    g.l = int(l);
    g.sp = kSmall;
    g.lp = int(up(l, 64));
    best.wide = std::min(g.lp / 64, kSmallWide);
    best.sums = 2 * batch * best.wide * 3 * 4096;  // of two launches, three fragments a workgroup
    return best;
  }
  for (int i = 0; i < kTileCount; ++i)
    for (int j = 0; j < kTileCount; ++j) {
      const TileCost &a = kTiles[i], &c = kTiles[j];
      const int pad = std::max(a.tile, c.tile);
      const int64_t sp = up(s, pad), lp = up(l, pad), n = sp / a.tile;
      Plan p{};
      p.g.rows = int(rows);
      p.g.cols = int(cols);
      p.g.turned = rows > cols;
      p.g.s = int(s);
      p.g.l = int(l);
      p.g.sp = int(sp);
      p.g.lp = int(lp);
      p.sym = i;
      p.next = j;
      p.gram = deal(a, n * (n + 1) / 2 * batch, lp / kBK, cu);
      p.poly = deal(a, n * (n + 1) / 2 * batch, sp / kBK, cu);
      p.update = deal(c, (sp / c.tile) * (lp / c.tile) * batch, sp / kBK, cu);
      const double time = p.gram.time + p.poly.time + p.update.time;
      if (least >= 0 && time >= least) continue;
      least = time;
      p.sums = std::max({p.gram.sum_bytes(a.tile), p.poly.sum_bytes(a.tile), p.update.sum_bytes(c.tile)});
      best = p;
    }
  return best;
}

// Scratch of a set of `batch` matrices: X twice, G, P, the squares and the
// partial sums.
int64_t head_bytes(int64_t batch) { return up(batch * (kNormParts * 8 + 4), 256); }
int64_t set_bytes(const Plan& p, int64_t batch) {
  if (p.wide) return batch * p.g.x_plane() * 4 + head_bytes(batch) + p.sums;
  return batch * (2 * p.g.x_plane() * 4 + 2 * p.g.g_plane() * 4) + head_bytes(batch) + p.sums;
}

// Matrices of one shape that go through the launches together.
struct Set {
  int64_t rows, cols;
  std::vector<int64_t> at;
};

template <class Shape>
std::vector<Set> sets_of(int64_t count, Shape&& shape) {
  std::vector<Set> sets;
  std::vector<size_t> open;  // one set per shape that still takes matrices
  for (int64_t i = 0; i < count; ++i) {
    int64_t rows, cols;
    shape(i, &rows, &cols);
    if (rows == 0 || cols == 0) continue;
    size_t at = open.size();
    for (size_t k = 0; k < open.size(); ++k)
      if (sets[open[k]].rows == rows && sets[open[k]].cols == cols) at = k;
    if (at == open.size()) {
      open.push_back(sets.size());
      sets.push_back({rows, cols, {}});
    } else {
      // Padding is at most a 256-row tile a side.
      const int64_t next = int64_t(sets[open[at]].at.size()) + 1, sp = up(std::min(rows, cols), 256);
      if (next > kBatch || next * 8 * sp * (up(std::max(rows, cols), 256) + sp) > kMaxScratch) {
        open[at] = sets.size();
        sets.push_back({rows, cols, {}});
      }
    }
    sets[open[at]].at.push_back(i);
  }
  return sets;
}

int64_t workspace_of(const std::vector<Set>& sets) {
  int64_t most = 0;
  for (const Set& f : sets) {
    const int64_t n = int64_t(f.at.size());
    most = std::max(most, set_bytes(plan_set(f.rows, f.cols, n), n));
  }
  return most;
}

// Scales of an iteration's pieces from bounds on its singular values, and what
// |X| can grow by from it to the end while it is small.
struct Scales {
  float x, g, p;
  double growth;
};
constexpr double kMostBound = 0x1p40;

float scale_for(double bound) {
  // The largest power of two that keeps bound (and 5% for rounding) below 60000.
  return float(std::exp2(std::floor(std::log2(60000.0 / (1.05 * std::max(bound, 0x1p-40))))));
}

// Bounds of X, G and P before and through each iteration, for singular values in
// [0, B]: X's is B, G's B^2.  P holds b t + c t^2 (t = sigma^2), and a besides in
// the last iteration; the next B is the largest of |sigma (a + b t + c t^2)|.
// Each is reached at an end or where the derivative vanishes.  What P holds without
// a can be the larger: of a = 1, b = -2 it is 2 where a + b t stays within 1.
int scales_of(const char* who, const mx_newton_schulz& ns, std::vector<Scales>* out) {
  const auto poly = [&](double t) { return ns.a + t * (ns.b + t * ns.c); };
  double b = 1.0;
  for (int64_t i = 0; i < ns.steps; ++i) {
    const double t1 = b * b, held = i + 1 < ns.steps ? ns.a : 0.0;  // what P leaves to the update
    double q = std::max(std::fabs(poly(0)), std::fabs(poly(t1))), n = b * std::fabs(poly(t1));
    double stored = std::max(std::fabs(poly(0) - held), std::fabs(poly(t1) - held));
    const auto inside = [&](double t) { return t > 0 && t < t1; };
    if (ns.c != 0) {
      const double turn = -ns.b / (2 * ns.c);
      if (inside(turn)) {
        q = std::max(q, std::fabs(poly(turn)));
        stored = std::max(stored, std::fabs(poly(turn) - held));
      }
      const double disc = 9 * ns.b * ns.b - 20 * ns.a * ns.c;  // a + 3 b t + 5 c t^2 = 0
      for (const double sign : {1.0, -1.0}) {
        const double t = disc >= 0 ? (-3 * ns.b + sign * std::sqrt(disc)) / (10 * ns.c) : -1.0;
        if (inside(t)) n = std::max(n, std::sqrt(t) * std::fabs(poly(t)));
      }
    } else if (ns.b != 0) {
      const double t = -ns.a / (3 * ns.b);
      if (inside(t)) n = std::max(n, std::sqrt(t) * std::fabs(poly(t)));
    }
    MX_REQUIRE(std::isfinite(q) && std::isfinite(n) && std::isfinite(stored) && q < kMostBound && n < kMostBound, MX_ERR_INVALID,
               who, ": the iterations diverge (step ", i, ")");
    out->push_back({scale_for(b), scale_for(t1), scale_for(stored), std::max(1.0, q)});
    b = n;
  }
  for (size_t i = out->size(); i-- > 1;) (*out)[i - 1].growth *= (*out)[i].growth;
  // A lifted X meets the scales of later iterations, which are larger where the
  // bounds shrink.
  double finest = 1;
  for (const Scales& c : *out) finest = std::max(finest, double(c.x) / (*out)[0].x);
  if (!out->empty()) (*out)[0].growth *= finest;
  return MX_OK;
}

int check_ns(const char* who, const mx_newton_schulz& ns) {
  MX_REQUIRE(ns.steps >= 0 && ns.steps <= 1000, MX_ERR_INVALID, who, ": steps must lie in [0, 1000], got ", ns.steps);
  MX_REQUIRE(std::isfinite(ns.a) && std::isfinite(ns.b) && std::isfinite(ns.c), MX_ERR_INVALID, who,
             ": coefficients must be finite");
  MX_REQUIRE(ns.eps > 0 && std::isfinite(ns.eps), MX_ERR_INVALID, who, ": eps must be positive");
  return MX_OK;
}

int check_shape(const char* who, int64_t i, int64_t rows, int64_t cols) {
  MX_REQUIRE(rows >= 0 && cols >= 0, MX_ERR_INVALID, who, ": negative size at ", i);
  // Byte offsets within a plane's groups of eight columns stay in int32.
  MX_REQUIRE(rows <= (1 << 24) && cols <= (1 << 24), MX_ERR_INVALID, who, ": side longer than 2^24 at ", i);
  return MX_OK;
}

struct Finish {
  Update up;
  double lr, decay;
  int adjust;
};

// All launches of one set; `ws` holds set_bytes.
int run_set(const Table& tab, int64_t batch, const Plan& plan, const mx_newton_schulz& ns, const std::vector<Scales>& sc,
            const Finish& fin, char* ws, hipStream_t s) {
  const Geometry& g = plan.g;
  double* const parts = reinterpret_cast<double*>(ws);
  float* const lift = reinterpret_cast<float*>(parts + batch * kNormParts);
  _Float16* x = reinterpret_cast<_Float16*>(ws + head_bytes(batch));
  _Float16* x2 = x + batch * 2 * g.x_plane();
  _Float16* const gram = x2 + batch * 2 * g.x_plane();
  _Float16* const poly = gram + batch * 2 * g.g_plane();
  const int64_t numel = int64_t(g.rows) * g.cols;
  // Four 16-byte loads a thread, up to eight workgroups a CU over the set.
  const int64_t most = std::min<int64_t>(kNormParts, std::max<int64_t>(1, int64_t(cu_count()) * 8 / batch));
  const int nparts = int(std::min<int64_t>(most, (numel + 4095) / 4096));
  const double r = fin.adjust == MX_MUON_MATCH_RMS_ADAMW ? 0.2 * std::sqrt(double(std::max(g.rows, g.cols)))
                                                         : std::sqrt(std::max(1.0, double(g.rows) / g.cols));
  const float decay = float(1.0 - fin.lr * fin.decay), step = float(fin.lr * r);
  bool vec = true;
  for (int64_t i = 0; i < batch; ++i)
    vec = vec && ((reinterpret_cast<uintptr_t>(tab.in[i]) | reinterpret_cast<uintptr_t>(tab.buf[i])) & 15) == 0;
  if (vec)
    hipLaunchKernelGGL(norm_kernel<true>, dim3(unsigned(nparts), unsigned(batch)), dim3(256), 0, s, tab, fin.up, numel, parts);
  else
    hipLaunchKernelGGL(norm_kernel<false>, dim3(unsigned(nparts), unsigned(batch)), dim3(256), 0, s, tab, fin.up, numel, parts);
  MX_LAUNCHED();
  if (ns.steps == 0) {
    hipLaunchKernelGGL(scaled_kernel, dim3(unsigned(nparts), unsigned(batch)), dim3(256), 0, s, tab, fin.up, numel, parts,
                       nparts, ns.eps, decay, step);
    MX_LAUNCHED();
    return MX_OK;
  }
  if (plan.wide) {
    SmallArgs a{};
    a.tab = tab;
    a.up = fin.up;
    a.g = g;
    a.norms = parts;
    a.nparts = nparts;
    a.eps = ns.eps;
    a.growth = sc[0].growth;
    a.scale = sc[0].x;
    a.lift = lift;
    a.x = x;
    a.decay = decay;
    a.step = step;
    a.to = reinterpret_cast<float*>(x + batch * 2 * g.x_plane());
    a.from = a.to + plan.sums / 8;
    const auto run = [&](int mode) -> int {
      const dim3 grid(unsigned(plan.wide), unsigned(batch)), block(256);
      if (mode == kSmallFirst) hipLaunchKernelGGL(small_kernel<kSmallFirst>, grid, block, 0, s, a);
      if (mode == kSmallNext) hipLaunchKernelGGL(small_kernel<kSmallNext>, grid, block, 0, s, a);
      if (mode == kSmallLast) hipLaunchKernelGGL(small_kernel<kSmallLast>, grid, block, 0, s, a);
      MX_LAUNCHED();
      float* const was = a.to;
      a.to = const_cast<float*>(a.from);
      a.from = was;
      return MX_OK;
    };
    MX_TRY(run(kSmallFirst));
    for (int64_t i = 0; i < ns.steps; ++i) {
      const Scales c = sc[size_t(i)];
      const bool last = i + 1 == ns.steps;
      a.gram = c.g / c.x / c.x;
      a.alpha = float(ns.c) * (c.p / c.g / c.g);
      a.diag = last ? float(ns.a) * c.p : 0.f;
      a.lin = float(ns.b) * c.p;
      a.unit = 1.f / c.g;
      a.move = (last ? 1.f : sc[size_t(i) + 1].x) / c.p / c.x;
      a.keep = last ? 0.f : float(ns.a) * (sc[size_t(i) + 1].x / c.x);
      MX_TRY(run(last ? kSmallLast : kSmallNext));
    }
    return MX_OK;
  }
  hipLaunchKernelGGL(pack_kernel, dim3(unsigned(g.lp / 64), unsigned(g.sp / 32), unsigned(batch)), dim3(256), 0, s, tab,
                     fin.up, g, parts, nparts, ns.eps, sc[0].x, sc[0].growth, x, lift);
  MX_LAUNCHED();
  StepArgs p{};
  p.g = g;
  p.tab = tab;
  p.lift = lift;
  p.muon = fin.up.muon;
  p.decay = decay;
  p.step = step;
  p.share.sums = reinterpret_cast<float*>(poly + batch * 2 * g.g_plane());
  const auto run = [&](int kind, const Deal& d, int t) -> int {
    const int tile = kTiles[t].tile;
    p.share.whole = int(d.whole);
    p.share.parts = d.parts;
    p.tiles_m = g.sp / tile;
    p.tiles_n = (symmetric(kind) ? g.sp : g.lp) / tile;
    if (t == kTile64Deep) return launch_kind<Tile64Deep>(kind, p, int(d.tiles), s);
    if (t == kTile64) return launch_kind<Tile64>(kind, p, int(d.tiles), s);
    if (t == kTile128) return launch_kind<Tile128>(kind, p, int(d.tiles), s);
    return launch_kind<Tile256>(kind, p, int(d.tiles), s);
  };
  for (int64_t i = 0; i < ns.steps; ++i) {
    const Scales c = sc[size_t(i)];
    p.a = p.b = x;
    p.a_plane = p.b_plane = g.x_plane();
    p.a_rows = p.b_rows = p.out_rows = g.sp;
    p.out = gram;
    p.out_plane = g.g_plane();
    p.nk = g.lp / kBK;
    p.alpha = c.g / c.x / c.x;
    MX_TRY(run(kGram, plan.gram, plan.sym));
    p.a = p.b = gram;
    p.a_plane = p.b_plane = g.g_plane();
    p.out = poly;
    p.nk = g.sp / kBK;
    p.alpha = float(ns.c) * (c.p / c.g / c.g);
    const bool last = i + 1 == ns.steps;
    p.diag = last ? float(ns.a) * c.p : 0.f;
    p.lin = float(ns.b) * c.p;
    p.unit = 1.f / c.g;
    MX_TRY(run(kPoly, plan.poly, plan.sym));
    p.a = poly;
    p.b = x;
    p.b_plane = p.out_plane = g.x_plane();
    p.out = x2;
    p.keep = last ? 0.f : float(ns.a) * (sc[size_t(i) + 1].x / c.x);
    p.alpha = (last ? 1.f : sc[size_t(i) + 1].x) / c.p / c.x;
    MX_TRY(run(!last ? kNext : g.turned ? kLast : kLastRows, plan.update, plan.next));
    std::swap(x, x2);
  }
  return MX_OK;
}

// Buffers of a call, which runs its matrices side by side and a set after the other:
// what it writes may not overlap anything else of it.
struct Buffer {
  uintptr_t at, end;
  int64_t matrix;
  bool written;
};
void add(std::vector<Buffer>* list, const float* p, int64_t rows, int64_t cols, int64_t matrix, bool written) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  if (rows > 0 && cols > 0) list->push_back({at, at + uintptr_t(rows) * uintptr_t(cols) * sizeof(float), matrix, written});
}
int check_apart(const char* who, std::vector<Buffer>* list) {
  std::sort(list->begin(), list->end(), [](const Buffer& a, const Buffer& b) { return a.at < b.at; });
  // The one that reaches furthest of those before, of all and of the written ones.
  const Buffer *any = nullptr, *out = nullptr;
  for (const Buffer& b : *list) {
    const Buffer* const over = b.written ? any : out;
    MX_REQUIRE(!over || over->end <= b.at, MX_ERR_INVALID, who, ": a written tensor appears twice or overlaps another (matrices ",
               over->matrix, " and ", b.matrix, ")");
    if (!any || b.end > any->end) any = &b;
    if (b.written && (!out || b.end > out->end)) out = &b;
  }
  return MX_OK;
}

template <class Fill>
int run_all(const char* who, const std::vector<Set>& sets, const mx_newton_schulz& ns, const Finish& fin, std::vector<Buffer>* buffers,
            void* workspace, int64_t workspace_bytes, hipStream_t s, Fill&& fill) {
  std::vector<Scales> sc;
  MX_TRY(scales_of(who, ns, &sc));
  Workspace ws;
  MX_TRY(ws.take(who, workspace, workspace_bytes, workspace_of(sets), s));
  MX_TRY(check_apart(who, buffers));
  for (const Set& f : sets) {
    const int64_t batch = int64_t(f.at.size());
    Table tab{};
    for (int64_t i = 0; i < batch; ++i) fill(f.at[size_t(i)], &tab, i);
    MX_TRY(run_set(tab, batch, plan_set(f.rows, f.cols, batch), ns, sc, fin, ws.as<char>(), s));
  }
  return MX_OK;
}

std::vector<Set> sets_of(const mx_matrix_pair* t, int64_t n) {
  return sets_of(n, [&](int64_t i, int64_t* r, int64_t* c) { *r = t[i].rows, *c = t[i].cols; });
}
std::vector<Set> sets_of(const mx_muon_tensor* t, int64_t n) {
  return sets_of(n, [&](int64_t i, int64_t* r, int64_t* c) { *r = t[i].rows, *c = t[i].cols; });
}

template <class E>
int check_list(const char* who, const E* t, int64_t count) {
  MX_REQUIRE(count >= 0, MX_ERR_INVALID, who, ": negative count");
  MX_REQUIRE(count == 0 || t, MX_ERR_INVALID, who, ": null list");
  for (int64_t i = 0; i < count; ++i) MX_TRY(check_shape(who, i, t[i].rows, t[i].cols));
  return MX_OK;
}

}  // namespace
}  // namespace mx

using namespace mx;

extern "C" int mx_orthogonalize_workspace(const mx_matrix_pair* matrices, int64_t count, int64_t* bytes) {
  MX_ABI_BEGIN
  MX_TRY(check_list("mx_orthogonalize", matrices, count));
  MX_REQUIRE(bytes, MX_ERR_INVALID, "mx_orthogonalize_workspace: null result");
  *bytes = workspace_of(sets_of(matrices, count));
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_orthogonalize_variant(int64_t rows, int64_t cols, int64_t count, char* buf, size_t len) {
  MX_ABI_BEGIN
  const char* const who = "mx_orthogonalize_variant";
  MX_TRY(check_shape(who, 0, rows, cols));
  MX_REQUIRE(count >= 0 && count <= kBatch && (buf || !len), MX_ERR_INVALID, who, ": count must lie in [0, ", kBatch, "]");
  std::string name = "none";
  if (rows > 0 && cols > 0 && count > 0) {
    const Plan p = plan_set(rows, cols, count);
    const auto product = [](const char* what, const Deal& d, int t) {
      return cat(what, "<", kTiles[t].tile, t == kTile64Deep ? ",deep>" : ">", d.whole, d.tiles > d.whole ? cat("+", d.tiles - d.whole, "x", d.parts) : "");
    };
    name = p.wide ? cat("one_launch<", p.wide, ">")
                  : product("gram", p.gram, p.sym) + product(" poly", p.poly, p.sym) + product(" update", p.update, p.next);
  }
  copy_name(name, buf, len);
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_orthogonalize(const mx_matrix_pair* matrices, int64_t count, const mx_newton_schulz* ns, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  const char* const who = "mx_orthogonalize";
  MX_REQUIRE(ns, MX_ERR_INVALID, who, ": null parameters");
  MX_TRY(check_ns(who, *ns));
  MX_TRY(check_list(who, matrices, count));
  for (int64_t i = 0; i < count; ++i)
    MX_REQUIRE(matrices[i].rows == 0 || matrices[i].cols == 0 || (matrices[i].in && matrices[i].out), MX_ERR_INVALID, who,
               ": null buffer at ", i);
  std::vector<Buffer> buffers;
  for (int64_t i = 0; i < count; ++i) {
    const mx_matrix_pair& t = matrices[i];
    add(&buffers, t.out, t.rows, t.cols, i, true);
    if (t.in != t.out) add(&buffers, t.in, t.rows, t.cols, i, false);
  }
  return run_all(who, sets_of(matrices, count), *ns, Finish{}, &buffers, workspace, workspace_bytes, resolve_stream(stream),
                 [&](int64_t i, Table* tab, int64_t at) {
                   tab->in[at] = matrices[i].in;
                   tab->out[at] = matrices[i].out;
                 });
  MX_ABI_END
}

extern "C" int mx_muon_workspace(const mx_muon_tensor* tensors, int64_t count, int64_t* bytes) {
  MX_ABI_BEGIN
  MX_TRY(check_list("mx_muon_step", tensors, count));
  MX_REQUIRE(bytes, MX_ERR_INVALID, "mx_muon_workspace: null result");
  *bytes = workspace_of(sets_of(tensors, count));
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_muon_step(const mx_muon_tensor* tensors, int64_t count, const mx_muon_hparams* hp, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  const char* const who = "mx_muon_step";
  MX_REQUIRE(hp, MX_ERR_INVALID, who, ": null hyperparameters");
  MX_REQUIRE(hp->lr >= 0 && hp->weight_decay >= 0 && hp->momentum >= 0 && hp->momentum <= 1 && std::isfinite(hp->lr) &&
                 std::isfinite(hp->weight_decay),
             MX_ERR_INVALID, who, ": invalid hyperparameters");
  MX_REQUIRE(hp->adjust_lr == MX_MUON_ORIGINAL || hp->adjust_lr == MX_MUON_MATCH_RMS_ADAMW, MX_ERR_INVALID, who,
             ": unknown learning rate adjustment ", hp->adjust_lr);
  MX_TRY(check_ns(who, hp->ns));
  MX_TRY(check_list(who, tensors, count));
  for (int64_t i = 0; i < count; ++i)
    MX_REQUIRE(tensors[i].rows == 0 || tensors[i].cols == 0 ||
                   (tensors[i].param && tensors[i].grad && tensors[i].momentum_buffer),
               MX_ERR_INVALID, who, ": null buffer at ", i);
  std::vector<Buffer> buffers;
  for (int64_t i = 0; i < count; ++i) {
    const mx_muon_tensor& t = tensors[i];
    add(&buffers, t.param, t.rows, t.cols, i, true);
    add(&buffers, t.momentum_buffer, t.rows, t.cols, i, true);
    add(&buffers, t.grad, t.rows, t.cols, i, false);
  }
  Finish fin{};
  fin.up = {1, hp->nesterov != 0, float(hp->momentum), float(1.0 - hp->momentum)};
  fin.lr = hp->lr;
  fin.decay = hp->weight_decay;
  fin.adjust = hp->adjust_lr;
  return run_all(who, sets_of(tensors, count), hp->ns, fin, &buffers, workspace, workspace_bytes, resolve_stream(stream),
                 [&](int64_t i, Table* tab, int64_t at) {
                   tab->in[at] = tensors[i].grad;
                   tab->buf[at] = tensors[i].momentum_buffer;
                   tab->out[at] = tensors[i].param;
                 });
  MX_ABI_END
}
