// Orthogonalised momentum: Newton-Schulz iterations on the matrices of one
// shape side by side, and the optimizer step around them (FP32).
//
//   X = U / max(|U|_F, eps), U turned so that its shorter side is the rows
//   steps times:  G = X X^T,  P = a I + b G + c G^2,  X = P X
//   out = X, or  param = param (1 - lr wd) - lr r X
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

constexpr int kBatch = 48;      // matrices of one set of launches
constexpr int kNormParts = 64;  // partial squares of one matrix
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
// vanish at 2^-75), and the new momentum.
__global__ __launch_bounds__(256) void norm_kernel(Table tab, Update up, int64_t numel, double* parts) {
  __shared__ double sum[4];
  const int b = blockIdx.y;
  const float* const in = tab.in[b];
  float* const buf = tab.buf[b];
  double s = 0;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < numel; i += int64_t(gridDim.x) * 256) {
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

struct Geometry {
  int rows, cols;     // of U
  int s, l;           // shorter and longer side
  int sp, lp;         // padded
  bool turned;        // X = U^T
  int64_t x_plane() const { return int64_t(sp) * lp; }
  int64_t g_plane() const { return int64_t(sp) * sp; }
};

// X's pieces: 32 rows of X and 64 of its columns to a workgroup, eight columns
// of a row to a thread.
__global__ __launch_bounds__(256) void pack_kernel(Table tab, Update up, Geometry g, const double* parts, int nparts,
                                                   double eps, float scale, double growth, _Float16* x,
                                                   float* lift) {
  __shared__ double inv;
  const int b = blockIdx.z;
  if (threadIdx.x < 64) {
    double s = int(threadIdx.x) < nparts ? parts[b * kNormParts + threadIdx.x] : 0.0;
    for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
    const double n = sqrt(s);
    if (threadIdx.x == 0) {
      // |X|_F is 1, unless eps is what divides: then X is kept times 2^e, which
      // no iteration's growth takes past the bounds, so that fp16 holds it.
      const double d = n < eps ? eps : n, small = n / d * growth;
      const int e = small > 0 && small < 1 ? int(floor(-log2(small))) : 0;
      inv = ldexp(double(scale), e) / d;
      if (blockIdx.x == 0 && blockIdx.y == 0) lift[b] = float(ldexp(1.0, -e));
    }
  }
  __syncthreads();
  const float* const in = tab.in[b];
  const float* const buf = tab.buf[b];
  const int row = blockIdx.y * 32 + (threadIdx.x & 31), col = blockIdx.x * 64 + (threadIdx.x >> 5) * 8;
  half8 hi, lo;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v = 0.f;
    if (row < g.s && col + e < g.l) {
      const int64_t at = g.turned ? int64_t(col + e) * g.cols + row : int64_t(row) * g.cols + col + e;
      float u = in[at];
      if (up.muon) u = up.u(buf[at], u);
      v = float(double(u) * inv);
    }
    hi[e] = _Float16(v);
    lo[e] = _Float16(v - float(hi[e]));
  }
  const int64_t plane = int64_t(g.sp) * g.lp;
  _Float16* const to = x + b * 2 * plane + (int64_t(col >> 3) * g.sp + row) * 8;
  *reinterpret_cast<half8*>(to) = hi;
  *reinterpret_cast<half8*>(to + plane) = lo;
}

enum Kind { kGram, kPoly, kNext, kLast };

struct StepArgs {
  const _Float16 *a, *b;  // operands (kPoly: both G)
  _Float16* out;          // pieces of the result
  int64_t a_plane, b_plane, out_plane;
  int a_rows, b_rows, out_rows;
  int nk;                 // slabs
  int tiles_m, tiles_n, batch;
  float alpha;            // product of pieces -> stored value
  float diag, lin, unit;  // kPoly: a, b and 1 / G's scale, times the stored scale
  const float* lift;      // X's pieces hold X / lift[matrix]
  // kLast
  Table tab;
  Geometry g;
  int muon;
  float decay, step;      // 1 - lr wd, lr r
};

template <class T, int KIND>
__global__ __launch_bounds__(T::THREADS) __attribute__((amdgpu_waves_per_eu(T::OCC, T::OCC))) void step_kernel(StepArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[T::SMEM];
  constexpr bool COLS = KIND == kNext || KIND == kLast;
  const int per = p.tiles_m * p.tiles_n;
  const int id = mfma::xcd_remap(blockIdx.x, per * p.batch), b = id / per;
  int tm, tn;
  mfma::tile_coords(id - b * per, p.tiles_m, p.tiles_n, tm, tn);
  const int m0 = tm * T::BM, n0 = tn * T::BN;
  const Planes pa{const_cast<_Float16*>(p.a) + b * 2 * p.a_plane, p.a_plane, p.a_rows};
  const Planes pb{const_cast<_Float16*>(p.b) + b * 2 * p.b_plane, p.b_plane, p.b_rows};
  f32x16 acc[T::FM][T::FN];
  product<T, COLS>(acc, pa, pb, m0, n0, p.nk, smem);
  // G's pieces hold G itself: where X is tiny, all of it that b G and c G^2 add
  // to a I lies below what G's scale can hold.
  float alpha = p.alpha;
  if constexpr (KIND == kGram) alpha *= p.lift[b] * p.lift[b];
  if constexpr (KIND == kLast) alpha *= p.lift[b];
  if constexpr (KIND == kLast) {
    float* const out = p.tab.out[b];
    for_each4<T>(acc, [&](int m, int n, const float(&v)[4]) {
      const int r = m0 + m, c = n0 + n;
      if (r >= p.g.s) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c + e >= p.g.l) break;
        const int64_t at = p.g.turned ? int64_t(c + e) * p.g.cols + r : int64_t(r) * p.g.cols + c + e;
        const float x = v[e] * alpha;
        out[at] = p.muon ? out[at] * p.decay - p.step * x : x;
      }
    });
  } else {
    const Planes po{p.out + b * 2 * p.out_plane, p.out_plane, p.out_rows};
    for_each4<T>(acc, [&](int m, int n, const float(&v)[4]) {
      const int r = m0 + m, c = n0 + n;
      const int64_t at = elem(po, r, c);
      float o[4];
      if constexpr (KIND == kPoly) {
        const half4 gh = *reinterpret_cast<const half4*>(pa.at + at), gl = *reinterpret_cast<const half4*>(pa.at + pa.plane + at);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[e] = (r == c + e ? p.diag : 0.f) + p.lin * ((float(gh[e]) + float(gl[e])) * p.unit) + alpha * v[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = alpha * v[e];
      }
      half4 hi, lo;
      split4(o, hi, lo);
      *reinterpret_cast<half4*>(po.at + at) = hi;
      *reinterpret_cast<half4*>(po.at + po.plane + at) = lo;
    });
  }
}

// steps == 0: the scaled matrix itself.
__global__ __launch_bounds__(256) void scaled_kernel(Table tab, Update up, int64_t numel, const double* parts, int nparts,
                                                     double eps, float decay, float step) {
  __shared__ double inv;
  const int b = blockIdx.y;
  if (threadIdx.x < 64) {
    double s = int(threadIdx.x) < nparts ? parts[b * kNormParts + threadIdx.x] : 0.0;
    for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
    const double n = sqrt(s);
    if (threadIdx.x == 0) inv = 1.0 / (n < eps ? eps : n);
  }
  __syncthreads();
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < numel; i += int64_t(gridDim.x) * 256) {
    float u = tab.in[b][i];
    if (up.muon) u = up.u(tab.buf[b][i], u);
    const float x = float(double(u) * inv);
    tab.out[b][i] = up.muon ? tab.out[b][i] * decay - step * x : x;
  }
}

using Tile64 = Tile<64, 64, 2, 2, 4, 2>;     // 4 waves of 32 x 32
using Tile128 = Tile<128, 128, 2, 2, 2, 2>;  // 4 waves of 64 x 64
using Tile256 = Tile<256, 256, 2, 4, 2, 2>;  // 8 waves of 128 x 64

template <class T>
int launch(int kind, StepArgs& p, int m, int n, hipStream_t s) {
  p.tiles_m = m / T::BM;
  p.tiles_n = n / T::BN;
  const dim3 grid(unsigned(p.tiles_m * p.tiles_n * p.batch)), block(T::THREADS);
  switch (kind) {
    case kGram: hipLaunchKernelGGL((step_kernel<T, kGram>), grid, block, 0, s, p); break;
    case kPoly: hipLaunchKernelGGL((step_kernel<T, kPoly>), grid, block, 0, s, p); break;
    case kNext: hipLaunchKernelGGL((step_kernel<T, kNext>), grid, block, 0, s, p); break;
    default: hipLaunchKernelGGL((step_kernel<T, kLast>), grid, block, 0, s, p);
  }
  MX_HIP(hipGetLastError());
  return MX_OK;
}

int launch_tile(int tile, int kind, StepArgs& p, int m, int n, hipStream_t s) {
  if (tile == 256) return launch<Tile256>(kind, p, m, n, s);
  if (tile == 128) return launch<Tile128>(kind, p, m, n, s);
  return launch<Tile64>(kind, p, m, n, s);
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Tile of a set: the largest that still gives every CU work in the smaller
// products (G and P have s x s entries).
int pick_tile(int64_t s, int64_t batch) {
  const auto tiles = [&](int64_t t) { return up(s, t) / t * (up(s, t) / t) * batch; };
  const int64_t cu = cu_count();
  if (tiles(256) >= cu) return 256;
  if (tiles(128) >= cu) return 128;
  return 64;
}

Geometry geometry(int64_t rows, int64_t cols, int tile) {
  Geometry g{};
  g.rows = int(rows);
  g.cols = int(cols);
  g.turned = rows > cols;
  g.s = int(std::min(rows, cols));
  g.l = int(std::max(rows, cols));
  g.sp = int(up(g.s, tile));
  g.lp = int(up(g.l, tile));
  return g;
}

// Scratch of a set of `batch` matrices: X twice, G, P, and the squares.
int64_t set_bytes(const Geometry& g, int64_t batch) {
  return batch * (2 * g.x_plane() * 4 + 2 * g.g_plane() * 4) + up(batch * (kNormParts * 8 + 4), 256);
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
      const Set& f = sets[open[at]];
      const int64_t next = int64_t(f.at.size()) + 1;
      if (next > kBatch || set_bytes(geometry(rows, cols, 256), next) > kMaxScratch) {
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
    most = std::max(most, set_bytes(geometry(f.rows, f.cols, pick_tile(std::min(f.rows, f.cols), n)), n));
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

// Bounds of X, G and P before and through each iteration: the largest of
// |sigma (a + b sigma^2 + c sigma^4)| on [0, B] is at an end or where the
// derivative vanishes.
int scales_of(const char* who, const mx_newton_schulz& ns, std::vector<Scales>* out) {
  const auto poly = [&](double t) { return ns.a + t * (ns.b + t * ns.c); };
  double b = 1.0;
  for (int64_t i = 0; i < ns.steps; ++i) {
    const double t1 = b * b;
    double q = std::max(std::fabs(poly(0)), std::fabs(poly(t1))), n = b * std::fabs(poly(t1));
    const auto at = [&](double t, bool deriv) {
      if (!(t > 0 && t < t1)) return;
      if (deriv)
        n = std::max(n, std::sqrt(t) * std::fabs(poly(t)));
      else
        q = std::max(q, std::fabs(poly(t)));
    };
    if (ns.c != 0) {
      at(-ns.b / (2 * ns.c), false);
      const double disc = 9 * ns.b * ns.b - 20 * ns.a * ns.c;  // a + 3 b t + 5 c t^2 = 0
      if (disc >= 0) {
        at((-3 * ns.b + std::sqrt(disc)) / (10 * ns.c), true);
        at((-3 * ns.b - std::sqrt(disc)) / (10 * ns.c), true);
      }
    } else if (ns.b != 0) {
      at(-ns.a / (3 * ns.b), true);
    }
    MX_REQUIRE(std::isfinite(q) && std::isfinite(n) && q < kMostBound && n < kMostBound, MX_ERR_INVALID, who,
               ": the iterations diverge (step ", i, ")");
    out->push_back({scale_for(b), scale_for(t1), scale_for(q), std::max(1.0, q)});
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
  // Tile counts and byte offsets within a plane's 16-byte groups stay in int32.
  MX_REQUIRE(rows <= (1 << 24) && cols <= (1 << 24), MX_ERR_INVALID, who, ": side longer than 2^24 at ", i);
  return MX_OK;
}

struct Finish {
  Update up;
  double lr, decay;
  int adjust;
};

// All launches of one set; `ws` holds set_bytes.
int run_set(const Table& tab, int64_t batch, const Geometry& g, int tile, const mx_newton_schulz& ns,
            const std::vector<Scales>& sc, const Finish& fin, char* ws, hipStream_t s) {
  double* const parts = reinterpret_cast<double*>(ws);
  float* const lift = reinterpret_cast<float*>(parts + batch * kNormParts);
  _Float16* x = reinterpret_cast<_Float16*>(ws + up(batch * (kNormParts * 8 + 4), 256));
  _Float16* x2 = x + batch * 2 * g.x_plane();
  _Float16* const gram = x2 + batch * 2 * g.x_plane();
  _Float16* const poly = gram + batch * 2 * g.g_plane();
  const int64_t numel = int64_t(g.rows) * g.cols;
  const int nparts = int(std::min<int64_t>(kNormParts, std::max<int64_t>(1, (numel + 2047) / 2048)));
  const double r = fin.adjust == MX_MUON_MATCH_RMS_ADAMW ? 0.2 * std::sqrt(double(std::max(g.rows, g.cols)))
                                                         : std::sqrt(std::max(1.0, double(g.rows) / g.cols));
  const float decay = float(1.0 - fin.lr * fin.decay), step = float(fin.lr * r);
  hipLaunchKernelGGL(norm_kernel, dim3(unsigned(nparts), unsigned(batch)), dim3(256), 0, s, tab, fin.up, numel, parts);
  MX_HIP(hipGetLastError());
  if (ns.steps == 0) {
    hipLaunchKernelGGL(scaled_kernel, dim3(unsigned(nparts), unsigned(batch)), dim3(256), 0, s, tab, fin.up, numel, parts,
                       nparts, ns.eps, decay, step);
    MX_HIP(hipGetLastError());
    return MX_OK;
  }
  hipLaunchKernelGGL(pack_kernel, dim3(unsigned(g.lp / 64), unsigned(g.sp / 32), unsigned(batch)), dim3(256), 0, s, tab,
                     fin.up, g, parts, nparts, ns.eps, sc[0].x, sc[0].growth, x, lift);
  MX_HIP(hipGetLastError());
  StepArgs p{};
  p.batch = int(batch);
  p.g = g;
  p.tab = tab;
  p.lift = lift;
  p.muon = fin.up.muon;
  p.decay = decay;
  p.step = step;
  for (int64_t i = 0; i < ns.steps; ++i) {
    const Scales c = sc[size_t(i)];
    p.a = p.b = x;
    p.a_plane = p.b_plane = g.x_plane();
    p.a_rows = p.b_rows = p.out_rows = g.sp;
    p.out = gram;
    p.out_plane = g.g_plane();
    p.nk = g.lp / kBK;
    p.alpha = c.g / c.x / c.x;
    MX_TRY(launch_tile(tile, kGram, p, g.sp, g.sp, s));
    p.a = p.b = gram;
    p.a_plane = p.b_plane = g.g_plane();
    p.out = poly;
    p.nk = g.sp / kBK;
    p.alpha = float(ns.c) * (c.p / c.g / c.g);
    p.diag = float(ns.a) * c.p;
    p.lin = float(ns.b) * c.p;
    p.unit = 1.f / c.g;
    MX_TRY(launch_tile(tile, kPoly, p, g.sp, g.sp, s));
    p.a = poly;
    p.b = x;
    p.b_plane = p.out_plane = g.x_plane();
    p.out = x2;
    const bool last = i + 1 == ns.steps;
    p.alpha = (last ? 1.f : sc[size_t(i) + 1].x) / c.p / c.x;
    MX_TRY(launch_tile(tile, last ? kLast : kNext, p, g.sp, g.lp, s));
    std::swap(x, x2);
  }
  return MX_OK;
}

template <class Fill>
int run_all(const char* who, const std::vector<Set>& sets, const mx_newton_schulz& ns, const Finish& fin, void* workspace,
            int64_t workspace_bytes, hipStream_t s, Fill&& fill) {
  std::vector<Scales> sc;
  MX_TRY(scales_of(who, ns, &sc));
  Workspace ws;
  MX_TRY(ws.take(who, workspace, workspace_bytes, workspace_of(sets), s));
  for (const Set& f : sets) {
    const int64_t batch = int64_t(f.at.size());
    const int tile = pick_tile(std::min(f.rows, f.cols), batch);
    Table tab{};
    for (int64_t i = 0; i < batch; ++i) fill(f.at[size_t(i)], &tab, i);
    MX_TRY(run_set(tab, batch, geometry(f.rows, f.cols, tile), tile, ns, sc, fin, ws.as<char>(), s));
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

extern "C" int mx_orthogonalize(const mx_matrix_pair* matrices, int64_t count, const mx_newton_schulz* ns, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  const char* const who = "mx_orthogonalize";
  MX_REQUIRE(ns, MX_ERR_INVALID, who, ": null parameters");
  MX_TRY(check_ns(who, *ns));
  MX_TRY(check_list(who, matrices, count));
  for (int64_t i = 0; i < count; ++i)
    MX_REQUIRE(matrices[i].rows == 0 || matrices[i].cols == 0 || (matrices[i].in && matrices[i].out), MX_ERR_INVALID, who,
               ": null buffer at ", i);
  return run_all(who, sets_of(matrices, count), *ns, Finish{}, workspace, workspace_bytes, resolve_stream(stream),
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
  Finish fin{};
  fin.up = {1, hp->nesterov != 0, float(hp->momentum), float(1.0 - hp->momentum)};
  fin.lr = hp->lr;
  fin.decay = hp->weight_decay;
  fin.adjust = hp->adjust_lr;
  return run_all(who, sets_of(tensors, count), hp->ns, fin, workspace, workspace_bytes, resolve_stream(stream),
                 [&](int64_t i, Table* tab, int64_t at) {
                   tab->in[at] = tensors[i].grad;
                   tab->buf[at] = tensors[i].momentum_buffer;
                   tab->out[at] = tensors[i].param;
                 });
  MX_ABI_END
}
