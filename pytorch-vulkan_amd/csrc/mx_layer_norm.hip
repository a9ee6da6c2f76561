// Layer normalisation over the last axis, forward and backward (FP32).
//
//   forward   mean = sum x / n,  var = sum (x - mean)^2 / n,  rstd = (var + eps)^-1/2
//             y = (x - mean) rstd gamma + beta
//   backward  g = dy gamma,  xh = (x - mean) rstd
//             dx = rstd (g - mean(g) - xh mean(g xh))
//             dgamma = sum_rows dy xh,  dbeta = sum_rows dy
//
// Both are bound by memory: the forward moves 8 bytes an element, the backward
// 12.  A row stays in the registers of the lanes that share it (16 lanes to a
// whole workgroup of 512 threads, chosen by the row's length), so x is read
// once although the variance is summed about the mean, and the backward's
// column sums ride along in registers from row to row.
//
// Every access is 16 bytes wide whatever the row length: the lane that holds a
// row's last elements reads the row's last four, and leaves those that its
// neighbour has too out of the sums (both write the same values).  Rows of odd
// length start at any multiple of four bytes, which global loads and stores take.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mx_internal.hpp"

namespace mx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// Sum over groups of L consecutive lanes (L a power of two up to 64).
template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int m = 1; m < L; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// The columns of one lane: V vectors of four, vector q at at(q), whose
// elements below skip(q) belong to the neighbour.
template <int L, int V>
struct Cols {
  int lane, cols;
  __device__ __forceinline__ int first(int q) const { return (q * L + lane) * 4; }
  __device__ __forceinline__ bool has(int q) const { return first(q) < cols; }
  __device__ __forceinline__ int at(int q) const { return min(first(q), cols - 4); }
  __device__ __forceinline__ int skip(int q) const { return has(q) ? first(q) - at(q) : 4; }
  __device__ __forceinline__ f32x4 load(const float* p, int q) const {
    return has(q) ? f32x4(*reinterpret_cast<const f32x4u*>(p + at(q))) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void store(float* p, int q, f32x4 v) const {
    if (has(q)) *reinterpret_cast<f32x4u*>(p + at(q)) = v;
  }
};

// A workgroup of B threads takes B / L rows at a time.  L <= 64: a row per
// group of L lanes.  L == B: a row per workgroup, whose waves exchange their
// sums through LDS, one barrier a row (the two halves of `part` in turn).
constexpr int block_of(int L) { return L <= 64 ? 256 : L; }

template <int L, int V>
__global__ __launch_bounds__(block_of(L)) void ln_fwd_kernel(const float* x, const float* gamma, const float* beta,
                                                             int64_t rows, int cols, float eps, float* y, float* mean,
                                                             float* rstd) {
  constexpr int B = block_of(L), RPB = B / L, LW = L < 64 ? L : 64, W = L / 64;
  __shared__ float part[2][W > 1 ? 2 * W : 1];
  const Cols<L, V> c{int(threadIdx.x % L), cols};
  f32x4 gm[V], bt[V];
#pragma unroll
  for (int q = 0; q < V; ++q) {
    gm[q] = gamma ? c.load(gamma, q) : f32x4{1.f, 1.f, 1.f, 1.f};
    bt[q] = beta ? c.load(beta, q) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Elements of this lane's wave (a wave past the row's end has none).
  const int wave0 = (int(threadIdx.x % L) & ~63) * 4;
  int in_wave = cols;
  if constexpr (W > 1) {
    in_wave = 0;
#pragma unroll
    for (int q = 0; q < V; ++q) in_wave += max(0, min(256, cols - (q * L * 4 + wave0)));
  }
  int flip = 0;
  const int64_t step = int64_t(gridDim.x) * RPB;
  for (int64_t row0 = int64_t(blockIdx.x) * RPB; row0 < rows; row0 += step) {
    // Groups past the last row read it again and store nothing: where y is x, the
    // row's own group may have stored it before they read.
    const int64_t mine = row0 + int(threadIdx.x) / L, row = min(mine, rows - 1);
    const float* xr = x + row * cols;
    f32x4 v[V];
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] = c.load(xr, q);
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < V; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) s += j >= c.skip(q) ? v[q][j] : 0.f;
    s = group_sum<LW>(s);
    float mu = s / float(max(in_wave, 1)), m2 = 0.f;
#pragma unroll
    for (int q = 0; q < V; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d = v[q][j] - mu;
        m2 += j >= c.skip(q) ? d * d : 0.f;
      }
    m2 = group_sum<LW>(m2);
    if constexpr (W > 1) {
      // Waves join by their sums and their squares about their own means:
      // sum (x - mean)^2 = sum of the waves' m2 + n_w (mean_w - mean)^2.
      float* const p = part[flip];
      flip ^= 1;
      if ((threadIdx.x & 63) == 0) {
        p[threadIdx.x >> 6] = s;
        p[W + (threadIdx.x >> 6)] = m2;
      }
      __syncthreads();
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) total += p[w];
      mu = total / float(cols);
      m2 = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        int n = 0;
#pragma unroll
        for (int q = 0; q < V; ++q) n += max(0, min(256, cols - (q * L * 4 + w * 256)));
        const float d = n > 0 ? p[w] / float(n) - mu : 0.f;
        m2 += p[W + w] + float(n) * d * d;
      }
    }
    if (mine >= rows) continue;  // at W > 1 a workgroup has one row, so none is here
    const float rs = 1.f / sqrtf(m2 / float(cols) + eps);
    float* yr = y + row * cols;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      f32x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = (v[q][j] - mu) * rs * gm[q][j] + bt[q][j];
      c.store(yr, q, o);
    }
    if (c.lane == 0) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = rs;
    }
  }
}

// dx, and the workgroup's column sums to part[blockIdx.x][2][cols] (dgamma,
// dbeta), or to dgamma / dbeta themselves when there is one workgroup.
// AFFINE: dgamma or dbeta wanted.
template <int L, int V, bool AFFINE>
__global__ __launch_bounds__(block_of(L)) void ln_bwd_kernel(const float* dy, const float* x, const float* mean,
                                                             const float* rstd, const float* gamma, int64_t rows,
                                                             int cols, float* dx, float* part, float* dgamma,
                                                             float* dbeta) {
  constexpr int B = block_of(L), RPB = B / L, LW = L < 64 ? L : 64, W = L / 64;
  __shared__ float red[2][W > 1 ? 2 * W : 1];
  __shared__ f32x4 colsum[AFFINE && RPB > 1 ? 2 * V * B : 1];
  const Cols<L, V> c{int(threadIdx.x % L), cols};
  f32x4 gm[V], ag[V], ab[V];
#pragma unroll
  for (int q = 0; q < V; ++q) {
    gm[q] = gamma ? c.load(gamma, q) : f32x4{1.f, 1.f, 1.f, 1.f};
    ag[q] = ab[q] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float inv_n = 1.f / float(cols);
  int flip = 0;
  const int64_t step = int64_t(gridDim.x) * RPB;
  for (int64_t row0 = int64_t(blockIdx.x) * RPB; row0 < rows; row0 += step) {
    const int64_t mine = row0 + int(threadIdx.x) / L, row = min(mine, rows - 1);
    const float *xr = x + row * cols, *dr = dy + row * cols;
    f32x4 v[V], d[V];
#pragma unroll
    for (int q = 0; q < V; ++q) {
      v[q] = c.load(xr, q);
      d[q] = c.load(dr, q);
    }
    const float mu = mean[row], rs = rstd[row];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int q = 0; q < V; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[q][j] = (v[q][j] - mu) * rs;
        const float g = j >= c.skip(q) ? d[q][j] * gm[q][j] : 0.f;
        s1 += g;
        s2 += g * (j >= c.skip(q) ? v[q][j] : 0.f);
      }
    if constexpr (AFFINE) {
      if (mine < rows) {
#pragma unroll
        for (int q = 0; q < V; ++q) {
          ag[q] += d[q] * v[q];
          ab[q] += d[q];
        }
      }
    }
    if (!dx) continue;
    s1 = group_sum<LW>(s1);
    s2 = group_sum<LW>(s2);
    if constexpr (W > 1) {
      float* const p = red[flip];
      flip ^= 1;
      if ((threadIdx.x & 63) == 0) {
        p[threadIdx.x >> 6] = s1;
        p[W + (threadIdx.x >> 6)] = s2;
      }
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        s1 += p[w];
        s2 += p[W + w];
      }
    }
    if (mine >= rows) continue;  // as in the forward, where dx is dy or x
    s1 *= inv_n;
    s2 *= inv_n;
    float* o = dx + row * cols;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      f32x4 t;
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = rs * (d[q][j] * gm[q][j] - s1 - v[q][j] * s2);
      c.store(o, q, t);
    }
  }
  if constexpr (AFFINE) {
    if constexpr (RPB > 1) {
      // The workgroup's rows side by side, summed in their order.
#pragma unroll
      for (int q = 0; q < V; ++q) {
        colsum[q * B + threadIdx.x] = ag[q];
        colsum[(V + q) * B + threadIdx.x] = ab[q];
      }
      __syncthreads();
      if (threadIdx.x >= L) return;
#pragma unroll
      for (int q = 0; q < V; ++q) {
        f32x4 g = colsum[q * B + threadIdx.x], b = colsum[(V + q) * B + threadIdx.x];
#pragma unroll
        for (int r = 1; r < RPB; ++r) {
          g += colsum[q * B + r * L + threadIdx.x];
          b += colsum[(V + q) * B + r * L + threadIdx.x];
        }
        ag[q] = g;
        ab[q] = b;
      }
    }
    const bool one = gridDim.x == 1;
    float* const pg = one ? dgamma : part + int64_t(blockIdx.x) * 2 * cols;
    float* const pb = one ? dbeta : pg + cols;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      if (pg) c.store(pg, q, ag[q]);
      if (pb) c.store(pb, q, ab[q]);
    }
  }
}

// Rows of more than 16384 elements or fewer than four: a workgroup walks its
// row from memory three times (forward) or twice (backward).
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = group_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < int(blockDim.x >> 6); ++w) t += part[w];
  return t;
}

__global__ __launch_bounds__(1024) void ln_fwd_walk_kernel(const float* x, const float* gamma, const float* beta,
                                                           int64_t rows, int64_t cols, float eps, float* y, float* mean,
                                                           float* rstd) {
  __shared__ float part[16];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float* xr = x + row * cols;
    float* yr = y + row * cols;
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < cols; i += blockDim.x) s += xr[i];
    const float mu = block_sum(s, part) / float(cols);
    s = 0.f;
    for (int64_t i = threadIdx.x; i < cols; i += blockDim.x) s += (xr[i] - mu) * (xr[i] - mu);
    const float rs = 1.f / sqrtf(block_sum(s, part) / float(cols) + eps);
    for (int64_t i = threadIdx.x; i < cols; i += blockDim.x)
      yr[i] = (xr[i] - mu) * rs * (gamma ? gamma[i] : 1.f) + (beta ? beta[i] : 0.f);
    if (threadIdx.x == 0) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = rs;
    }
  }
}

__global__ __launch_bounds__(1024) void ln_bwd_walk_kernel(const float* dy, const float* x, const float* mean,
                                                           const float* rstd, const float* gamma, int64_t rows,
                                                           int64_t cols, float* dx) {
  __shared__ float part[16];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float *xr = x + row * cols, *dr = dy + row * cols;
    const float mu = mean[row], rs = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t i = threadIdx.x; i < cols; i += blockDim.x) {
      const float g = dr[i] * (gamma ? gamma[i] : 1.f);
      s1 += g;
      s2 += g * ((xr[i] - mu) * rs);
    }
    s1 = block_sum(s1, part) / float(cols);
    s2 = block_sum(s2, part) / float(cols);
    for (int64_t i = threadIdx.x; i < cols; i += blockDim.x)
      dx[row * cols + i] = rs * (dr[i] * (gamma ? gamma[i] : 1.f) - s1 - (xr[i] - mu) * rs * s2);
  }
}

// The walked rows' column sums: a thread per column, rows dealt to the grid's
// second axis, part[blockIdx.y][2][cols].
__global__ __launch_bounds__(256) void ln_cols_walk_kernel(const float* dy, const float* x, const float* mean,
                                                           const float* rstd, int64_t rows, int64_t cols, float* part) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= cols) return;
  float g = 0.f, b = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float d = dy[row * cols + i];
    g += d * ((x[row * cols + i] - mean[row]) * rstd[row]);
    b += d;
  }
  float* const p = part + int64_t(blockIdx.y) * 2 * cols;
  p[i] = g;
  p[cols + i] = b;
}

// Column sums of the `parts` partial rows of [2][cols]: 32 columns and 32
// groups of partials to a workgroup, the groups joined in order.
__global__ __launch_bounds__(1024) void ln_cols_kernel(const float* part, int parts, int64_t cols, float* dgamma,
                                                       float* dbeta) {
  __shared__ float sum[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t at = int64_t(blockIdx.x) * 32 + tx;
  float s = 0.f;
  if (at < 2 * cols) {
#pragma unroll 8
    for (int p = ty; p < parts; p += 32) s += part[int64_t(p) * 2 * cols + at];
  }
  sum[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && at < 2 * cols) {
#pragma unroll
    for (int g = 1; g < 32; ++g) s += sum[g][tx];
    float* const out = at < cols ? dgamma : dbeta;
    if (out) out[at < cols ? at : at - cols] = s;
  }
}

__global__ void ln_zero_kernel(float* a, float* b, int64_t n) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    if (a) a[i] = 0.f;
    if (b) b[i] = 0.f;
  }
}

// Lanes to a row and vectors to a lane: the smallest that hold it, the walk for rows
// that none holds.  Microseconds forward / backward of 2^25 elements, so and with
// the next one:
//   columns    64           128          256          512          1024
//              52/89        45/98        48/79        47/78        45/80
//              52/171       50/102       51/104       46/91        57/112
//   columns    2048         4096         8192         16384 (next: walked)
//              47/77        45/84        48/85        57/97
//              49/95        56/95        67/89        82/159
// (2^20 elements take 8 / 11 to 14 us, the calls' own, with any of them.)
enum { kWalk = -1 };
struct Shape {
  int lanes, vecs;
};
constexpr Shape kShapes[] = {{16, 1}, {16, 2}, {32, 2}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {512, 4}, {512, 8}};

int pick(int64_t cols) {
  if (cols < 4) return kWalk;
  for (int i = 0; i < int(sizeof(kShapes) / sizeof(kShapes[0])); ++i)
    if (cols <= kShapes[i].lanes * kShapes[i].vecs * 4) return i;
  return kWalk;
}

// Calls f(lanes, vecs) with shape i's constants.
template <class F>
void with_shape(int i, F&& f) {
  using std::integral_constant;
#define MX_LN_SHAPE(I, L, V) \
  case I: return f(integral_constant<int, L>{}, integral_constant<int, V>{});
  switch (i) {
    MX_LN_SHAPE(0, 16, 1)
    MX_LN_SHAPE(1, 16, 2)
    MX_LN_SHAPE(2, 32, 2)
    MX_LN_SHAPE(3, 64, 2)
    MX_LN_SHAPE(4, 64, 4)
    MX_LN_SHAPE(5, 256, 2)
    MX_LN_SHAPE(6, 256, 4)
    MX_LN_SHAPE(7, 512, 4)
    default: return f(integral_constant<int, 512>{}, integral_constant<int, 8>{});
  }
#undef MX_LN_SHAPE
}

// Workgroups of the backward: each leaves 8 bytes a column for the second
// launch to sum, so no more than fill the chip.
int bwd_blocks(int shape, int64_t rows) {
  const int lanes = kShapes[shape].lanes, block = block_of(lanes), rpb = block / lanes;
  return int(std::min<int64_t>((rows + rpb - 1) / rpb, int64_t(cu_count()) * std::max(1, 512 / block)));
}
int walk_parts(int64_t rows) { return int(std::min<int64_t>(rows, 64)); }

int64_t bwd_workspace(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  const int shape = pick(cols);
  const int parts = shape == kWalk ? walk_parts(rows) : bwd_blocks(shape, rows);
  return shape != kWalk && parts == 1 ? 0 : int64_t(parts) * 2 * cols * 4;
}

int check(const char* who, int64_t rows, int64_t cols) {
  MX_REQUIRE(rows >= 0 && cols >= 0, MX_ERR_INVALID, who, ": negative size");
  MX_REQUIRE(rows == 0 || cols > 0, MX_ERR_INVALID, who, ": empty rows");
  MX_REQUIRE(cols <= INT32_MAX && rows <= (int64_t(1) << 60) / std::max<int64_t>(cols, 1), MX_ERR_INVALID, who,
             ": size out of range");
  return MX_OK;
}

}  // namespace
}  // namespace mx

using namespace mx;

extern "C" int mx_layer_norm_forward(const float* x, const float* gamma, const float* beta, int64_t rows, int64_t cols,
                                     float eps, float* y, float* mean, float* rstd, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  MX_TRY(check("mx_layer_norm_forward", rows, cols));
  if (rows == 0) return MX_OK;
  MX_REQUIRE(x && y, MX_ERR_INVALID, "mx_layer_norm_forward: null buffer");
  hipStream_t s = resolve_stream(stream);
  const int shape = pick(cols);
  if (shape == kWalk) {
    const int threads = cols < 1024 ? 64 : 1024;
    hipLaunchKernelGGL(ln_fwd_walk_kernel, dim3(unsigned(std::min<int64_t>(rows, 65535))), dim3(threads), 0, s, x, gamma,
                       beta, rows, cols, eps, y, mean, rstd);
  } else {
    with_shape(shape, [&](auto l, auto v) {
      constexpr int L = decltype(l)::value, V = decltype(v)::value, B = block_of(L), RPB = B / L;
      const int64_t blocks = std::min<int64_t>((rows + RPB - 1) / RPB, int64_t(cu_count()) * (2048 / B));
      hipLaunchKernelGGL((ln_fwd_kernel<L, V>), dim3(unsigned(blocks)), dim3(B), 0, s, x, gamma, beta, rows, int(cols),
                         eps, y, mean, rstd);
    });
  }
  MX_LAUNCHED();
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_layer_norm_backward_workspace(int64_t rows, int64_t cols, int64_t* bytes) {
  MX_ABI_BEGIN
  MX_TRY(check("mx_layer_norm_backward", rows, cols));
  MX_REQUIRE(bytes, MX_ERR_INVALID, "mx_layer_norm_backward_workspace: null result");
  *bytes = bwd_workspace(rows, cols);
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_layer_norm_backward(const float* dy, const float* x, const float* mean, const float* rstd,
                                      const float* gamma, int64_t rows, int64_t cols, float* dx, float* dgamma,
                                      float* dbeta, void* workspace, int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  MX_TRY(check("mx_layer_norm_backward", rows, cols));
  const bool affine = dgamma || dbeta;
  if (!dx && !affine) return MX_OK;
  hipStream_t s = resolve_stream(stream);
  if (rows == 0) {
    if (!affine || cols == 0) return MX_OK;
    hipLaunchKernelGGL(ln_zero_kernel, dim3(unsigned(std::min<int64_t>((cols + 255) / 256, 1024))), dim3(256), 0, s,
                       dgamma, dbeta, cols);
    MX_LAUNCHED();
    return MX_OK;
  }
  MX_REQUIRE(dy && x && mean && rstd, MX_ERR_INVALID, "mx_layer_norm_backward: null buffer");
  const int shape = pick(cols);
  Workspace ws;
  const int64_t need = affine ? bwd_workspace(rows, cols) : 0;
  MX_TRY(ws.take("mx_layer_norm_backward", workspace, workspace_bytes, need, s));
  float* const part = ws.as<float>();
  int parts = 1;
  if (shape == kWalk) {
    if (affine) {  // before dx, which may be stored over dy or x
      parts = walk_parts(rows);
      hipLaunchKernelGGL(ln_cols_walk_kernel, dim3(unsigned((cols + 255) / 256), unsigned(parts)), dim3(256), 0, s, dy, x,
                         mean, rstd, rows, cols, part);
      MX_LAUNCHED();
    }
    if (dx) {
      const int threads = cols < 1024 ? 64 : 1024;
      hipLaunchKernelGGL(ln_bwd_walk_kernel, dim3(unsigned(std::min<int64_t>(rows, 65535))), dim3(threads), 0, s, dy, x,
                         mean, rstd, gamma, rows, cols, dx);
      MX_LAUNCHED();
    }
    if (!affine) return MX_OK;
  } else {
    parts = bwd_blocks(shape, rows);
    with_shape(shape, [&](auto l, auto v) {
      constexpr int L = decltype(l)::value, V = decltype(v)::value, B = block_of(L), RPB = B / L;
      if (affine) {
        hipLaunchKernelGGL((ln_bwd_kernel<L, V, true>), dim3(unsigned(parts)), dim3(B), 0, s, dy, x, mean, rstd, gamma,
                           rows, int(cols), dx, part, dgamma, dbeta);
      } else {
        const int64_t blocks = std::min<int64_t>((rows + RPB - 1) / RPB, int64_t(cu_count()) * (2048 / B));
        hipLaunchKernelGGL((ln_bwd_kernel<L, V, false>), dim3(unsigned(blocks)), dim3(B), 0, s, dy, x, mean, rstd,
                           gamma, rows, int(cols), dx, part, dgamma, dbeta);
      }
    });
    MX_LAUNCHED();
    if (!affine || parts == 1) return MX_OK;
  }
  hipLaunchKernelGGL(ln_cols_kernel, dim3(unsigned((2 * cols + 31) / 32)), dim3(1024), 0, s, part, parts, cols, dgamma,
                     dbeta);
  MX_LAUNCHED();
  return MX_OK;
  MX_ABI_END
}
