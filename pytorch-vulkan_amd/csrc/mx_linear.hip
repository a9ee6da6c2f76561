// Linear layer with its bias, activation and residual in the product's
// epilogue, and its backward (FP32, contiguous).
//
//   z = x w^T + bias,  y = act(z) + residual
//   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = sum_m dz
//
// The forward is one product (mx_gemm.hip) whose stores apply the rest.  The
// backward makes dz in one pass that sums its columns on the way (the products
// would otherwise evaluate the slope once for every tile that reads the
// element), then takes the two products of it.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mx_activation.hpp"
#include "mx_internal.hpp"

namespace mx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// dz = dy * act'(z) (not written where dz is null; z null: the slope is 1), and
// the column sums of dz over the workgroup's rows to part[blockIdx.y][n] where
// part is not null.  A thread holds W columns; 64 threads lie along a row and
// the workgroup's four waves take a row each.  W == 4 for n >= 4: the last
// thread of a row takes its last four elements (it and its neighbour write the
// same values).
template <int W>
__global__ __launch_bounds__(256) void slope_kernel(const float* dy, const float* z, int act, int64_t m, int n,
                                                    int64_t rows_per, float* dz, float* part) {
  typedef float vec __attribute__((ext_vector_type(W)));
  typedef float vecu __attribute__((ext_vector_type(W), aligned(4)));
  __shared__ vec sums[256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = (int64_t(blockIdx.x) * 64 + lane) * W;
  const bool in = col < n;
  const int64_t at = min(col, int64_t(n - W));
  const int64_t r0 = blockIdx.y * rows_per, r1 = min(m, r0 + rows_per);
  vec s = 0.f;
  if (in) {
#pragma unroll 4
    for (int64_t r = r0 + wave; r < r1; r += 4) {
      vec d = *reinterpret_cast<const vecu*>(dy + r * n + at);
      if (z) {
        const vec t = *reinterpret_cast<const vecu*>(z + r * n + at);
#pragma unroll
        for (int e = 0; e < W; ++e) d[e] *= activate_slope(act, t[e]);
        if (dz) *reinterpret_cast<vecu*>(dz + r * n + at) = d;
      }
      s += d;
    }
  }
  if (!part) return;
  sums[threadIdx.x] = s;
  __syncthreads();
  if (wave == 0 && in) {
    s += sums[64 + lane];
    s += sums[128 + lane];
    s += sums[192 + lane];
    *reinterpret_cast<vecu*>(part + int64_t(blockIdx.y) * n + at) = s;
  }
}

// out[c] = sum of part[p][c] in the order of p: 32 columns and 32 groups of
// partials to a workgroup.
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

// Row ranges of the elementwise pass: enough workgroups to fill the chip
// without splitting a range below 16 rows.
struct SlopePlan {
  int64_t rows_per;
  int parts, col_blocks;
};
SlopePlan plan_slope(int64_t m, int64_t n) {
  SlopePlan p{};
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

struct BackwardPlan {
  int64_t dz, sums, gemm;  // bytes
};
int plan_backward(int64_t m, int64_t k, int64_t n, int act, BackwardPlan* p) {
  *p = BackwardPlan{};
  if (m == 0 || n == 0) return MX_OK;
  if (act != MX_ACT_NONE) p->dz = up256(m * n * 4);
  const SlopePlan sp = plan_slope(m, n);
  if (sp.parts > 1) p->sums = up256(int64_t(sp.parts) * n * 4);
  if (k == 0) return MX_OK;
  int64_t a = 0, b = 0;
  MX_TRY(partials(dx_desc(m, k, n), &a));
  MX_TRY(partials(dw_desc(m, k, n), &b));
  p->gemm = std::max(a, b);
  return MX_OK;
}

}  // namespace
}  // namespace mx

using namespace mx;

extern "C" int mx_linear_workspace(int64_t m, int64_t k, int64_t n, int activation, int backward, int64_t* bytes) {
  MX_ABI_BEGIN
  MX_TRY(check("mx_linear_workspace", m, k, n, activation));
  MX_REQUIRE(bytes, MX_ERR_INVALID, "mx_linear_workspace: null result");
  *bytes = 0;
  if (m == 0 || n == 0) return MX_OK;
  if (backward) {
    BackwardPlan p;
    MX_TRY(plan_backward(m, k, n, activation, &p));
    *bytes = p.dz + p.sums + p.gemm;
  } else if (k > 0) {
    MX_TRY(partials(forward_desc(m, k, n, true), bytes));
  }
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_linear_forward(const float* x, const float* w, const float* bias, const float* residual, int64_t m,
                                 int64_t k, int64_t n, int activation, float* y, float* z, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  MX_TRY(check("mx_linear_forward", m, k, n, activation));
  if (m == 0 || n == 0) return MX_OK;
  MX_REQUIRE(y && (k == 0 || (x && w)), MX_ERR_INVALID, "mx_linear_forward: null buffer");
  const mx_gemm_desc d = forward_desc(m, k, n, bias != nullptr);
  int64_t need = 0;
  if (workspace && k > 0) {
    MX_TRY(partials(d, &need));
    MX_REQUIRE(workspace_bytes >= need, MX_ERR_WORKSPACE, "mx_linear_forward: workspace of ", workspace_bytes, " bytes, ",
               need, " needed");
  }
  const GemmEpilogue epi{activation, residual, z};
  return gemm_within(&d, x, w, bias, y, kPartials, resolve_stream(stream), &epi, workspace);
  MX_ABI_END
}

extern "C" int mx_linear_backward(const float* dy, const float* x, const float* w, const float* z, int64_t m, int64_t k,
                                  int64_t n, int activation, float* dx, float* dw, float* db, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  MX_TRY(check("mx_linear_backward", m, k, n, activation));
  hipStream_t s = resolve_stream(stream);
  const auto zero = [&](float* p, int64_t count) -> int {
    if (!p || count == 0) return MX_OK;
    hipLaunchKernelGGL(zero_kernel, dim3(unsigned(std::min<int64_t>((count + 255) / 256, 65535))), dim3(256), 0, s, p, count);
    MX_HIP(hipGetLastError());
    return MX_OK;
  };
  if (m == 0 || n == 0) {  // empty sums
    MX_TRY(zero(dx, m * k));
    MX_TRY(zero(dw, n * k));
    return zero(db, n);
  }
  const bool slope = activation != MX_ACT_NONE;
  MX_REQUIRE(dy && (!slope || z) && (k == 0 || ((!dx || w) && (!dw || x))), MX_ERR_INVALID,
             "mx_linear_backward: null buffer");
  if (k == 0) dx = dw = nullptr;
  if (!dx && !dw && !db) return MX_OK;
  BackwardPlan plan;
  MX_TRY(plan_backward(m, k, n, activation, &plan));
  const bool products = dx || dw;
  if (!products) plan.dz = plan.gemm = 0;
  if (!db) plan.sums = 0;
  // Captured calls without a workspace take the products in one pass each.
  const bool caller = workspace != nullptr;
  if (!caller) plan.gemm = 0;
  Workspace ws;
  MX_TRY(ws.take("mx_linear_backward", workspace, workspace_bytes, plan.dz + plan.sums + plan.gemm, s));
  char* const base = ws.as<char>();
  float* const dz = plan.dz ? reinterpret_cast<float*>(base) : nullptr;
  const SlopePlan sp = plan_slope(m, n);
  if (db || dz) {
    float* const part = !db ? nullptr : sp.parts > 1 ? reinterpret_cast<float*>(base + plan.dz) : db;
    const dim3 grid{unsigned(sp.col_blocks), unsigned(sp.parts)};
    const float* const zz = slope ? z : nullptr;
    if (n >= 4)
      hipLaunchKernelGGL(slope_kernel<4>, grid, dim3(256), 0, s, dy, zz, activation, m, int(n), sp.rows_per, dz, part);
    else
      hipLaunchKernelGGL(slope_kernel<1>, grid, dim3(256), 0, s, dy, zz, activation, m, int(n), sp.rows_per, dz, part);
    MX_HIP(hipGetLastError());
    if (db && sp.parts > 1) {
      hipLaunchKernelGGL(column_sum_kernel, dim3(unsigned((n + 31) / 32)), dim3(1024), 0, s, part, sp.parts, int(n), db);
      MX_HIP(hipGetLastError());
    }
  }
  const float* const g = dz ? dz : dy;
  void* const partial = caller && plan.gemm ? base + plan.dz + plan.sums : nullptr;
  if (dx) {
    const mx_gemm_desc d = dx_desc(m, k, n);
    MX_TRY(gemm_within(&d, g, w, nullptr, dx, kPartials, s, nullptr, partial));
  }
  if (dw) {
    const mx_gemm_desc d = dw_desc(m, k, n);
    MX_TRY(gemm_within(&d, g, x, nullptr, dw, kPartials, s, nullptr, partial));
  }
  return MX_OK;
  MX_ABI_END
}
