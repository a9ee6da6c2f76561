// Norm of queries and keys for each head and rotary positions, in one pass (FP32).
//
//   forward   r = (mean x^2 + eps)^-1/2,  xh = x r w   (without a norm xh = x)
//             y_a = xh_a c - xh_b s,  y_b = xh_b c + xh_a s   on the pairs (a, b) of the
//             head's first rotary_dim elements, c and s = magnitude (cos, sin)(position f_i)
//   backward  g = the same rotation by the opposite angle of dy,  gw = g w,
//             dx = r (gw - x r mean(gw x r)),  dw = sum over tokens and heads g x r
//
// Bound by memory: 8 bytes an element forward, 12 backward with a norm.  A row (one
// head of one token) stays in the registers of a group of 8 to 64 lanes, four
// elements each; what an element is paired with is read again from the row, which the
// first-level cache holds.  A workgroup takes all heads of its tokens, so an angle is
// evaluated once a token: in 64 bits down to a fraction of a turn (a position of 10^6
// at frequency 1 has 20 bits before the point, and FP32 would leave 4 behind), then
// sine and cosine of that fraction in FP32, corrected by what its rounding left
// (over 4000 positions up to 2^20, 64 pairs: off by 1.3 2^-24 at most and 0.32 in the mean square, without that 1.9 and 0.55).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "mx_internal.hpp"

namespace mx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kMaxDim = 256, kThreads = 256, kAngles = 2048;  // kAngles: pairs of a workgroup's tokens in LDS
// Rows of a lane group at a time.  (The backward has three loads to a row: two rows and four measure
// the same, 95 us for both directions of 8192 tokens x 20 heads x 128, three 101.)
constexpr int unroll(bool back) { return back ? 2 : 4; }

struct Rotary {
  int tokens, q_heads, k_heads, dim, rot;
  int64_t q_token, q_head, k_token, k_head;
  const int64_t* positions;
  float magnitude, eps, per;  // per: 1 / dim
  int interleaved, norm, group;  // group: tokens that a workgroup turns together
  double turns[kMaxDim / 2];     // frequencies / 2 pi
};

struct Operands {  // q's and k's
  const float *x[2], *dy[2], *w[2];
  float *out[2], *part;
  bool wanted[2];  // a side that nothing is asked of is not read
};

// v of another lane of the same 16, by a fixed pattern.
template <int PATTERN>
__device__ __forceinline__ float row_move(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), PATTERN, 0xF, 0xF, true));
}
// Sum over groups of L lanes: neighbours, pairs, then the mirror images of halves and wholes of 16.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  v += row_move<0xB1>(v);
  v += row_move<0x4E>(v);
  v += row_move<0x141>(v);
  if constexpr (L > 8) v += row_move<0x140>(v);
#pragma unroll
  for (int m = 16; m < L; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// Elements e .. e + 3 of a row of n, zero past its end.
__device__ __forceinline__ f32x4 load4(const float* row, int e, int n) {
  if (e + 4 <= n) return *reinterpret_cast<const f32x4u*>(row + e);
  f32x4 v{};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (e + i < n) v[i] = row[e + i];
  return v;
}
__device__ __forceinline__ void store4(float* row, int e, int n, f32x4 v) {
  if (e + 4 <= n) {
    *reinterpret_cast<f32x4u*>(row + e) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (e + i < n) row[e + i] = v[i];
}

// Which element e is paired with, and whether it is a pair's first.
__device__ __forceinline__ int partner(const Rotary& p, int e, bool& first) {
  if (e >= p.rot) return first = true, e;
  const int half = p.rot >> 1;
  first = p.interleaved ? !(e & 1) : e < half;
  return p.interleaved ? e ^ 1 : first ? e + half : e - half;
}

// cos and sin (times the magnitude) of a workgroup's tokens, [token][pair].
__device__ __forceinline__ void angles(const Rotary& p, int first, int count, float* cs, float* sn) {
  const int half = p.rot >> 1;
  for (int i = threadIdx.x; i < count * half; i += kThreads) {
    const int t = i / half, pair = i - t * half;
    const double turn = double(p.positions[first + t]) * p.turns[pair];
    const double part = turn - rint(turn);
    const float frac = float(part), rest = float((part - frac) * 6.283185307179586476925286766559);
    float s, c;
    sincospif(2.f * frac, &s, &c);
    // (the rest is below 2^-26 of a turn: its square is nothing)
    cs[i] = fmaf(-s, rest, c) * p.magnitude;
    sn[i] = fmaf(c, rest, s) * p.magnitude;
  }
  __syncthreads();
}

// A row of the workgroup's tokens: q's heads of each, then k's.
struct RowAt {
  int k, place, token, head;  // which of q and k; the token's place among the workgroup's
  bool live;
};

__device__ __forceinline__ int64_t flat(const Rotary& p, const RowAt& r) {
  return (int64_t(r.token) * (r.k ? p.k_heads : p.q_heads) + r.head) * p.dim;
}
template <int L>
__device__ __forceinline__ float rstd(const Rotary& p, f32x4 x) {
  return rsqrtf(lanes_sum<L>(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]) * p.per + p.eps);
}

// 8192 tokens of 20 heads of 128: forward 36 us (4.7 TB/s), backward 51 + 5 (4.5 TB/s).
template <int L, bool BACK>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const Rotary p, const Operands o) {
  constexpr int U = unroll(BACK);
  __shared__ __attribute__((aligned(16))) float cs[kAngles], sn[kAngles];
  __shared__ float sums[BACK ? 2 * kMaxDim : 1];
  const int lane = threadIdx.x % L, e = lane * 4, half = p.rot >> 1;
  f32x4 w[2] = {f32x4{1, 1, 1, 1}, f32x4{1, 1, 1, 1}};
  int with[4], pair[4];  // each element's partner and pair
  bool head[4];
  // (an element that is not turned has 0 for a partner, in its row and its weight: what lies beside it may be anything)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    with[i] = min(partner(p, e + i, head[i]), p.dim - 1);
    pair[i] = e + i >= p.rot ? -1 : p.interleaved ? (e + i) >> 1 : (e + i) % half;
  }
  // A lane's four partners lie together, the same four for neighbouring pairs.
  const bool own = p.interleaved || p.rot == 0, run = !own && half % 4 == 0 && e < p.rot;
  float wp[2][4];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (p.norm && o.w[k]) w[k] = load4(o.w[k], e, p.dim);
#pragma unroll
    for (int i = 0; i < 4; ++i) wp[k][i] = pair[i] < 0 ? 0.f : p.norm && o.w[k] ? o.w[k][with[i]] : 1.f;
  }
  f32x4 dw[2] = {};
  for (int first = blockIdx.x * p.group; first < p.tokens; first += gridDim.x * p.group) {
    const int count = min(p.group, p.tokens - first);
    // A group of L lanes takes every kThreads / L-th row, U at a time (their loads are in
    // flight together), whichever side is wanted: the weights' sums keep their order.
    const int heads = p.q_heads + p.k_heads;
    int place = threadIdx.x / L / heads, h = threadIdx.x / L - place * heads;  // of the next row
    for (int turn = 0; turn < count * heads; turn += U * (kThreads / L)) {
      RowAt at[U];
      f32x4 v[U], u[U], x[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        at[j].k = h >= p.q_heads;
        at[j].place = place;
        at[j].head = at[j].k ? h - p.q_heads : h;
        at[j].token = first + place;
        at[j].live = place < count && (at[j].k ? o.wanted[1] : o.wanted[0]);
        for (h += kThreads / L; h >= heads; h -= heads) ++place;
        v[j] = u[j] = x[j] = f32x4{};
        if (!at[j].live) continue;
        const float* const in = (at[j].k ? o.x[1] : o.x[0]) + at[j].token * (at[j].k ? p.k_token : p.q_token) + at[j].head * (at[j].k ? p.k_head : p.q_head);
        // the row that the rotation is applied to, its elements' partners, and the norm's input
        const float* const turned = BACK ? (at[j].k ? o.dy[1] : o.dy[0]) + flat(p, at[j]) : in;
        v[j] = load4(turned, e, p.dim);
        if (run) {
          u[j] = *reinterpret_cast<const f32x4u*>(turned + with[0]);
        } else if (!own && e < p.rot) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float other = turned[with[i]];
            u[j][i] = pair[i] < 0 ? 0.f : other;
          }
        }
        if (BACK && p.norm) x[j] = load4(in, e, p.dim);
      }
      if (half && turn == 0) angles(p, first, count, cs, sn);  // while the first rows are on their way
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (!at[j].live) continue;
        const int k = at[j].k;
        if (own && p.rot) {
#pragma unroll
          for (int i = 0; i < 4; ++i) u[j][i] = pair[i] < 0 ? 0.f : v[j][i ^ 1];
        }
        f32x4 c{1, 1, 1, 1}, s{};
        if (run) {  // four neighbouring pairs
          c = *reinterpret_cast<const f32x4*>(&cs[at[j].place * half + pair[0]]);
          s = *reinterpret_cast<const f32x4*>(&sn[at[j].place * half + pair[0]]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (pair[i] >= 0) c[i] = cs[at[j].place * half + pair[i]], s[i] = sn[at[j].place * half + pair[i]];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (head[i] != BACK) s[i] = -s[i];
        f32x4 y;
        if constexpr (!BACK) {
          float r = 1;
          if (p.norm) r = rstd<L>(p, v[j]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float xh = p.norm ? v[j][i] * r * (k ? w[1][i] : w[0][i]) : v[j][i];
            const float xp = p.norm ? u[j][i] * r * (k ? wp[1][i] : wp[0][i]) : u[j][i];
            y[i] = fmaf(xp, s[i], xh * c[i]);  // (unturned: cosine 1, sine 0)
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = fmaf(u[j][i], s[i], v[j][i] * c[i]);
          if (p.norm) {
            const float r = rstd<L>(p, x[j]);
            const f32x4 g = y, xr = x[j] * r, gw = g * (k ? w[1] : w[0]);
            const float m = lanes_sum<L>(gw[0] * xr[0] + gw[1] * xr[1] + gw[2] * xr[2] + gw[3] * xr[3]) * p.per;
            y = (gw - xr * m) * r;
            if (k) dw[1] += g * xr;
            else dw[0] += g * xr;
          }
        }
        if (float* const out = k ? o.out[1] : o.out[0]) store4(out + flat(p, at[j]), e, p.dim, y);
      }
    }
    if (half) __syncthreads();
  }
  if constexpr (BACK) {
    if (!o.part) return;
    // Column sums of the workgroup, its lane groups one after the other.
    for (int g = 0; g < kThreads / L; ++g) {
      if (int(threadIdx.x) / L == g) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float* const at = sums + k * kMaxDim + e + i;
            *at = g ? *at + dw[k][i] : dw[k][i];
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * p.dim; i += kThreads)
      o.part[int64_t(blockIdx.x) * 2 * p.dim + i] = sums[i / p.dim * kMaxDim + i % p.dim];
  }
}

// dw[i] = the sum of the workgroups' parts: 8 columns to a workgroup, 128 rows of threads.
__global__ __launch_bounds__(1024) void rotary_weights_kernel(const float* part, int parts, int dim, float* dqw, float* dkw) {
  __shared__ float sums[128][9];
  const int i = threadIdx.x & 7, col = blockIdx.x * 8 + i, row = threadIdx.x >> 3;
  float s = 0;
  if (col < 2 * dim)
    for (int k = row; k < parts; k += 128) s += part[int64_t(k) * 2 * dim + col];
  sums[row][i] = s;
  __syncthreads();
  for (int n = 64; n; n >>= 1) {
    if (row < n) sums[row][i] += sums[row + n][i];
    __syncthreads();
  }
  if (row || col >= 2 * dim) return;
  float* const out = col < dim ? dqw : dkw;
  if (out) out[col % dim] = sums[0][i];
}

__global__ void rotary_zero_kernel(float* a, float* b, int dim) {
  const int i = threadIdx.x;
  if (i < dim && a) a[i] = 0;
  if (i < dim && b) b[i] = 0;
}

int check(const char* who, const mx_rotary_desc* d) {
  MX_REQUIRE(d, MX_ERR_INVALID, who, ": null descriptor");
  MX_REQUIRE(d->tokens >= 0 && d->q_heads >= 0 && d->k_heads >= 0, MX_ERR_INVALID, who, ": negative size");
  MX_REQUIRE(d->head_dim >= 1 && d->head_dim <= kMaxDim, MX_ERR_INVALID, who, ": head_dim must be 1 to ", kMaxDim, ", got ",
             d->head_dim);
  MX_REQUIRE(d->rotary_dim >= 0 && d->rotary_dim <= d->head_dim && d->rotary_dim % 2 == 0, MX_ERR_INVALID, who,
             ": rotary_dim must be even and at most head_dim, got ", d->rotary_dim);
  MX_REQUIRE(d->tokens <= (1 << 30) && d->q_heads <= (1 << 20) && d->k_heads <= (1 << 20), MX_ERR_INVALID, who,
             ": size out of range");
  MX_REQUIRE(d->rotary_dim == 0 || d->frequencies, MX_ERR_INVALID, who, ": null frequencies");
  for (int64_t i = 0; i < d->rotary_dim / 2; ++i)
    MX_REQUIRE(std::isfinite(d->frequencies[i]), MX_ERR_INVALID, who, ": frequencies must be finite");
  MX_REQUIRE(std::isfinite(d->magnitude), MX_ERR_INVALID, who, ": the magnitude must be finite");
  MX_REQUIRE(!d->norm || (std::isfinite(d->eps) && d->eps >= 0), MX_ERR_INVALID, who, ": eps must not be negative");
  return MX_OK;
}

Rotary params(const mx_rotary_desc* d) {
  Rotary p{};
  p.tokens = int(d->tokens), p.q_heads = int(d->q_heads), p.k_heads = int(d->k_heads);
  p.dim = int(d->head_dim), p.rot = int(d->rotary_dim);
  p.q_token = d->q_token, p.q_head = d->q_head, p.k_token = d->k_token, p.k_head = d->k_head;
  p.positions = d->positions;
  p.magnitude = float(d->magnitude), p.eps = float(d->eps), p.per = 1.f / float(d->head_dim);
  p.interleaved = d->interleaved, p.norm = d->norm;
  for (int i = 0; i < p.rot / 2; ++i) p.turns[i] = d->frequencies[i] / 6.283185307179586476925286766559;
  return p;
}

int lanes_of(int dim) {
  for (int l = 8; l < 64; l *= 2)
    if (dim <= 4 * l) return l;
  return 64;
}

// Tokens that a workgroup turns together: as far as their angles fit LDS and every CU
// has four workgroups, the number whose rows fill its lane groups' pairs best.
int group_of(int dim, int rot, int64_t heads, int64_t tokens, bool back) {
  const int64_t slots = unroll(back) * kThreads / lanes_of(dim);
  int64_t most = std::max<int64_t>(1, std::max<int64_t>(slots / heads, std::min<int64_t>(8, tokens / (int64_t(cu_count()) * 4))));
  if (rot) most = std::min<int64_t>(most, kAngles / (rot / 2));
  int64_t best = 1;
  for (int64_t g = 2; g <= most; ++g) {  // rows over the places that their turns have
    const int64_t a = g * heads * ((best * heads + slots - 1) / slots), b = best * heads * ((g * heads + slots - 1) / slots);
    if (a > b) best = g;
  }
  return int(best);
}

int blocks_of(const Rotary& p, bool parts) {
  const int64_t all = (p.tokens + p.group - 1) / p.group;
  return int(std::min<int64_t>(all, int64_t(cu_count()) * (parts ? 4 : 64)));
}

template <bool BACK>
void launch(const Rotary& p, const Operands& o, int blocks, hipStream_t s) {
  switch (lanes_of(p.dim)) {
    case 8: hipLaunchKernelGGL((rotary_kernel<8, BACK>), dim3(blocks), dim3(kThreads), 0, s, p, o); break;
    case 16: hipLaunchKernelGGL((rotary_kernel<16, BACK>), dim3(blocks), dim3(kThreads), 0, s, p, o); break;
    case 32: hipLaunchKernelGGL((rotary_kernel<32, BACK>), dim3(blocks), dim3(kThreads), 0, s, p, o); break;
    default: hipLaunchKernelGGL((rotary_kernel<64, BACK>), dim3(blocks), dim3(kThreads), 0, s, p, o); break;
  }
}

}  // namespace
}  // namespace mx

using namespace mx;

extern "C" int mx_qk_norm_rotary_forward(const mx_rotary_desc* d, const float* q, const float* k, const float* q_weight,
                                         const float* k_weight, float* q_out, float* k_out, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  const char* const who = "mx_qk_norm_rotary_forward";
  MX_TRY(check(who, d));
  const int64_t heads = d->q_heads + d->k_heads;
  if (d->tokens == 0 || heads == 0) return MX_OK;
  MX_REQUIRE((d->q_heads == 0 || (q && q_out)) && (d->k_heads == 0 || (k && k_out)) && (d->rotary_dim == 0 || d->positions),
             MX_ERR_INVALID, who, ": null buffer");
  Rotary p = params(d);
  p.group = group_of(p.dim, p.rot, heads, p.tokens, false);
  const Operands o{{q, k}, {nullptr, nullptr}, {q_weight, k_weight}, {q_out, k_out}, nullptr, {true, true}};
  launch<false>(p, o, blocks_of(p, false), resolve_stream(stream));
  MX_LAUNCHED();
  return MX_OK;
  MX_ABI_END
}

namespace {
// Bytes of the workgroups' parts of the weights' gradients.
int64_t rotary_workspace(const mx_rotary_desc* d) {
  const int64_t heads = d->q_heads + d->k_heads;
  if (!d->norm || d->tokens == 0 || heads == 0) return 0;
  const int64_t group = group_of(int(d->head_dim), int(d->rotary_dim), heads, d->tokens, true);
  return std::min<int64_t>((d->tokens + group - 1) / group, int64_t(cu_count()) * 4) * 2 * d->head_dim * 4;
}
}  // namespace

extern "C" int mx_qk_norm_rotary_workspace(const mx_rotary_desc* d, int64_t* bytes) {
  MX_ABI_BEGIN
  MX_TRY(check("mx_qk_norm_rotary_workspace", d));
  MX_REQUIRE(bytes, MX_ERR_INVALID, "mx_qk_norm_rotary_workspace: null result");
  *bytes = rotary_workspace(d);
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_qk_norm_rotary_backward(const mx_rotary_desc* d, const float* dq_out, const float* dk_out, const float* q,
                                          const float* k, const float* q_weight, const float* k_weight, float* dq,
                                          float* dk, float* dq_weight, float* dk_weight, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  const char* const who = "mx_qk_norm_rotary_backward";
  MX_TRY(check(who, d));
  MX_REQUIRE(d->norm || (!dq_weight && !dk_weight), MX_ERR_INVALID, who, ": gradients of weights without a norm");
  const int64_t heads = d->q_heads + d->k_heads;
  hipStream_t s = resolve_stream(stream);
  const bool weights = dq_weight || dk_weight;
  if (d->tokens == 0 || heads == 0) {
    if (!weights) return MX_OK;
    hipLaunchKernelGGL(rotary_zero_kernel, dim3(1), dim3(kMaxDim), 0, s, dq_weight, dk_weight, int(d->head_dim));
    MX_LAUNCHED();
    return MX_OK;
  }
  if (!dq && !dk && !weights) return MX_OK;
  const bool qs = dq || dq_weight, ks = dk || dk_weight;
  MX_REQUIRE((!qs || d->q_heads == 0 || (dq_out && (!d->norm || q))) && (!ks || d->k_heads == 0 || (dk_out && (!d->norm || k))) &&
                 (d->rotary_dim == 0 || d->positions),
             MX_ERR_INVALID, who, ": null buffer");
  Workspace ws;
  if (weights) MX_TRY(ws.take(who, workspace, workspace_bytes, rotary_workspace(d), s));
  Rotary p = params(d);
  p.group = group_of(p.dim, p.rot, heads, p.tokens, true);
  const Operands o{{q, k}, {dq_out, dk_out}, {q_weight, k_weight}, {dq, dk}, ws.as<float>(), {qs, ks}};
  const int blocks = blocks_of(p, weights);
  launch<true>(p, o, blocks, s);
  MX_LAUNCHED();
  if (!weights) return MX_OK;
  hipLaunchKernelGGL(rotary_weights_kernel, dim3((2 * p.dim + 7) / 8), dim3(1024), 0, s, ws.as<float>(), blocks, p.dim,
                     dq_weight, dk_weight);
  MX_LAUNCHED();
  return MX_OK;
  MX_ABI_END
}
