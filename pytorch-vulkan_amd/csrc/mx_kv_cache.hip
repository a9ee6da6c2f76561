// A paged cache of keys and values: writing new tokens into it and reading them back.
//
//   k [pages, heads, page_size, head_dim],  v [pages, heads, head_dim, page_size]
//   8 bits: scale = max|x| / 127 over a row (one head of one token), n = x / scale
//   rounded half to even
//
// Keys lie by token and values by element, each as the attention over the cache reads
// it: both of its products then take what they run along from consecutive bytes.
// Bound by memory: a new element is read once (4 bytes) and written once (1 or 4).
// A workgroup takes 16 places of one head that lie within a page's aligned group of 16, so
// the values, gathered through LDS, go out four places a lane, the group's 16 a line.  3 x 1365
// tokens, 8 heads of 128, 8 bits: 16 us to write (42 MB; 5 of them waiting for starts, lengths, table and rows in
// turn), 10 to read.
#include "mx_kv_cache.hpp"

#include <algorithm>

namespace mx {
namespace {

using kv::Batch;
using kv::Cache;

constexpr int kThreads = 256, kGroup = 16, kMaxDim = 128;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
template <class E>
struct alignas(4 * sizeof(E)) Four {
  E e[4];
};

struct Rows {  // one of k and v, outside the cache
  float* at;
  int64_t token, head;
};

// x / scale rounded half to even, of the exact quotient: a product with the reciprocal is off
// by a step at most, and what it leaves of x is exact (a fused multiply-add; FP32's least numbers
// would round it away: small rows are lifted first).
struct Steps {
  float lift, scale, half, inv;
  __device__ __forceinline__ explicit Steps(float s) {
    lift = s < 0x1p-60f ? 0x1p90f : 1.f;
    scale = s * lift;
    half = s > 0 ? 0.5f * scale : __builtin_inff();
    inv = s > 0 ? 1.f / scale : 0.f;  // (rows of a scale of 0 or NaN: no steps)
  }
  __device__ __forceinline__ int operator()(float x) const {
    x *= lift;
    float n = rintf(x * inv);
    const float rest = fmaf(-n, scale, x);
    const bool odd = int(n) & 1;
    if (rest > half || (rest == half && odd)) n += 1;
    if (rest < -half || (rest == -half && odd)) n -= 1;
    return int(fminf(fmaxf(n, -127.f), 127.f));
  }
};

template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int m = 1; m < L; m <<= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}

// The group of places of this workgroup: the positions first .. first + 15 of the
// sequence, of which rows lo .. hi - 1 (of the group's 16) are new tokens.
struct Places {
  int page, place, lo, hi;
  int64_t row;  // of place 0, so row + lo is a token of k and v
};
__device__ __forceinline__ bool places(const Cache& c, const Batch& b, int tile, Places& g) {
  SequenceTile t;
  if (!locate<kGroup, 2>(b.seqs, tile, t) || t.len == 0) return false;
  const int last = b.lengths[t.seq];
  const int64_t from = int64_t(last) - t.len;  // position of the first new token
  const int64_t group = (from >= 0 ? from / kGroup : -((-from + kGroup - 1) / kGroup)) + t.index;
  if (group * kGroup >= last) return false;
  g.lo = int(max(from - group * kGroup, int64_t(0)));
  g.hi = int(min(last - group * kGroup, int64_t(kGroup)));
  g.row = t.start + (group * kGroup - from);
  g.page = group < 0 ? -1 : kv::page_of(c, b, t.seq, int(group), g.place);
  return true;
}

template <bool I8>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(const Cache c, const Batch b, const Rows k, const Rows v) {
  using E = std::conditional_t<I8, int8_t, float>;
  __shared__ __attribute__((aligned(16))) E held[kGroup][kMaxDim + 4];  // values by row (the pitch keeps banks apart)
  Places g;
  if (!places(c, b, blockIdx.x, g) || g.page < 0) return;
  const int head = blockIdx.y, row = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const bool mine = row >= g.lo && row < g.hi;
  const int64_t at = (int64_t(g.page) * c.heads + head) * c.page_size + g.place;  // place 0's row in the cache
  // A row's 16 lanes have every sixteenth four of its elements.
  constexpr int N = kMaxDim / 64;
  f32x4 val[2][N];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const Rows& src = which ? v : k;
    const float* const x = src.at + (g.row + row) * src.token + head * src.head;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = (i * 16 + lane) * 4;
      val[which][i] = mine && d < c.dim ? *reinterpret_cast<const f32x4u*>(x + d) : f32x4{};
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float scale = 0;
    if constexpr (I8) {
      float most = 0, bad = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          most = fmaxf(most, fabsf(val[which][i][j]));
          bad = fmaxf(bad, fabsf(val[which][i][j]) <= 3.402823466e38f ? 0.f : 1.f);
        }
      scale = lanes_max<16>(most) / 127.f;
      if (lanes_max<16>(bad) > 0) scale = __builtin_nanf("");
      if (mine && lane == 0) (which ? c.vs : c.ks)[at + row] = scale;
    }
    const Steps steps(scale);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = (i * 16 + lane) * 4;
      if (d >= c.dim || !mine) continue;
      Four<E> e;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (I8) e.e[j] = E(steps(val[which][i][j]));
        else e.e[j] = val[which][i][j];
      }
      *reinterpret_cast<Four<E>*>(which ? &held[row][d] : static_cast<E*>(c.k) + (at + row) * c.dim + d) = e;
    }
  }
  __syncthreads();
  E* const out = static_cast<E*>(c.v) + (at - g.place) * c.dim + g.place;
  for (int i = threadIdx.x; i < c.dim * 4; i += kThreads) {
    const int d = i >> 2, p = (i & 3) * 4;
    E* const to = out + int64_t(d) * c.page_size + p;
    if (p >= g.lo && p + 4 <= g.hi) {
      *reinterpret_cast<Four<E>*>(to) = Four<E>{held[p][d], held[p + 1][d], held[p + 2][d], held[p + 3][d]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (p + j >= g.lo && p + j < g.hi) to[j] = held[p + j][d];
    }
  }
}

template <bool I8>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(const Cache c, const Batch b, const Rows k, const Rows v) {
  using E = std::conditional_t<I8, int8_t, float>;
  __shared__ __attribute__((aligned(16))) E held[kGroup][kMaxDim + 4];  // values by row (the pitch keeps banks apart)
  Places g;
  if (!places(c, b, blockIdx.x, g)) return;
  const bool here = g.page >= 0;
  const int head = blockIdx.y, row = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int64_t at = here ? (int64_t(g.page) * c.heads + head) * c.page_size + g.place : 0;
  if (here) {
    const E* const in = static_cast<const E*>(c.v) + (at - g.place) * c.dim + g.place;
    for (int i = threadIdx.x; i < c.dim * 4; i += kThreads) {
      const int d = i >> 2, p = (i & 3) * 4;
      const Four<E> f = *reinterpret_cast<const Four<E>*>(in + int64_t(d) * c.page_size + p);
#pragma unroll
      for (int j = 0; j < 4; ++j) held[p + j][d] = f.e[j];
    }
  }
  __syncthreads();
  if (row < g.lo || row >= g.hi) return;
  float ks = 1, vs = 1;
  if (I8 && here) ks = c.ks[at + row], vs = c.vs[at + row];
  float* const ko = k.at + (g.row + row) * k.token + head * k.head;
  float* const vo = v.at + (g.row + row) * v.token + head * v.head;
  for (int d = lane * 4; d < c.dim; d += 64) {
    f32x4 a{}, b{};
    if (here) {
      const Four<E> e = *reinterpret_cast<const Four<E>*>(static_cast<const E*>(c.k) + (at + row) * c.dim + d);
      const Four<E> f = *reinterpret_cast<const Four<E>*>(&held[row][d]);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = float(e.e[j]) * ks, b[j] = float(f.e[j]) * vs;
    }
    *reinterpret_cast<f32x4u*>(ko + d) = a;
    *reinterpret_cast<f32x4u*>(vo + d) = b;
  }
}

}  // namespace

int kv::check(const char* who, const mx_kv_cache* c, const mx_kv_batch* b) {
  MX_REQUIRE(c && b, MX_ERR_INVALID, who, ": null cache or batch");
  MX_REQUIRE(c->type == MX_KV_F32 || c->type == MX_KV_I8, MX_ERR_INVALID, who, ": unknown cache type ", c->type);
  MX_REQUIRE(c->pages >= 0 && c->heads >= 0 && b->tokens >= 0 && b->sequences >= 0 && b->table_width >= 0, MX_ERR_INVALID,
             who, ": negative size");
  MX_REQUIRE(c->page_size >= 16 && c->page_size % 16 == 0, MX_ERR_INVALID, who, ": page_size must be a multiple of 16, got ",
             c->page_size);
  MX_REQUIRE(c->head_dim >= 16 && c->head_dim % 16 == 0 && c->head_dim <= kMaxDim, MX_ERR_INVALID, who,
             ": head_dim must be a multiple of 16 up to ", kMaxDim, ", got ", c->head_dim);
  MX_REQUIRE(c->pages < (int64_t(1) << 31) && c->heads <= 65535 && c->page_size <= (1 << 20) && b->tokens <= (1 << 27) &&
                 b->sequences <= (1 << 21) && b->table_width <= (int64_t(1) << 30) / c->page_size,
             MX_ERR_INVALID, who, ": size out of range");
  MX_REQUIRE(b->tokens == 0 || b->sequences > 0, MX_ERR_INVALID, who, ": tokens of no sequence");
  MX_REQUIRE(b->starts || b->sequences == 0 || b->tokens % b->sequences == 0, MX_ERR_INVALID, who, ": ", b->tokens,
             " tokens do not divide into ", b->sequences, " sequences");
  return MX_OK;
}

int kv::check_buffers(const char* who, const mx_kv_cache* c, const mx_kv_batch* b) {
  MX_REQUIRE(b->lengths && (b->table || b->table_width == 0), MX_ERR_INVALID, who, ": null lengths or table");
  MX_REQUIRE(c->pages == 0 || (c->k && c->v && (c->type == MX_KV_F32 || (c->k_scale && c->v_scale))), MX_ERR_INVALID, who,
             ": null buffer of the cache");
  for (const void* p : {static_cast<const void*>(c->k), static_cast<const void*>(c->v),
                        static_cast<const void*>(c->k_scale), static_cast<const void*>(c->v_scale)})
    MX_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15u) == 0, MX_ERR_INVALID, who, ": the cache is not 16-byte aligned");
  return MX_OK;
}

kv::Cache kv::cache_of(const mx_kv_cache* c) {
  return {c->k, c->v, c->k_scale, c->v_scale, int(c->pages), int(c->heads), int(c->page_size), int(c->head_dim)};
}
kv::Batch kv::batch_of(const mx_kv_batch* b) {
  return {{b->starts, int(b->tokens), int(b->sequences)}, b->lengths, b->table, int(b->table_width)};
}

namespace {

template <bool WRITE>
int run(const char* who, const mx_kv_cache* c, const mx_kv_batch* b, const Rows& k, const Rows& v, void* stream) {
  MX_TRY(kv::check(who, c, b));
  if (b->tokens == 0 || c->heads == 0) return MX_OK;
  MX_REQUIRE(k.at && v.at, MX_ERR_INVALID, who, ": null buffer");
  MX_TRY(kv::check_buffers(who, c, b));
  const dim3 grid(unsigned(sequence_tiles(b->tokens, b->sequences, kGroup, 2)), unsigned(c->heads));
  hipStream_t s = resolve_stream(stream);
  const Cache cache = kv::cache_of(c);
  const Batch batch = kv::batch_of(b);
  if constexpr (WRITE) {
    if (c->type == MX_KV_I8) hipLaunchKernelGGL((kv_write_kernel<true>), grid, dim3(kThreads), 0, s, cache, batch, k, v);
    else hipLaunchKernelGGL((kv_write_kernel<false>), grid, dim3(kThreads), 0, s, cache, batch, k, v);
  } else {
    if (c->type == MX_KV_I8) hipLaunchKernelGGL((kv_read_kernel<true>), grid, dim3(kThreads), 0, s, cache, batch, k, v);
    else hipLaunchKernelGGL((kv_read_kernel<false>), grid, dim3(kThreads), 0, s, cache, batch, k, v);
  }
  MX_LAUNCHED();
  return MX_OK;
}

}  // namespace
}  // namespace mx

using namespace mx;

extern "C" int mx_kv_cache_write(const mx_kv_cache* c, const mx_kv_batch* b, const float* k, int64_t k_token, int64_t k_head,
                                 const float* v, int64_t v_token, int64_t v_head, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  return run<true>("mx_kv_cache_write", c, b, {const_cast<float*>(k), k_token, k_head}, {const_cast<float*>(v), v_token, v_head},
                   stream);
  MX_ABI_END
}

extern "C" int mx_kv_cache_read(const mx_kv_cache* c, const mx_kv_batch* b, float* k, float* v, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  const int64_t dim = c ? c->head_dim : 0, token = c ? c->heads * dim : 0;
  return run<false>("mx_kv_cache_read", c, b, {k, token, dim}, {v, token, dim}, stream);
  MX_ABI_END
}
