// Attention of new tokens over a paged cache of keys and values (FP32 or 8 bits).
//
//   s = scale q k,  p = softmax over the keys that the row sees,  out = sum p v
//   8 bits: k = n scale, so s = scale (q n) scale_k, and p v = (p scale_v) n
//
// A single token is bound by the bytes of the cache, a chunk of many by the matrix
// instructions.  The rows of a tile are the new tokens of one sequence with all query
// heads that share a key head, so a key or value is read once for all of them.  A signed
// byte is a bf16 number: products with it take three matrix instructions (the row's
// three pieces) in place of six, and the scales go to the scores and the probabilities.
//
// A wave takes tiles of 32 keys straight from the cache into operand fragments: lane l
// reads 16 elements of key tile_row(l % 32) and 16 keys of element tile_row(l % 32), each
// from consecutive places, in half l / 32 of the tile (which may lie in another page).
// The keys of a row tile are dealt to the workgroup's waves, and to several workgroups
// where there are few rows; waves join through LDS, workgroups through the workspace and a
// second launch, both in a fixed order.
#include <algorithm>
#include <cmath>

#include "mx_attention.hpp"
#include "mx_kv_cache.hpp"

namespace mx {
namespace {

using namespace attn;
using kv::Batch;
using kv::Cache;
using mfma::bf16x2;
using mfma::f32x2;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = 4;

struct PagedArgs {
  Cache c;
  Batch b;
  const float* q;
  int64_t q_token, q_head;
  int heads, group, tiles, splits;
  Mask mask;
  float scale;
  float *out, *part;
};

// The workgroups' parts: [tile][kv head][split] of 32 maxima, 32 sums and 32 rows of dim.
__device__ __forceinline__ int64_t part_at(const PagedArgs& a, int tile, int head, int split) {
  return ((int64_t(tile) * a.c.heads + head) * a.splits + split) * (kTile * (2 + a.c.dim));
}

// 16 elements as operand pieces: one where they are bytes, three where they are FP32.
template <bool I8>
struct Sixteen;
template <>
struct Sixteen<true> {
  i32x4 raw;
  __device__ __forceinline__ void load(const void* p) { raw = *static_cast<const i32x4*>(p); }
  // Elements 8 t .. 8 t + 7.
  __device__ __forceinline__ bf16x8 half(int t) const {
    mfma::u32x4 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int x = raw[2 * t + i];
      w[2 * i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{float(int8_t(x)), float(int8_t(x >> 8))}), bf16x2));
      w[2 * i + 1] =
          __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{float(int8_t(x >> 16)), float(x >> 24)}), bf16x2));
    }
    return __builtin_bit_cast(bf16x8, w);
  }
};
template <>
struct Sixteen<false> {
  f32x4 raw[4];
  __device__ __forceinline__ void load(const void* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = static_cast<const f32x4*>(p)[i];
  }
  __device__ __forceinline__ Frag3 half(int t) const { return split8(raw[2 * t], raw[2 * t + 1]); }
};

__device__ __forceinline__ void mma_all(const bf16x8& a, const Frag3& b, f32x16& small, f32x16& large) {
  small = mma(a, b.lo, small);
  small = mma(a, b.mid, small);
  large = mma(a, b.hi, large);
}
__device__ __forceinline__ void mma_all(const Frag3& a, const Frag3& b, f32x16& small, f32x16& large) {
  small = mma_small(a, b, small);
  large = mma_large(a, b, large);
}

template <int DP, bool I8>
__global__ __launch_bounds__(kThreads) void paged_kernel(const PagedArgs a) {
  constexpr int kUnits = DP / 32, kPitch = DP + 4;
  __shared__ float stat[2][kWaves][kTile], sum[kTile][kPitch];
  using E = std::conditional_t<I8, int8_t, float>;
  const Cache& c = a.c;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int kv_head = blockIdx.y;
  SequenceTile t;
  if (!locate<kTile>(a.b.seqs, blockIdx.x, t) || t.index * kTile >= t.len) return;
  const int length = int(min(int64_t(max(a.b.lengths[t.seq], 0)), int64_t(a.b.width) * c.page_size));
  const int first = a.b.lengths[t.seq] - t.len / a.group;  // position of the sequence's first new token
  // The lane's row: a token and a query head.
  const int row = t.index * kTile + (lane & 31), last_row = min(t.len, (t.index + 1) * kTile) - 1;
  const int token = min(row, t.len - 1) / a.group, pos = first + token;
  const int head = kv_head * a.group + min(row, t.len - 1) - token * a.group;
  const int64_t flat = t.start / a.group + token;
  Frag3 q[2 * kUnits];
  {
    const float* const src = a.q + flat * a.q_token + head * a.q_head + 16 * h;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      f32x4 v[4] = {};
      if (32 * u + 16 * h < c.dim) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const f32x4u*>(src + 32 * u + 4 * i);
      }
      q[2 * u] = split8(v[0], v[1]);
      q[2 * u + 1] = split8(v[2], v[3]);
    }
  }
  const int i0 = first + t.index * kTile / a.group, i1 = min(first + last_row / a.group, length - 1);
  const float scale = a.scale * kLog2E;
  f32x16 o[kUnits] = {};
  float m = -__builtin_inff(), l = 0;
  const KeyTiles keys(a.mask, max(i0, 0), i1);
  const int64_t token_bytes = c.dim * int64_t(sizeof(E));
  const int count = c.pages ? keys.count : 0;
  for (int n = blockIdx.z * kWaves + wave; n < count; n += kWaves * a.splits) {
    const int j0 = keys.tile(n) * kTile;
    int place[2], page[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) page[g] = kv::page_of(c, a.b, t.seq, (j0 >> 4) + g, place[g]);
    const bool whole = page[0] >= 0 && page[1] >= 0 && j0 + kTile <= length;
    int64_t at[2];  // places' rows in the cache; those of absent pages are page 0's, and seen by no row
#pragma unroll
    for (int g = 0; g < 2; ++g) at[g] = (int64_t(max(page[g], 0)) * c.heads + kv_head) * c.page_size;
    const int kg = lane >> 2 & 1, kr = (lane & 31) >> 3 << 2 | (lane & 3);  // tile_row's half and rest
    const char* const krow = static_cast<const char*>(c.k) + ((kg ? at[1] + place[1] : at[0] + place[0]) + kr) * token_bytes;
    const int64_t mine = h ? at[1] : at[0];
    const int in_page = h ? place[1] : place[0];
    // ---- scores
    f32x16 x{}, small{};
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      Sixteen<I8> k{};
      if (32 * u + 16 * h < c.dim) k.load(krow + (32 * u + 16 * h) * sizeof(E));
      mma_all(k.half(0), q[2 * u], small, x);
      mma_all(k.half(1), q[2 * u + 1], small, x);
    }
    x += small;
    f32x16 vscale;
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 ks = *reinterpret_cast<const f32x4*>(c.ks + mine + in_page + 4 * i);
        const f32x4 vs = *reinterpret_cast<const f32x4*>(c.vs + mine + in_page + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * i + e] *= ks[e], vscale[4 * i + e] = vs[e];
      }
    }
    const bool part = !whole || !a.mask.all(i0, i1, j0, j0 + kTile - 1);
    const bool here = (h ? page[1] : page[0]) >= 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= scale;
    if (part) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = j0 + 16 * h + r;
        if (!here || j >= length || !a.mask.sees(pos, j)) x[r] = -__builtin_inff();
      }
    }
    // ---- values
    Sixteen<I8> v[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int d = 32 * u + tile_row(lane & 31);
      v[u] = {};
      if (d < c.dim) v[u].load(static_cast<const E*>(c.v) + mine * c.dim + int64_t(d) * c.page_size + in_page);
    }
    if constexpr (!I8) {
      // What no row sees counts as zero, and a value that is not finite as a NaN score of its key.
      if (part) {
        uint32_t bad = 0;
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float e = v[u].raw[r >> 2][r & 3];
            const bool no = !here || j0 + 16 * h + r >= length, odd = !(fabsf(e) <= 3.402823466e38f);
            if (odd && !no) bad |= 1u << r;
            if (no || odd) v[u].raw[r >> 2][r & 3] = 0;
          }
        if (__any(bad != 0)) {
#pragma unroll
          for (int s = 1; s < 32; s <<= 1) bad |= __shfl_xor(int(bad), s, 64);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (bad >> r & 1 && x[r] != -__builtin_inff()) x[r] = __builtin_nanf("");
        }
      }
    }
    // ---- softmax so far
    float top = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float next = fmaxf(m, top), base = next == -__builtin_inff() ? 0.f : next;
    const float keep = exp2_(m - base);
    float add = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = exp2_(x[r] - base);
      add += x[r];
    }
    l = fmaf(l, keep, add);
    m = next;
    if constexpr (I8) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = x[r] == 0 ? 0.f : x[r] * vscale[r];  // an unseen scale may be anything
    }
    const Frag3 p[2] = {split_half(x, 0), split_half(x, 1)};
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      f32x16 acc{}, lower{};
      mma_all(v[u].half(0), p[0], lower, acc);
      mma_all(v[u].half(1), p[1], lower, acc);
      o[u] = o[u] * keep + (acc + lower);
    }
  }
  l += __shfl_xor(l, 32, 64);
  // ---- the workgroup's waves, in order
  if (h == 0) stat[0][wave][lane] = m, stat[1][wave][lane] = l;
  __syncthreads();
  float all = -__builtin_inff(), total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all = fmaxf(all, stat[0][w][lane & 31]);
  const float base = all == -__builtin_inff() ? 0.f : all;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) total = fmaf(stat[1][w][lane & 31], exp2_(stat[0][w][lane & 31] - base), total);
  const float mul = exp2_(m - base);
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4* const to = reinterpret_cast<f32x4*>(&sum[lane & 31][32 * u + 16 * h + 4 * i]);
          f32x4 add;
#pragma unroll
          for (int e = 0; e < 4; ++e) add[e] = o[u][4 * i + e] * mul;
          *to = w ? *to + add : add;
        }
    }
    __syncthreads();
  }
  // ---- out: 8 threads a row
  const int r = threadIdx.x >> 3, cc = threadIdx.x & 7, orow = t.index * kTile + r;
  if (wave == 0 && h == 0) stat[0][0][lane] = all, stat[1][0][lane] = total;
  __syncthreads();
  if (orow >= t.len) return;
  if (a.splits > 1) {
    float* const to = a.part + part_at(a, blockIdx.x, kv_head, blockIdx.z);
    if (cc == 0) to[r] = stat[0][0][r], to[kTile + r] = stat[1][0][r];
    for (int e = cc * 4; e < c.dim; e += 32)
      *reinterpret_cast<f32x4*>(to + 2 * kTile + r * c.dim + e) = *reinterpret_cast<const f32x4*>(&sum[r][e]);
    return;
  }
  const float den = stat[1][0][r], inv = den == 0 ? 0.f : 1.f / den;
  const int otoken = orow / a.group;
  float* const to = a.out + ((t.start / a.group + otoken) * int64_t(a.heads) + kv_head * a.group + orow - otoken * a.group) * c.dim;
  for (int e = cc * 4; e < c.dim; e += 32) *reinterpret_cast<f32x4u*>(to + e) = *reinterpret_cast<const f32x4*>(&sum[r][e]) * inv;
}

// The workgroups that shared a row tile's keys, in order: 8 threads a row.
__global__ __launch_bounds__(kThreads) void paged_join_kernel(const PagedArgs a) {
  SequenceTile t;
  if (!locate<kTile>(a.b.seqs, blockIdx.x, t) || t.index * kTile >= t.len) return;
  const int r = threadIdx.x >> 3, cc = threadIdx.x & 7, row = t.index * kTile + r, kv_head = blockIdx.y;
  if (row >= t.len) return;
  const float* const part = a.part + part_at(a, blockIdx.x, kv_head, 0);
  const int64_t step = kTile * (2 + a.c.dim);
  float all = -__builtin_inff(), total = 0;
  for (int i = 0; i < a.splits; ++i) all = fmaxf(all, part[i * step + r]);
  const float base = all == -__builtin_inff() ? 0.f : all;
  for (int i = 0; i < a.splits; ++i) total = fmaf(part[i * step + kTile + r], exp2_(part[i * step + r] - base), total);
  const float inv = total == 0 ? 0.f : 1.f / total;
  const int token = row / a.group;
  float* const to = a.out + ((t.start / a.group + token) * int64_t(a.heads) + kv_head * a.group + row - token * a.group) * a.c.dim;
  for (int e = cc * 4; e < a.c.dim; e += 32) {
    f32x4 v{};
    for (int i = 0; i < a.splits; ++i)
      v += *reinterpret_cast<const f32x4*>(part + i * step + 2 * kTile + r * a.c.dim + e) * exp2_(part[i * step + r] - base);
    *reinterpret_cast<f32x4u*>(to + e) = v * inv;
  }
}

int check(const char* who, const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b) {
  MX_REQUIRE(d, MX_ERR_INVALID, who, ": null descriptor");
  MX_TRY(kv::check(who, c, b));
  MX_REQUIRE(d->heads >= 0, MX_ERR_INVALID, who, ": negative size");
  MX_REQUIRE(d->heads == 0 || (c->heads > 0 && d->heads % c->heads == 0), MX_ERR_INVALID, who, ": ", d->heads,
             " heads do not share ", c->heads, " key heads evenly");
  MX_REQUIRE(d->heads <= (1 << 20) && b->tokens * std::max<int64_t>(d->heads, 1) <= (int64_t(1) << 30), MX_ERR_INVALID, who,
             ": size out of range");
  MX_REQUIRE(d->window >= 0 && d->sinks >= 0, MX_ERR_INVALID, who, ": negative window or sinks");
  MX_REQUIRE(std::isfinite(d->scale), MX_ERR_INVALID, who, ": the scale must be finite");
  return MX_OK;
}

// How many workgroups share a row tile's keys: as many as fill the chip twice, each wave
// with two tiles of keys at least.
int splits_of(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b, int64_t tiles) {
  int64_t keys = b->table_width * c->page_size;
  if (d->window) keys = std::min(keys, d->window + d->sinks + b->tokens);
  const int64_t most = std::max<int64_t>(1, keys / (kTile * kWaves * 2));
  return int(std::max<int64_t>(1, std::min<int64_t>({most, int64_t(cu_count()) * 2 / std::max<int64_t>(1, tiles * c->heads), 64})));
}

int64_t row_tiles(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b) {
  return sequence_tiles(b->tokens * (d->heads / c->heads), b->sequences, kTile);
}

int64_t paged_workspace(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b) {
  if (b->tokens == 0 || d->heads == 0) return 0;
  const int64_t tiles = row_tiles(d, c, b), splits = splits_of(d, c, b, tiles);
  return splits == 1 ? 0 : tiles * c->heads * splits * kTile * (2 + c->head_dim) * 4;
}

template <int DP>
void launch(const PagedArgs& a, int type, dim3 grid, hipStream_t s) {
  if (type == MX_KV_I8) hipLaunchKernelGGL((paged_kernel<DP, true>), grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL((paged_kernel<DP, false>), grid, dim3(kThreads), 0, s, a);
}

}  // namespace
}  // namespace mx

using namespace mx;

extern "C" int mx_attention_paged_workspace(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b, int64_t* bytes) {
  MX_ABI_BEGIN
  MX_TRY(check("mx_attention_paged_workspace", d, c, b));
  MX_REQUIRE(bytes, MX_ERR_INVALID, "mx_attention_paged_workspace: null result");
  *bytes = paged_workspace(d, c, b);
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_attention_paged(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b, const float* q, float* out,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  const char* const who = "mx_attention_paged";
  MX_TRY(check(who, d, c, b));
  if (b->tokens == 0 || d->heads == 0) return MX_OK;
  MX_REQUIRE(q && out, MX_ERR_INVALID, who, ": null buffer");
  MX_TRY(kv::check_buffers(who, c, b));
  hipStream_t s = resolve_stream(stream);
  Workspace ws;
  MX_TRY(ws.take(who, workspace, workspace_bytes, paged_workspace(d, c, b), s));
  PagedArgs a{};
  a.c = kv::cache_of(c);
  a.b = kv::batch_of(b);
  a.heads = int(d->heads), a.group = int(d->heads / c->heads);
  a.b.seqs.per = a.group;
  a.q = q, a.q_token = d->q_token, a.q_head = d->q_head;
  a.tiles = int(row_tiles(d, c, b));
  a.splits = splits_of(d, c, b, a.tiles);
  a.mask = {int(std::min<int64_t>(d->window, 1 << 30)), int(std::min<int64_t>(d->sinks, 1 << 30))};
  a.scale = float(d->scale);
  a.out = out, a.part = ws.as<float>();
  const dim3 grid(unsigned(a.tiles), unsigned(a.c.heads), unsigned(a.splits));
  switch ((a.c.dim + 31) / 32) {
    case 1: launch<32>(a, c->type, grid, s); break;
    case 2: launch<64>(a, c->type, grid, s); break;
    case 3: launch<96>(a, c->type, grid, s); break;
    default: launch<128>(a, c->type, grid, s); break;
  }
  MX_LAUNCHED();
  if (a.splits > 1) {
    hipLaunchKernelGGL(paged_join_kernel, dim3(grid.x, grid.y), dim3(kThreads), 0, s, a);
    MX_LAUNCHED();
  }
  return MX_OK;
  MX_ABI_END
}
