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
// A wave takes tiles of 64 keys straight from the cache into operand fragments of
// v_mfma_f32_16x16x32_bf16 (16 rows: a token's query heads seldom are more, and both its
// registers and its matrix instructions are half of the 32 x 32 form's).  Quarter g of the
// wave holds keys 16 g .. 16 g + 15 of a tile: the scores that it ends with, and the
// values that it reads, 16 consecutive places of one element; a key's elements are read 16
// at a time too.  Keys are read a tile ahead of their products, their pages two.
// The keys of a row tile are dealt to the workgroup's waves, and to several workgroups
// where there are few rows; waves join through LDS, workgroups through the workspace and a
// second launch, both in a fixed order.
#include <algorithm>
#include <cmath>

#include "mx_attention_paged.hpp"

namespace mx {
namespace {

using namespace attn;
using kv::Batch;
using kv::Cache;

constexpr int kThreads = 256, kWaves = 4, kRows = 16, kKeys = 64;

struct PagedArgs : Paged {
  int tiles, splits, span;  // span: tiles of keys to a workgroup
  float* part;
};

// The workgroups' parts: [row tile][kv head][split] of 16 maxima, 16 sums and 16 rows of dim.
__device__ __forceinline__ int64_t part_at(const PagedArgs& a, int tile, int head, int split) {
  return ((int64_t(tile) * a.c.heads + head) * a.splits + split) * (kRows * (2 + a.c.dim));
}

__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma_all(const bf16x8& a, const Frag3& b, f32x4 c) {
  return mma16(a, b.hi, mma16(a, b.mid, mma16(a, b.lo, c)));
}
__device__ __forceinline__ f32x4 mma_all(const Frag3& a, const Frag3& b, f32x4 c) {
  c = mma16(a.lo, b.hi, c);
  c = mma16(a.hi, b.lo, c);
  c = mma16(a.mid, b.mid, c);
  c = mma16(a.mid, b.hi, c);
  return mma16(a.hi, b.hi, mma16(a.hi, b.mid, c));
}

// Over the wave's quarters, which hold the same 16 rows.
__device__ __forceinline__ float quarters_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}

// The page of a lane's group of 16 keys, and the group's first place in it.
struct Place {
  int page, place;
  __device__ __forceinline__ void find(const Cache& c, const Batch& b, int seq, int tile, int group) {
    page = kv::page_of(c, b, seq, tile * (kKeys / 16) + group, place);
  }
};

// 64 tokens, 32 heads over 8 key heads of 128, 8-bit contexts of 819 to 8192: 186 to 197 us, 3.4 to 3.6 TB/s (equal contexts
// of 8192 4.2 TB/s with the join; reads alone reach 7.0): waves wait 53 % of their cycles, and uneven lengths leave the chip
// half full at the end.  Without reading keys ahead 335 us.  17 x 2 tokens, FP32, contexts up to 3001, 9 heads of 80:
// 50 us, 4.2 TB/s; keys read ahead, at one wave a SIMD, 74.
template <int DP, bool I8>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void paged_kernel(const PagedArgs a) {
  constexpr int kUnits = DP / 64, kBlocks = DP / 16, kPitch = DP + 4;
  __shared__ __attribute__((aligned(16))) float stat[2][kWaves][kRows], sum[kWaves][kRows][kPitch];
  using E = std::conditional_t<I8, int8_t, float>;
  const Cache& c = a.c;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const int kv_head = blockIdx.y;
  RowTile<kRows> rt;
  if (!rt.find(a, blockIdx.x)) return;
  const SequenceTile& t = rt.t;
  const KeyTiles<kKeys> keys(a.mask, max(rt.i0, 0), rt.end);
  // This workgroup's tiles of keys, dealt to its waves.
  const int begin = blockIdx.z * a.span, end = c.pages ? min(keys.count, begin + a.span) : 0;
  if (blockIdx.z && begin >= end) return;
  // The lane's row: a token and a query head.
  const int row = min(t.index * kRows + col, t.len - 1), token = row / a.group, pos = rt.first + token;
  const int head = kv_head * a.group + row - token * a.group;
  const int kg = col >> 2;  // the group of the keys whose elements this lane reads
  Place kp, vp;             // of this tile's keys and values
  const auto find = [&](int n, Place& k, Place& v) {
    const int tile = keys.tile(min(n, end - 1));
    k.find(c, a.b, t.seq, tile, kg);
    v.find(c, a.b, t.seq, tile, g);
  };
  // Key 16 kg + 4 i + col % 4 is row col of the tile's i-th block of 16.  (FP32 keys have no registers
  // to wait in with two waves a SIMD, which gains more than reading ahead does.)
  constexpr bool kAhead = I8;
  Sixteen<I8> k[kAhead ? 4 : 1][kUnits];
  const auto fetch = [&](const Place& at, int i0, int i1) {
    const E* const from = static_cast<const E*>(c.k) +
                          ((int64_t(max(at.page, 0)) * c.heads + kv_head) * c.page_size + at.place + (col & 3)) * c.dim + 16 * g;
#pragma unroll
    for (int i = i0; i < i1; ++i)
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        Sixteen<I8>& to = k[kAhead ? i : 0][u];
        to = {};
        if (64 * u + 16 * g < c.dim) to.load(from + 4 * i * c.dim + 64 * u);
      }
  };
  const int from = begin + wave;
  Frag3 q[2 * kUnits];
  if (from < end) {
    find(from, kp, vp);
    const float* const src = a.q + (t.start / a.group + token) * a.q_token + head * a.q_head + 16 * g;
    const float scale = a.scale * kLog2E;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      f32x4 v[4] = {};
      if (64 * u + 16 * g < c.dim) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const f32x4u*>(src + 64 * u + 4 * i) * scale;
      }
      q[2 * u] = split8(v[0], v[1]);
      q[2 * u + 1] = split8(v[2], v[3]);
    }
    if (kAhead) fetch(kp, 0, 4);
  }
  f32x4 o[kBlocks] = {};
  float m = -__builtin_inff(), l = 0;  // of the exponents
  for (int n = from; n < end; n += kWaves) {
    const int j0 = keys.tile(n) * kKeys, j = j0 + 16 * g;  // the lane's 16 keys: j ..
    const bool here = vp.page >= 0;
    const int64_t places = (int64_t(max(vp.page, 0)) * c.heads + kv_head) * c.page_size;
    Place kn, vn;
    find(n + kWaves, kn, vn);
    // ---- scales and values, while the scores are computed
    f32x4 ks[4], vs[4];
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ks[i] = *reinterpret_cast<const f32x4*>(c.ks + places + vp.place + 4 * i);
        vs[i] = *reinterpret_cast<const f32x4*>(c.vs + places + vp.place + 4 * i);
      }
    }
    const E* const vfrom = static_cast<const E*>(c.v) + places * c.dim + int64_t(col) * c.page_size + vp.place;
    const auto values = [&](int b) {
      Sixteen<I8> v{};
      if (16 * b < c.dim) v.load(vfrom + int64_t(16 * b) * c.page_size);
      return v;
    };
    Sixteen<I8> v[kAhead ? kBlocks : 1];
    if constexpr (kAhead) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) v[b] = values(b);
    }
    // ---- scores: block i gives the lane keys j + 4 i .. + 3
    float x[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 acc{};
      if (!kAhead) fetch(kp, i, i + 1);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (64 * u >= c.dim) continue;
        acc = mma_all(k[kAhead ? i : 0][u].half(0), q[2 * u], acc);
        acc = mma_all(k[kAhead ? i : 0][u].half(1), q[2 * u + 1], acc);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = I8 ? fmaf(vs[i][e], 0.f, acc[e] * ks[i][e]) : acc[e];  // (a NaN value: a NaN score)
    }
    if (kAhead && n + kWaves < end) fetch(kn, 0, 4);
    const bool part = __any(!here || j + 16 > rt.length) || !a.mask.all(rt.i0, rt.i1, j0, j0 + kKeys - 1);
    if (part) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!here || j + r >= rt.length || !a.mask.sees(pos, j + r)) x[r] = -__builtin_inff();
      if constexpr (!I8) {
        // A value that is not finite is a NaN score of its key, and zero (below).
        uint32_t bad = 0;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          if (16 * b >= c.dim) continue;
          const Sixteen<I8> e = values(b);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!finite(e.raw[r >> 2][r & 3]) && here && j + r < rt.length) bad |= 1u << r;
        }
        if (__any(bad != 0)) {
#pragma unroll
          for (int s = 1; s < 16; s <<= 1) bad |= __shfl_xor(int(bad), s, 64);
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
    const float next = fmaxf(m, quarters_max(top)), base = next == -__builtin_inff() ? 0.f : next;
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
      for (int r = 0; r < 16; ++r) x[r] = times(x[r], vs[r >> 2][r & 3]);  // an unseen scale may be anything
    }
    const Frag3 p[2] = {split8(f32x4{x[0], x[1], x[2], x[3]}, f32x4{x[4], x[5], x[6], x[7]}),
                        split8(f32x4{x[8], x[9], x[10], x[11]}, f32x4{x[12], x[13], x[14], x[15]})};
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      if (16 * b >= c.dim) continue;
      if constexpr (!kAhead) {
        v[0] = values(b);
        if (part) {  // what no row sees, or no finite number, counts as zero
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!here || j + r >= rt.length || !finite(v[0].raw[r >> 2][r & 3])) v[0].raw[r >> 2][r & 3] = 0;
        }
      }
      const Sixteen<I8>& e = v[kAhead ? b : 0];
      o[b] = o[b] * keep + mma_all(e.half(1), p[1], mma_all(e.half(0), p[0], f32x4{}));
    }
    kp = kn, vp = vn;
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  // ---- the workgroup's waves, in order: 16 threads a row
  if (g == 0) stat[0][wave][col] = m, stat[1][wave][col] = l;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) *reinterpret_cast<f32x4*>(&sum[wave][col][16 * b + 4 * g]) = o[b];
  __syncthreads();
  const int r = threadIdx.x >> 4, cc = threadIdx.x & 15, orow = t.index * kRows + r;
  if (orow >= t.len) return;
  float all = -__builtin_inff(), total = 0, weight[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all = fmaxf(all, stat[0][w][r]);
  const float base = all == -__builtin_inff() ? 0.f : all;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    weight[w] = exp2_(stat[0][w][r] - base);
    total = fmaf(stat[1][w][r], weight[w], total);
  }
  const auto joined = [&](int e) {
    f32x4 v{};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += *reinterpret_cast<const f32x4*>(&sum[w][r][e]) * weight[w];
    return v;
  };
  if (a.splits > 1) {
    float* const to = a.part + part_at(a, blockIdx.x, kv_head, blockIdx.z);
    if (cc == 0) to[r] = all, to[kRows + r] = total;
    for (int e = cc * 4; e < c.dim; e += 64) *reinterpret_cast<f32x4*>(to + 2 * kRows + r * c.dim + e) = joined(e);
    return;
  }
  const float inv = total == 0 ? 0.f : 1.f / total;
  const int otoken = orow / a.group;
  float* const to = a.out + ((t.start / a.group + otoken) * int64_t(a.heads) + kv_head * a.group + orow - otoken * a.group) * c.dim;
  for (int e = cc * 4; e < c.dim; e += 64) *reinterpret_cast<f32x4u*>(to + e) = joined(e) * inv;
}

// The workgroups that shared a row tile's keys, in order: 16 threads a row, which first share
// out the workgroups' weights.
constexpr int kMaxSplits = 64;
__global__ __launch_bounds__(kThreads) void paged_join_kernel(const PagedArgs a) {
  __shared__ float weight[kRows][kMaxSplits];
  RowTile<kRows> rt;
  if (!rt.find(a, blockIdx.x)) return;
  const SequenceTile& t = rt.t;
  const int r = threadIdx.x >> 4, cc = threadIdx.x & 15, row = t.index * kRows + r, kv_head = blockIdx.y;
  const KeyTiles<kKeys> keys(a.mask, max(rt.i0, 0), rt.end);
  const int splits = a.c.pages ? max(1, (keys.count + a.span - 1) / a.span) : 1;  // those that have left a part
  const float* const part = a.part + part_at(a, blockIdx.x, kv_head, 0);
  const int64_t step = kRows * (2 + a.c.dim);
  float m[kMaxSplits / 16], l[kMaxSplits / 16], all = -__builtin_inff(), total = 0;
#pragma unroll
  for (int i = 0; i < kMaxSplits / 16; ++i) {
    const int at = cc + 16 * i;
    const bool has = at < splits && row < t.len;
    m[i] = has ? part[at * step + r] : -__builtin_inff();
    l[i] = has ? part[at * step + kRows + r] : 0.f;
    all = fmaxf(all, m[i]);
  }
#pragma unroll
  for (int s = 1; s < 16; s <<= 1) all = fmaxf(all, __shfl_xor(all, s, 64));
  const float base = all == -__builtin_inff() ? 0.f : all;
#pragma unroll
  for (int i = 0; i < kMaxSplits / 16; ++i) {
    const float w = exp2_(m[i] - base);
    weight[r][cc + 16 * i] = w;
    total = fmaf(l[i], w, total);
  }
#pragma unroll
  for (int s = 1; s < 16; s <<= 1) total += __shfl_xor(total, s, 64);
  __syncthreads();
  if (row >= t.len) return;
  const float inv = total == 0 ? 0.f : 1.f / total;
  const int token = row / a.group;
  float* const to = a.out + ((t.start / a.group + token) * int64_t(a.heads) + kv_head * a.group + row - token * a.group) * a.c.dim;
  for (int e = cc * 4; e < a.c.dim; e += 64) {
    const float* const from = part + 2 * kRows + r * a.c.dim + e;
    f32x4 v{};
#pragma unroll 8
    for (int i = 0; i < splits; ++i) v += *reinterpret_cast<const f32x4*>(from + i * step) * weight[r][i];
    *reinterpret_cast<f32x4u*>(to + e) = v * inv;
  }
}

int check(const char* who, const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b) {
  MX_REQUIRE(d, MX_ERR_INVALID, who, ": null descriptor");
  MX_TRY(kv::check(who, c, b));
  MX_REQUIRE(d->heads >= 0, MX_ERR_INVALID, who, ": negative size");
  MX_REQUIRE(d->heads == 0 || (c->heads > 0 && d->heads % c->heads == 0), MX_ERR_INVALID, who, ": ", d->heads,
             " heads do not share ", c->heads, " key heads evenly");
  MX_REQUIRE(d->heads <= (1 << 20) && b->tokens * std::max<int64_t>(d->heads, 1) <= (1 << 27), MX_ERR_INVALID, who,
             ": size out of range");
  MX_REQUIRE(d->window >= 0 && d->sinks >= 0, MX_ERR_INVALID, who, ": negative window or sinks");
  MX_REQUIRE(std::isfinite(d->scale), MX_ERR_INVALID, who, ": the scale must be finite");
  return MX_OK;
}

int64_t row_tiles(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b) {
  return sequence_tiles(b->tokens * (d->heads / c->heads), b->sequences, kRows);
}

// How a row tile's keys are dealt: `span` tiles of 64 to a workgroup, as many workgroups as even out
// lengths that the host does not know: eight a CU if all were of the table's length (the batch
// above: 220 us with up to four, 189 with eight, 188 with 16, 199 with 32; 16 contexts of up to 16384
// 121, 105, 109 and 109).  The table's width stands for the lengths, so a wide table leaves short contexts to few workgroups
// (one token over 4096, 4 key heads of 128: 12.8 us with a table of 4096 positions, 33.6 of 131072).
struct Split {
  int splits, span;
};
Split split_of(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b) {
  int64_t keys = b->table_width * c->page_size;
  // (never less than a row tile's keys: its window may begin and end inside a tile of 64; a window may be any number)
  if (d->window) keys = std::min(keys, std::min(d->window, keys) + std::min(d->sinks, keys) + b->tokens + 2 * kKeys);
  const int64_t most = std::max<int64_t>(1, (keys + kKeys - 1) / kKeys), rows = std::max<int64_t>(1, row_tiles(d, c, b) * c->heads);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(int64_t(cu_count()) * 8 / rows, kMaxSplits));
  // a tile of keys to a wave where even that leaves CUs idle (one token over 4096 keys 13.9 us, with two
  // tiles 16.0, before waves joined behind one barrier: 12.7 now), else four
  const int64_t least = rows * ((most + kWaves - 1) / kWaves) <= cu_count() * 2 ? kWaves : kWaves * 4;
  const int64_t span = std::max<int64_t>(((most + want - 1) / want + kWaves - 1) / kWaves * kWaves, least);
  return {int((most + span - 1) / span), int(span)};
}

int64_t paged_workspace(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b) {
  if (b->tokens == 0 || d->heads == 0) return 0;
  if (const int64_t chunk = chunk_workspace(d, c, b)) return chunk;
  const int64_t splits = split_of(d, c, b).splits;
  return splits == 1 ? 0 : row_tiles(d, c, b) * c->heads * splits * kRows * (2 + c->head_dim) * 4;
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
  a.out = out, a.q = q, a.q_token = d->q_token, a.q_head = d->q_head;
  // (positions go up to 2^31 - 2, keys to 2^30 - 1: these limits hide nothing)
  a.mask = {int(std::min<int64_t>(d->window, INT32_MAX)), int(std::min<int64_t>(d->sinks, 1 << 30))};
  a.scale = float(d->scale);
  if (chunk_workspace(d, c, b)) return chunk_attention(a, d, c, b, ws.as<char>(), s);
  a.tiles = int(row_tiles(d, c, b));
  const Split split = split_of(d, c, b);
  a.splits = split.splits, a.span = split.span;
  a.part = ws.as<float>();
  const dim3 grid(unsigned(a.tiles), unsigned(a.c.heads), unsigned(a.splits));
  if (a.c.dim <= 64) launch<64>(a, c->type, grid, s);
  else launch<128>(a, c->type, grid, s);
  MX_LAUNCHED();
  if (a.splits > 1) {
    hipLaunchKernelGGL(paged_join_kernel, dim3(grid.x, grid.y), dim3(kThreads), 0, s, a);
    MX_LAUNCHED();
  }
  return MX_OK;
  MX_ABI_END
}
