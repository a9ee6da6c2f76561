// Causal attention of packed sequences, forward and backward (FP32).
//
//   s_ij = scale q_i k_j,  p_ij = exp(s_ij - lse_i),  out_i = sum_j p_ij v_j
//   delta_i = dout_i out_i,  ds_ij = scale p_ij (dout_i v_j - delta_i)
//   dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
//
// Bound by the matrix instructions: 4 head_dim operations a visible pair forward and 14
// backward, each FP32 product six bf16 products of pieces.
//
// Every call first packs its operands (pack_kernel): a tile of 32 rows of one head is
// split into pieces once and stored in the order in which a wave's lanes feed the
// matrix instruction, 1 KiB a fragment and piece, so that the products read whole
// fragments from consecutive addresses whatever the strides, the head's size (padded
// with zeros to 32, 64, 96 or 128) or a sequence's first row.  Two orders are needed:
//   R  what runs along the head's elements (q k, dout v): lane l holds row
//      tile_row(l % 32), elements 16 s + 8 (l / 32) + 0 .. 7 of step s
//   T  what runs along the tile's rows (p v, ds k, p dout, ds q): lane l holds element
//      32 b + tile_row(l % 32) of block b, rows 16 (l / 32) + 8 t + 0 .. 7 of step t
// Forward: each wave has 32 queries and walks over the keys that any of them sees with a
// running maximum and sum.  Backward: one kernel in that form for dq, and one in which
// each wave has 32 keys and walks over the queries (of all heads that share the key
// head) for dk and dv, so nothing is added up in an order that changes.
//
// A NaN or an infinity among a tile's rows would reach every row of a product along
// those rows, times a probability of 0.  T fragments hold zeros in their place, and the
// row's scores are NaN instead (R fragments, or lse in the backward), which the mask
// keeps from rows that do not see it.
#include "mx_attention.hpp"

#include <algorithm>
#include <cmath>
#include <string>

namespace mx {
namespace {

using namespace attn;

constexpr int kThreads = 256, kMaxDim = 128;

struct Shape {
  Sequences seqs;
  int heads, kv_heads, group, dim, tiles;  // tiles: of 32 rows, of all sequences
  Mask mask;
  float scale;
};

struct Strided {
  const float* at;
  int64_t token, head;
};

// Fragments of a tensor: [head][tile][step or block][piece][lane], DP / 16 steps a tile;
// lanes' parts of a tile, and where a head's tile starts.
template <int DP>
constexpr int kTileParts = DP / 16 * 3 * 64;
template <int DP>
__device__ __forceinline__ int64_t tile_at(const Shape& s, int head, int tile) {
  return (int64_t(head) * s.tiles + tile) * kTileParts<DP>;
}
__device__ __forceinline__ Frag3 frag(const bf16x8* tile, int step, int lane) {
  const bf16x8* const f = tile + step * 3 * 64 + lane;
  return {f[0], f[64], f[128]};
}

// ------------------------------------------------------------------ packing
struct PackArgs {
  Shape s;
  Strided q, k, v, dout, out;
  const float* lse;
  bf16x8 *qr, *qt, *kr, *kt, *vr, *vt, *dr, *dt;  // null: not needed
  float *stats;                                     // [head][tile][2][32]: lse log2(e), delta
};

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// A tile's rows into LDS (zeros past the sequence's end and the head's), and per row whether
// all of it is finite.
template <int DP>
struct Stage {
  static constexpr int kPitch = DP + 4;
  float x[kTile][kPitch];
  __device__ __forceinline__ bool load(const Strided& t, int head, int row0, int rows, int dim) {
    constexpr int C = DP / 8;  // a row's elements of each of the 8 threads that share it
    const int r = threadIdx.x >> 3, c = threadIdx.x & 7;
    const float* const src = t.at + (int64_t(row0) + r) * t.token + head * t.head;
    bool ok = true;
#pragma unroll
    for (int i = 0; i < C; i += 4) {
      const int e = i * 8 + c * 4;
      f32x4 v{};
      if (r < rows) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (e + j < dim) v[j] = src[e + j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) ok = ok && finite(v[j]);
      *reinterpret_cast<f32x4*>(&x[r][e]) = v;
    }
    return ok;
  }
  // Fragments of the staged tile; rows whose bit is set in `bad` are NaN in R and 0 in T.
  __device__ __forceinline__ void rows_out(bf16x8* to, uint32_t bad) const {
    const int lane = threadIdx.x & 63, row = tile_row(lane & 31), h = lane >> 5;
    for (int s = threadIdx.x >> 6; s < DP / 16; s += 4) {
      const float* const at = &x[row][s * 16 + h * 8];
      f32x4 a = *reinterpret_cast<const f32x4*>(at), b = *reinterpret_cast<const f32x4*>(at + 4);
      if (bad >> row & 1) a = f32x4{1, 1, 1, 1} * __builtin_nanf(""), b = a;
      put(to, s, lane, split8(a, b));
    }
  }
  __device__ __forceinline__ void cols_out(bf16x8* to, uint32_t bad) const {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    for (int s = threadIdx.x >> 6; s < DP / 16; s += 4) {
      const int e = (s >> 1) * 32 + tile_row(lane & 31), r0 = h * 16 + (s & 1) * 8;
      f32x4 v[2];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j >> 2][j & 3] = bad >> (r0 + j) & 1 ? 0.f : x[r0 + j][e];
      put(to, s, lane, split8(v[0], v[1]));
    }
  }
  static __device__ __forceinline__ void put(bf16x8* to, int s, int lane, const Frag3& f) {
    bf16x8* const at = to + s * 3 * 64 + lane;
    at[0] = f.hi, at[64] = f.mid, at[128] = f.lo;
  }
};

// One bit a row: whether any of the row's 8 threads has `flag`.
__device__ __forceinline__ uint32_t row_bits(bool flag, uint32_t* lds) {
  const uint64_t b = __ballot(flag);
  uint32_t bits = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) bits |= uint32_t((b >> (8 * r) & 0xFF) != 0) << r;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = bits;
  __syncthreads();
  const uint32_t all = lds[0] | lds[1] << 8 | lds[2] << 16 | lds[3] << 24;
  return all;
}

// grid (tiles, heads + kv_heads): a query head's q (and dout, delta, lse), or a key head's k and v.
template <int DP>
__global__ __launch_bounds__(kThreads) void pack_kernel(const PackArgs a) {
  __shared__ Stage<DP> st[2];
  __shared__ uint32_t bits[2][4];
  const Shape& s = a.s;
  SequenceTile t;
  if (!locate<kTile>(s.seqs, blockIdx.x, t) || t.index * kTile >= t.len) return;
  const int row0 = t.start + t.index * kTile, rows = min(kTile, t.len - t.index * kTile);
  const bool key = int(blockIdx.y) >= s.heads;
  const int head = key ? blockIdx.y - s.heads : blockIdx.y;
  const int64_t o = tile_at<DP>(s, head, blockIdx.x);
  if (key) {
    const bool k_ok = st[0].load(a.k, head, row0, rows, s.dim), v_ok = st[1].load(a.v, head, row0, rows, s.dim);
    const uint32_t bad = row_bits(!(k_ok && v_ok), bits[0]);
    if (a.kr) st[0].rows_out(a.kr + o, bad);
    if (a.vr) st[1].rows_out(a.vr + o, bad);
    if (a.kt) st[0].cols_out(a.kt + o, bad);
    if (a.vt) st[1].cols_out(a.vt + o, bad);
    return;
  }
  const uint32_t bad_q = row_bits(!st[0].load(a.q, head, row0, rows, s.dim), bits[0]);
  if (a.qr) st[0].rows_out(a.qr + o, bad_q);
  if (a.qt) st[0].cols_out(a.qt + o, bad_q);
  if (!a.stats) return;
  const uint32_t bad_o = row_bits(!st[1].load(a.dout, head, row0, rows, s.dim), bits[1]);
  if (a.dr) st[1].rows_out(a.dr + o, bad_o);
  if (a.dt) st[1].cols_out(a.dt + o, bad_o);
  // delta, and lse in the exponent's base.  Past the end lse is infinite: no probability.
  const int r = threadIdx.x >> 3, c = threadIdx.x & 7;
  float delta = 0;
  if (r < rows) {
    const float* const out = a.out.at + (int64_t(row0) + r) * a.out.token + head * a.out.head;
    for (int e = c; e < s.dim; e += 8) delta = fmaf(st[1].x[r][e], out[e], delta);
  }
#pragma unroll
  for (int m = 1; m < 8; m <<= 1) delta += __shfl_xor(delta, m, 64);
  if (c == 0) {
    float* const to = a.stats + (int64_t(head) * s.tiles + blockIdx.x) * 64 + r;
    float l = __builtin_inff();
    if (r < rows) l = (bad_q | bad_o) >> r & 1 ? __builtin_nanf("") : a.lse[int64_t(head) * s.seqs.tokens + row0 + r] * kLog2E;
    to[0] = l, to[32] = delta;
  }
}

// ------------------------------------------------------------------ forward
struct FwdArgs {
  Shape s;
  const bf16x8 *qr, *kr, *vt;
  float *out, *lse;
};

template <int DP>
__device__ __forceinline__ void load_frags(Frag3 (&f)[DP / 16], const bf16x8* tile, int lane) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) f[s] = frag(tile, s, lane);
}

// a b along the head's elements: a's fragments from memory, b's in registers.
template <int DP>
__device__ __forceinline__ f32x16 product(const bf16x8* a, const Frag3 (&b)[DP / 16], int lane) {
  f32x16 small{}, large{};
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const Frag3 f = frag(a, s, lane);
    small = mma_small(f, b[s], small);
    large = mma_large(f, b[s], large);
  }
  return large + small;
}

// Block b of a p along the tile's rows: a's T fragments, p's pieces.
__device__ __forceinline__ f32x16 product_rows(const bf16x8* a, int b, const Frag3 (&p)[2], int lane) {
  f32x16 acc{};
  const Frag3 f0 = frag(a, 2 * b, lane), f1 = frag(a, 2 * b + 1, lane);
  acc = mma_small(f0, p[0], acc);
  acc = mma_small(f1, p[1], acc);
  acc = mma_large(f0, p[0], acc);
  return mma_large(f1, p[1], acc);
}

// Stores a lane's 16 elements of block b of one row.
__device__ __forceinline__ void store_block(float* row, const f32x16& v, int b, int h, int dim) {
  const int e0 = b * 32 + h * 16;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (e0 + i < dim) row[e0 + i] = v[i];
}

template <int DP>
__global__ __launch_bounds__(kThreads) void fwd_kernel(const FwdArgs a) {
  const Shape& s = a.s;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int tile = blockIdx.x * 4 + wave, head = blockIdx.y;
  SequenceTile t;
  if (!locate<kTile>(s.seqs, tile, t) || t.index * kTile >= t.len) return;
  const int64_t keys0 = tile_at<DP>(s, head / s.group, t.base);
  Frag3 q[DP / 16];
  load_frags<DP>(q, a.qr + tile_at<DP>(s, head, tile), lane);
  const int i0 = t.index * kTile, i1 = min(i0 + kTile, t.len) - 1, qi = i0 + tile_row(lane & 31);
  const float c = s.scale * kLog2E;
  f32x16 o[DP / 32] = {};
  float m = -__builtin_inff(), l = 0;  // of the exponents
  const KeyTiles keys(s.mask, i0, i1);
  for (int n = 0; n < keys.count; ++n) {
    const int j = keys.tile(n), j0 = j * kTile;
    const int64_t at = keys0 + int64_t(j) * kTileParts<DP>;
    f32x16 x = product<DP>(a.kr + at, q, lane);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= c;
    if (!s.mask.all(i0, i1, j0, j0 + kTile - 1)) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!s.mask.sees(qi, j0 + 16 * h + r)) x[r] = -__builtin_inff();
    }
    float top = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float next = fmaxf(m, top), base = next == -__builtin_inff() ? 0.f : next;
    const float keep = exp2_(m - base);
    float sum = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = exp2_(x[r] - base);
      sum += x[r];
    }
    l = fmaf(l, keep, sum);
    m = next;
    const Frag3 p[2] = {split_half(x, 0), split_half(x, 1)};
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) o[b] = o[b] * keep + product_rows(a.vt + at, b, p, lane);
  }
  l += __shfl_xor(l, 32, 64);
  if (qi >= t.len) return;
  const float r = 1.f / l;
  const int64_t row = t.start + qi;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) store_block(a.out + (row * s.heads + head) * s.dim, o[b] * r, b, h, s.dim);
  if (a.lse && h == 0) a.lse[int64_t(head) * s.seqs.tokens + row] = (m + log2f(l)) * kLn2;
}

// ----------------------------------------------------------------- backward
struct BwdArgs {
  Shape s;
  const bf16x8 *qr, *qt, *kr, *kt, *vr, *dr, *dt;
  const float* stats;
  float *dq, *dk, *dv;
};

template <int DP>
__global__ __launch_bounds__(kThreads) void dq_kernel(const BwdArgs a) {
  const Shape& s = a.s;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int tile = blockIdx.x * 4 + wave, head = blockIdx.y;
  SequenceTile t;
  if (!locate<kTile>(s.seqs, tile, t) || t.index * kTile >= t.len) return;
  const int64_t mine = tile_at<DP>(s, head, tile), keys0 = tile_at<DP>(s, head / s.group, t.base);
  Frag3 q[DP / 16], g[DP / 16];
  load_frags<DP>(q, a.qr + mine, lane);
  load_frags<DP>(g, a.dr + mine, lane);
  const int row = tile_row(lane & 31);
  const float* const st = a.stats + (int64_t(head) * s.tiles + tile) * 64 + row;
  const float lse = st[0], delta = st[32], c = s.scale * kLog2E;
  const int i0 = t.index * kTile, i1 = min(i0 + kTile, t.len) - 1, qi = i0 + row;
  f32x16 dq[DP / 32] = {};
  const KeyTiles keys(s.mask, i0, i1);
  for (int n = 0; n < keys.count; ++n) {
    const int j = keys.tile(n), j0 = j * kTile;
    const int64_t o = keys0 + int64_t(j) * kTileParts<DP>;
    f32x16 x = product<DP>(a.kr + o, q, lane);
    const f32x16 dp = product<DP>(a.vr + o, g, lane);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = exp2_(fmaf(x[r], c, -lse)) * (dp[r] - delta);
    if (!s.mask.all(i0, i1, j0, j0 + kTile - 1)) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!s.mask.sees(qi, j0 + 16 * h + r)) x[r] = 0;
    }
    const Frag3 p[2] = {split_half(x, 0), split_half(x, 1)};
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) dq[b] += product_rows(a.kt + o, b, p, lane);
  }
  if (qi >= t.len) return;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
    store_block(a.dq + ((t.start + qi) * int64_t(s.heads) + head) * s.dim, dq[b] * s.scale, b, h, s.dim);
}

template <int DP>
__global__ __launch_bounds__(kThreads) void dkv_kernel(const BwdArgs a) {
  const Shape& s = a.s;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int tile = blockIdx.x * 4 + wave, kv_head = blockIdx.y;
  SequenceTile t;
  if (!locate<kTile>(s.seqs, tile, t) || t.index * kTile >= t.len) return;
  const int64_t mine = tile_at<DP>(s, kv_head, tile);
  Frag3 k[DP / 16], v[DP / 16];
  load_frags<DP>(k, a.kr + mine, lane);
  load_frags<DP>(v, a.vr + mine, lane);
  const int j0 = t.index * kTile, j1 = j0 + kTile - 1, kj = j0 + tile_row(lane & 31);
  const float c = s.scale * kLog2E;
  // The last query that sees any of these keys.
  const int last = s.mask.window && j0 >= s.mask.sinks ? min(t.len - 1, j1 + min(s.mask.window, t.len) - 1) : t.len - 1;
  f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
  for (int head = kv_head * s.group; head < (kv_head + 1) * s.group; ++head) {
    for (int i = t.index; i <= last / kTile; ++i) {
      const int64_t o = tile_at<DP>(s, head, t.base + i);
      const float* const st = a.stats + (int64_t(head) * s.tiles + t.base + i) * 64 + 16 * h;
      f32x16 x = product<DP>(a.qr + o, k, lane);
      f32x16 dp = product<DP>(a.dr + o, v, lane);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[r] = exp2_(fmaf(x[r], c, -st[r]));
        dp[r] = x[r] * (dp[r] - st[32 + r]);
      }
      const int i0 = i * kTile;
      if (!s.mask.all(i0, i0 + kTile - 1, j0, j1)) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!s.mask.sees(i0 + 16 * h + r, kj)) x[r] = 0, dp[r] = 0;
      }
      const Frag3 p[2] = {split_half(x, 0), split_half(x, 1)}, ds[2] = {split_half(dp, 0), split_half(dp, 1)};
#pragma unroll
      for (int b = 0; b < DP / 32; ++b) {
        dv[b] += product_rows(a.dt + o, b, p, lane);
        dk[b] += product_rows(a.qt + o, b, ds, lane);
      }
    }
  }
  if (kj >= t.len) return;
  const int64_t row = ((t.start + kj) * int64_t(s.kv_heads) + kv_head) * s.dim;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) {
    if (a.dk) store_block(a.dk + row, dk[b] * s.scale, b, h, s.dim);
    if (a.dv) store_block(a.dv + row, dv[b], b, h, s.dim);
  }
}

// --------------------------------------------------------------------- host
int check(const char* who, const mx_attention_desc* d) {
  MX_REQUIRE(d, MX_ERR_INVALID, who, ": null descriptor");
  MX_REQUIRE(d->tokens >= 0 && d->sequences >= 0 && d->heads >= 0 && d->kv_heads >= 0, MX_ERR_INVALID, who,
             ": negative size");
  MX_REQUIRE(d->head_dim >= 1 && d->head_dim <= kMaxDim, MX_ERR_INVALID, who, ": head_dim must be 1 to ", kMaxDim, ", got ",
             d->head_dim);
  MX_REQUIRE(d->heads == 0 || (d->kv_heads > 0 && d->heads % d->kv_heads == 0), MX_ERR_INVALID, who, ": ", d->heads,
             " heads do not share ", d->kv_heads, " key heads evenly");
  MX_REQUIRE(d->tokens <= (1 << 30) && d->sequences <= (1 << 24) && d->heads + d->kv_heads <= 65535, MX_ERR_INVALID, who,
             ": size out of range");
  MX_REQUIRE(d->tokens == 0 || d->sequences > 0, MX_ERR_INVALID, who, ": tokens of no sequence");
  MX_REQUIRE(d->starts || d->sequences == 0 || d->tokens % d->sequences == 0, MX_ERR_INVALID, who, ": ", d->tokens,
             " tokens do not divide into ", d->sequences, " sequences");
  MX_REQUIRE(d->window >= 0 && d->sinks >= 0, MX_ERR_INVALID, who, ": negative window or sinks");
  MX_REQUIRE(std::isfinite(d->scale), MX_ERR_INVALID, who, ": the scale must be finite");
  return MX_OK;
}

Shape shape_of(const mx_attention_desc* d) {
  Shape s{};
  s.seqs = {d->starts, int(d->tokens), int(d->sequences)};
  s.heads = int(d->heads), s.kv_heads = int(d->kv_heads), s.group = int(d->heads / d->kv_heads), s.dim = int(d->head_dim);
  s.tiles = int(sequence_tiles(d->tokens, d->sequences, kTile));
  s.mask = {int(std::min<int64_t>(d->window, 1 << 30)), int(std::min<int64_t>(d->sinks, 1 << 30))};
  s.scale = float(d->scale);
  return s;
}

int padded(int64_t dim) { return int((dim + 31) / 32 * 32); }

// Scratch: the packed tensors in the order in which take() hands them out.
struct Carve {
  char* at;
  int64_t used = 0;
  template <class T>
  T* take(int64_t bytes) {
    T* const p = at ? reinterpret_cast<T*>(at + used) : nullptr;
    used += bytes;
    return p;
  }
};

struct Buffers {
  bf16x8 *qr, *qt, *kr, *kt, *vr, *vt, *dr, *dt;
  float* stats;
};
Buffers carve(const Shape& s, bool backward, Carve& c) {
  const int64_t tile = padded(s.dim) / 16 * 3 * 1024, q = tile * s.tiles * s.heads, k = tile * s.tiles * s.kv_heads;
  Buffers b{};
  b.qr = c.take<bf16x8>(q);
  b.kr = c.take<bf16x8>(k);
  if (!backward) {
    b.vt = c.take<bf16x8>(k);
    return b;
  }
  b.qt = c.take<bf16x8>(q);
  b.dr = c.take<bf16x8>(q);
  b.dt = c.take<bf16x8>(q);
  b.kt = c.take<bf16x8>(k);
  b.vr = c.take<bf16x8>(k);
  b.stats = c.take<float>(int64_t(s.heads) * s.tiles * 256);
  return b;
}

int64_t workspace_bytes_of(const mx_attention_desc* d, bool backward) {
  if (d->tokens == 0 || d->heads == 0) return 0;
  Carve c{nullptr};
  carve(shape_of(d), backward, c);
  return c.used;
}

template <class F>
void with_dim(int dim, F&& f) {
  switch (padded(dim)) {
    case 32: return f(std::integral_constant<int, 32>{});
    case 64: return f(std::integral_constant<int, 64>{});
    case 96: return f(std::integral_constant<int, 96>{});
    default: return f(std::integral_constant<int, 128>{});
  }
}

}  // namespace
}  // namespace mx

using namespace mx;

extern "C" int mx_attention_workspace(const mx_attention_desc* d, int backward, int64_t* bytes) {
  MX_ABI_BEGIN
  MX_TRY(check("mx_attention_workspace", d));
  MX_REQUIRE(bytes, MX_ERR_INVALID, "mx_attention_workspace: null result");
  *bytes = workspace_bytes_of(d, backward != 0);
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_attention_forward(const mx_attention_desc* d, const float* q, const float* k, const float* v, float* out,
                                    float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  const char* const who = "mx_attention_forward";
  MX_TRY(check(who, d));
  if (d->tokens == 0 || d->heads == 0) return MX_OK;
  MX_REQUIRE(q && k && v && out, MX_ERR_INVALID, who, ": null buffer");
  const Shape s = shape_of(d);
  hipStream_t st = resolve_stream(stream);
  Workspace ws;
  MX_TRY(ws.take(who, workspace, workspace_bytes, workspace_bytes_of(d, false), st));
  Carve c{ws.as<char>()};
  const Buffers b = carve(s, false, c);
  PackArgs p{};
  p.s = s;
  p.q = {q, d->q_token, d->q_head}, p.k = {k, d->k_token, d->k_head}, p.v = {v, d->v_token, d->v_head};
  p.qr = b.qr, p.kr = b.kr, p.vt = b.vt;
  const FwdArgs f{s, b.qr, b.kr, b.vt, out, lse};
  with_dim(s.dim, [&](auto dp) {
    hipLaunchKernelGGL((pack_kernel<decltype(dp)::value>), dim3(s.tiles, s.heads + s.kv_heads), dim3(kThreads), 0, st, p);
  });
  MX_LAUNCHED();
  with_dim(s.dim, [&](auto dp) {
    hipLaunchKernelGGL((fwd_kernel<decltype(dp)::value>), dim3((s.tiles + 3) / 4, s.heads), dim3(kThreads), 0, st, f);
  });
  MX_LAUNCHED();
  return MX_OK;
  MX_ABI_END
}

extern "C" int mx_attention_backward(const mx_attention_desc* d, const float* dout, const float* q, const float* k,
                                     const float* v, const float* out, const float* lse, float* dq, float* dk, float* dv,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  MX_ABI_BEGIN
  const CountedCall counted;
  const char* const who = "mx_attention_backward";
  MX_TRY(check(who, d));
  if (d->tokens == 0 || d->heads == 0 || (!dq && !dk && !dv)) return MX_OK;
  MX_REQUIRE(dout && q && k && v && out && lse, MX_ERR_INVALID, who, ": null buffer");
  const Shape s = shape_of(d);
  hipStream_t st = resolve_stream(stream);
  Workspace ws;
  MX_TRY(ws.take(who, workspace, workspace_bytes, workspace_bytes_of(d, true), st));
  Carve c{ws.as<char>()};
  const Buffers b = carve(s, true, c);
  PackArgs p{};
  p.s = s;
  p.q = {q, d->q_token, d->q_head}, p.k = {k, d->k_token, d->k_head}, p.v = {v, d->v_token, d->v_head};
  p.dout = {dout, d->heads * d->head_dim, d->head_dim}, p.out = {out, d->heads * d->head_dim, d->head_dim};
  p.lse = lse;
  p.qr = b.qr, p.kr = b.kr, p.vr = b.vr, p.dr = b.dr;
  if (dk || dv) p.qt = b.qt, p.dt = b.dt;
  if (dq) p.kt = b.kt;
  p.stats = b.stats;
  const BwdArgs g{s, b.qr, b.qt, b.kr, b.kt, b.vr, b.dr, b.dt, b.stats, dq, dk, dv};
  with_dim(s.dim, [&](auto dp) {
    hipLaunchKernelGGL((pack_kernel<decltype(dp)::value>), dim3(s.tiles, s.heads + s.kv_heads), dim3(kThreads), 0, st, p);
  });
  MX_LAUNCHED();
  if (dq) {
    with_dim(s.dim, [&](auto dp) {
      hipLaunchKernelGGL((dq_kernel<decltype(dp)::value>), dim3((s.tiles + 3) / 4, s.heads), dim3(kThreads), 0, st, g);
    });
    MX_LAUNCHED();
  }
  if (dk || dv) {
    with_dim(s.dim, [&](auto dp) {
      hipLaunchKernelGGL((dkv_kernel<decltype(dp)::value>), dim3((s.tiles + 3) / 4, s.kv_heads), dim3(kThreads), 0, st, g);
    });
    MX_LAUNCHED();
  }
  return MX_OK;
  MX_ABI_END
}
