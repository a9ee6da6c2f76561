// Causal attention of packed sequences, forward and backward (FP32).
//
//   s_ij = scale q_i k_j,  p_ij = exp(s_ij - lse_i),  out_i = sum_j p_ij v_j
//   delta_i = dout_i out_i,  ds_ij = scale p_ij (dout_i v_j - delta_i)
//   dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
//
// Bound by the matrix instructions: 4 head_dim operations a visible pair forward and 14
// backward, each FP32 product six bf16 products of pieces.
//
// Every call first packs what is read many times (pack_kernel): a tile of 32 rows of one
// head is split into pieces once and stored in the order in which a wave's lanes feed the
// matrix instruction, 1 KiB a fragment and piece, whatever the strides, the head's size
// (padded with zeros to 32, 64, 96 or 128) or a sequence's first row: lane l holds row
// tile_row(l % 32), elements 16 s + 8 (l / 32) + 0 .. 7 of step s.  So tiles go from memory
// to LDS in whole lines without passing through registers, for all four waves of a
// workgroup, one tile ahead of the products; what runs along the head's elements (q k,
// dout v) takes fragments as they lie, and what runs along the tile's rows (p v, ds k, p
// dout, ds q) through transposing reads.
// Forward: each wave has 32 queries and walks over the keys that any of its workgroup's
// sees, with a running maximum and sum.  Backward: one kernel in that form for dq, and
// one in which each wave has 32 keys and walks over the queries (of all heads that share
// the key head) for dk and dv, so nothing is added up in an order that changes.
//
// A NaN or an infinity among a tile's rows would reach every row of a product along
// those rows, times a probability of 0.  Such rows are packed as zeros, and what sees
// them is made NaN through the scores, which the mask keeps apart: by a NaN in the key's
// other operand in the forward, by lse (the forward's, or its own) in the backward.
#include "mx_attention.hpp"

#include <algorithm>
#include <cmath>
#include <string>

namespace mx {
namespace {

using namespace attn;

constexpr int kThreads = 256, kMaxDim = 128;

// Kernels take a head's elements in steps of 16 (E) where products run along them, and in blocks of 32 where
// they are the products' columns, as tiles hold them (12 heads of 80 in steps of 96: gradients of 5006 tokens 311 us,
// of 80 292).
constexpr int blocked(int e) { return (e + 31) / 32 * 32; }

struct Shape {
  Sequences seqs;
  int heads, kv_heads, group, dim, tiles;  // tiles: of 32 rows, of all sequences
  Mask mask;
  float scale;
};

// Where a head's tile of a packed tensor [head][tile] starts.
template <int DP>
__device__ __forceinline__ int64_t tile_at(const Shape& s, int head, int tile) {
  return (int64_t(head) * s.tiles + tile) * kTileBytes<DP>;
}
// ------------------------------------------------------------------ packing
struct PackArgs {
  Shape s;
  Strided q, k, v, dout, out;
  const float* lse;
  char *qp, *kp, *vp, *dp;  // kp, vp: by key head; qp, dp: by head, null in the forward
  float* stats;             // [head][tile][2][32]: lse log2(e), delta
};

// One bit a row, from its two lanes (l and l + 32) in a wave that has all rows.
__device__ __forceinline__ uint32_t row_bits(bool flag) {
  const uint64_t b = __ballot(flag);
  return uint32_t(b) | uint32_t(b >> 32);
}

// A tile of one head, straight from memory to fragments: a wave takes every fourth step, so
// the rows that are not finite are known to the workgroup before anything is stored.
template <int DP>
struct Pack {
  static constexpr int N = (DP / 16 + 3) / 4;
  f32x4 x[N][2];
  bool bad = false;
  // rows: of the tile; r and h: the lane's row and half.  (What is packed is looked at, so scaled.)
  __device__ __forceinline__ void load(const Strided& t, int head, int row0, int rows, int dim, int wave, int r, int h, float scale) {
    const float* const row = t.at + (int64_t(row0) + r) * t.token + head * t.head;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = wave + 4 * i;
      x[i][0] = x[i][1] = f32x4{};
      if (s < DP / 16 && r < rows) load8(row, s * 16 + h * 8, dim, x[i]);
      x[i][0] *= scale, x[i][1] *= scale;
#pragma unroll
      for (int j = 0; j < 8; ++j) bad = bad || !finite(x[i][j >> 2][j & 3]);
    }
  }
  __device__ __forceinline__ void store(char* to, int wave, int lane, bool replace, float with) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = wave + 4 * i;
      if (s >= DP / 16) break;
      f32x4 v[2] = {x[i][0], x[i][1]};
      if (replace) v[0] = v[1] = f32x4{with, with, with, with};
      const Frag3 f = split8(v[0], v[1]);
      bf16x8* const at = reinterpret_cast<bf16x8*>(to) + s * 3 * 64 + slot(lane);
      at[0] = f.hi, at[64] = f.mid, at[128] = f.lo;
    }
  }
};

// grid (tiles, heads + kv_heads, or kv_heads alone): a key head's k and v, or a query head's q, dout,
// lse and delta.
// Bound by memory: 4 bytes read and 6 written an element (45 us for q, dout, out, k and v of 2 x 2048
// tokens, 16 and 4 heads of 128: 4.9 TB/s).
template <int DP>
__global__ __launch_bounds__(kThreads) void pack_kernel(const PackArgs a) {
  __shared__ uint32_t bits[2][4];
  __shared__ float sums[4][kTile];
  const Shape& s = a.s;
  SequenceTile t;
  if (!locate<kTile>(s.seqs, blockIdx.x, t) || t.index * kTile >= t.len) return;
  const int row0 = t.start + t.index * kTile, rows = min(kTile, t.len - t.index * kTile);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int r = tile_row(lane & 31);
  const bool key = int(blockIdx.y) < s.kv_heads;
  const int head = key ? blockIdx.y : blockIdx.y - s.kv_heads;
  const int64_t o = tile_at<DP>(s, head, blockIdx.x);
  Pack<DP> x, y;
  x.load(key ? a.k : a.q, head, row0, rows, s.dim, wave, r, h, key ? 1.f : s.scale * kLog2E);
  y.load(key ? a.v : a.dout, head, row0, rows, s.dim, wave, r, h, 1.f);
  const uint32_t bx = row_bits(x.bad), by = row_bits(y.bad);
  if (lane == 0) bits[0][wave] = bx, bits[1][wave] = by;
  if (!key) {
    // A row's part of delta in this wave's steps.
    float delta = 0;
    const float* const out = a.out.at + (int64_t(row0) + r) * a.out.token + head * a.out.head;
#pragma unroll
    for (int i = 0; i < Pack<DP>::N; ++i) {
      f32x4 v[2] = {};
      if (wave + 4 * i < DP / 16 && r < rows) load8(out, (wave + 4 * i) * 16 + h * 8, s.dim, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf(y.x[i][j >> 2][j & 3], v[j >> 2][j & 3], delta);
    }
    delta += __shfl_xor(delta, 32, 64);
    if (h == 0) sums[wave][r] = delta;
  }
  __syncthreads();
  const uint32_t bad_x = bits[0][0] | bits[0][1] | bits[0][2] | bits[0][3];
  const uint32_t bad_y = bits[1][0] | bits[1][1] | bits[1][2] | bits[1][3];
  const bool bad = (bad_x | bad_y) >> (lane & 31) & 1;
  if (key) {
    x.store(a.kp + o, wave, lane, bad, a.stats ? 0.f : __builtin_nanf(""));
    y.store(a.vp + o, wave, lane, bad, 0.f);
    return;
  }
  x.store(a.qp + o, wave, lane, bad, 0.f);
  y.store(a.dp + o, wave, lane, bad, 0.f);
  // Past the sequence's end lse is infinite: no probability.
  if (wave == 0 && h == 0) {
    float* const to = a.stats + (int64_t(head) * s.tiles + blockIdx.x) * 64 + r;
    float l = __builtin_inff();
    if (r < rows) l = bad ? __builtin_nanf("") : a.lse[int64_t(head) * s.seqs.tokens + row0 + r] * kLog2E;
    to[0] = l, to[32] = r < rows ? sums[0][r] + sums[1][r] + sums[2][r] + sums[3][r] : 0.f;
  }
}

// Own rows from a packed tile.
template <int N>
__device__ __forceinline__ void own_rows(Frag3 (&f)[N], const char* tile, int lane) {
  const bf16x8* const at = reinterpret_cast<const bf16x8*>(tile) + slot(lane);
#pragma unroll
  for (int s = 0; s < N; ++s) f[s] = {at[s * 192], at[s * 192 + 64], at[s * 192 + 128]};
}

// Blocks of 128 rows, four tiles of one sequence; the workgroups' order puts what has the most
// to do first and keeps a head's on as few XCDs as there are heads for.
constexpr int kBlock = 4 * kTile;

// A block of a wave's sums in LDS.
__device__ __forceinline__ void put_block(uint32_t at, int b, const f32x16& v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) *pieces::lds_at<f32x4>(at + b * 4096 + i * 1024) = f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
}
__device__ __forceinline__ f32x16 get_block(uint32_t at, int b) {
  f32x16 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 x = *pieces::lds_at<const f32x4>(at + b * 4096 + i * 1024);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[4 * i + e] = x[e];
  }
  return v;
}

// A workgroup's walk over tiles of two tensors, SPLIT of them at a time: of its four (or more) waves each
// SPLIT share their rows, and take every SPLIT-th tile.  Both tensors' next tiles are loaded while these are
// in use; where two stages of both do not fit LDS (kSingle), the second's are in one, and loaded
// between its last use and the next step's first.
struct Source {
  const char *first, *second, *stats;
};
struct Staged {
  uint32_t first, second, stats;
};
struct Halves {
  Frag3 of[2];
};
template <int DP, int WAVES, int SPLIT, int STATS>
struct Walk {
  using St = Stages<DP, 3, WAVES, STATS>;
  static constexpr bool kSingle = SPLIT > 1 && DP == 128;
  static constexpr int kTensor = kTileBytes<DP>, kSlot = kSingle ? St::kBytes - kTensor : St::kBytes;
  static constexpr int kGroups = WAVES / SPLIT, kRows = kGroups * kTile, kBytes = SPLIT * (2 * kSlot + (kSingle ? kTensor : 0));
  St st;
  int wave, lane, count;
  __device__ __forceinline__ int rows() const { return wave % kGroups * kTile; }
  __device__ __forceinline__ int turn() const { return wave / kGroups; }
  // Where step n's tile of that turn lies.
  __device__ __forceinline__ Staged at(int n, int turn) const {
    const uint32_t first = st.lds + ((n & 1) * SPLIT + turn) * kSlot;
    if (kSingle) return {first, st.lds + 2 * SPLIT * kSlot + turn * kTensor, first + kTensor};
    return {first, first + kTensor, first + 2 * kTensor};
  }
  // load(tile, its place) for each of step n's
  template <class F>
  __device__ __forceinline__ void fetch(int n, F&& load) const {
#pragma unroll
    for (int u = 0; u < SPLIT; ++u)
      if (n * SPLIT + u < count) load(n * SPLIT + u, at(n, u));
  }
  // Both tensors' of step n from source(tile), the second's later where it is staged once.
  template <class F>
  __device__ __forceinline__ void fetch_both(int n, F&& source) const {
    fetch(n, [&](int tile, const Staged& to) {
      const Source s = source(tile);
      if constexpr (kSingle) {
        St::load_one(to.first, s.first, wave, lane);
        St::load_stats(to.stats, s.stats, wave, lane);
      } else {
        const St slot{to.first};
        slot.load(0, s.first, s.second, s.stats, wave, lane);
      }
    });
  }
  template <class F>
  __device__ __forceinline__ void fetch_second(int n, F&& source) const {
    fetch(n, [&](int tile, const Staged& to) { St::load_one(to.second, source(tile).second, wave, lane); });
  }
  template <class F>
  __device__ __forceinline__ void start(F&& source) const {
    fetch_both(0, source);
    if constexpr (kSingle) fetch_second(0, source);
  }
  // use(tile, at), then finish(at, what that gave), which does not read the second tensor, for each of the
  // wave's tiles that it sees.
  template <class F, class S, class U, class V>
  __device__ __forceinline__ void run(F&& source, S&& seen, U&& use, V&& finish) const {
    for (int n = 0; n * SPLIT < count; ++n) {
      pieces::wait_loads<0>();
      pieces::barrier();
      fetch_both(n + 1, source);
      const int mine = n * SPLIT + turn();
      const Staged here = at(n, turn());
      if constexpr (kSingle) {
        const bool on = mine < count && seen(mine);
        std::remove_const_t<decltype(use(mine, here))> x;
        if (on) x = use(mine, here);
        pieces::barrier();
        fetch_second(n + 1, source);
        if (on) finish(here, x);
      } else {
        if ((SPLIT > 1 && mine >= count) || !seen(mine)) continue;
        auto x = use(mine, here);
        finish(here, x);
      }
    }
  }
  // Behind the walk: adds what the waves that share rows have (BLOCKS blocks) to the first one's,
  // through LDS.  False in the others.
  template <int BLOCKS, class F>
  __device__ __forceinline__ bool join(F&& block) const {
    if constexpr (SPLIT > 1) {
      static_assert(SPLIT <= 2 && BLOCKS * 4096 * kGroups <= kBytes);
      const uint32_t at = st.lds + wave % kGroups * (BLOCKS * 4096) + lane * 16;
      __syncthreads();
      if (turn())
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) put_block(at, b, block(b));
      __syncthreads();
      if (turn()) return false;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) block(b) += get_block(at, b);
    }
    return true;
  }
};
// ------------------------------------------------------------------ forward
struct FwdArgs {
  Shape s;
  Strided q;
  const char *kp, *vp;
  float *out, *lse;
};

// Steps whose queries' smallest piece waits in LDS, where two waves a SIMD have no registers for it.
constexpr int aside(int steps, int waves) { return steps > 6 && waves == 8 ? 7 : 0; }

// A wave's 32 queries stay in registers as pieces, with their sums.  Bound by the matrix
// instructions: 16384 tokens, 16 heads of 64, window 4096 1290 us, 187 TFLOP/s, six piece products of which
// are 1.12 PFLOP/s (a library's bf16 product of 8192^3 1.25 to 1.33); 2 x 2048, 16 heads of 128 207 us,
// 166 TFLOP/s.  There a wave is alone on its SIMD, which hides neither LDS's latency nor the softmax
// behind products unless those are another tile's: 250 us with a tile's scores and exponents in turn.
// Workgroups of eight waves, two a SIMD (4.5 us a tile of 256 rows for 3.7 of 128 then), have too
// uneven work (289 us).
template <int E, int WAVES, int SPLIT>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(SPLIT == 1 && (WAVES == 8 || E <= 96) ? 2 : 1))) void fwd_kernel(const FwdArgs a) {
  constexpr int DP = blocked(E);
  using W = Walk<DP, WAVES, SPLIT, 0>;
  constexpr int kRows = W::kRows;
  constexpr int kAside = aside(E / 16, WAVES);
  __shared__ __attribute__((aligned(1024))) char smem[W::kBytes + kAside * WAVES * 1024];
  const Shape& s = a.s;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int head = blockIdx.x % s.heads, block = gridDim.x / s.heads - 1 - blockIdx.x / s.heads;
  SequenceTile t;
  if (!locate<kRows>(s.seqs, block, t) || t.index * kRows >= t.len) return;
  const int64_t keys0 = tile_at<DP>(s, head / s.group, t.start / kTile + t.seq);
  const int b0 = t.index * kRows;
  const KeyTiles<> keys(s.mask, b0, min(b0 + kRows, t.len) - 1);
  const W walk{{lds_address(smem)}, wave, lane, keys.count};
  // Waves alone on their SIMD take the next tile's scores between this one's exponents, keys a step
  // ahead of values, unless one of them is staged once (the keys, which are done with first).
  constexpr bool kAhead = !W::kSingle && (SPLIT > 1 || (DP == 128 && WAVES == 4));
  const auto source = [&](int n) {
    const int64_t at = keys0 + int64_t(keys.tile(n)) * kTileBytes<DP>;
    return W::kSingle ? Source{a.vp + at, a.kp + at} : Source{a.kp + at, a.vp + at};
  };
  walk.start(source);
  const int i0 = b0 + walk.rows(), i1 = min(i0 + kTile, t.len) - 1, qi = i0 + tile_row(lane & 31);
  Frag3 q[E / 16];
  own_rows(q, a.q, head, int64_t(t.start) + qi, qi < t.len, s.dim, h, s.scale * kLog2E);
  bf16x8* const mine = reinterpret_cast<bf16x8*>(smem + W::kBytes) + wave * kAside * 64 + lane;
#pragma unroll
  for (int i = 0; i < kAside; ++i) mine[i * 64] = q[i].lo;
  const auto low = [&](int i) { return i < kAside ? mine[i * 64] : q[i].lo; };
  f32x16 o[DP / 32] = {};
  float m = -__builtin_inff(), l = 0;  // of the exponents
  const uint32_t columns = column_base(lane);
  const auto seen = [&](int n) {
    const int j0 = keys.tile(n) * kTile;
    return i0 < t.len && !s.mask.none(i0, i1, j0, j0 + kTile - 1);
  };
  const auto scores = [&](uint32_t tile) { return product<3>(tile, q, lane, low); };
  const auto masked = [&](int n, f32x16& x) {
    const int j0 = keys.tile(n) * kTile;
    if (!s.mask.all(i0, i1, j0, j0 + kTile - 1)) hide(x, [&](int r) { return s.mask.sees(qi, j0 + 16 * h + r); });
  };
  const auto add = [&](f32x16& x, uint32_t values) {
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
    for (int b = 0; b < DP / 32; ++b) {
      if (WAVES == 8 && DP > 96) __builtin_amdgcn_sched_barrier(0);  // one block's fragments at a time
      o[b] = o[b] * keep + product_columns(values + columns, b, p);
    }
  };
  if constexpr (kAhead) {
    pieces::wait_loads<0>();
    pieces::barrier();
    const auto load_keys = [&](int n, const Staged& to) { W::St::load_one(to.first, source(n).first, wave, lane); };
    walk.fetch(1, load_keys);
    f32x16 x{};
    const auto at = [&](int n) { return walk.at(n, walk.turn()); };
    bool live = walk.turn() < keys.count && seen(walk.turn());
    if (live) x = scores(at(0).first), masked(walk.turn(), x);
    for (int n = 0; n * SPLIT < keys.count; ++n) {
      pieces::wait_loads<0>();
      pieces::barrier();
      walk.fetch(n + 2, load_keys);
      walk.fetch_second(n + 1, source);
      const int ahead = (n + 1) * SPLIT + walk.turn();
      const bool next = ahead < keys.count && seen(ahead);
      f32x16 y;
      if (live) {
        // (what lies there where no tile is left is not looked at)
        y = scores(at(n + 1).first);
        add(x, at(n).second);
      } else {
        asm volatile("");
        y = scores(at(n + 1).first);
      }
      if (next) masked(ahead, y);
      x = y, live = next;
    }
  } else {
    const auto use = [&](int n, const Staged& at) {
      f32x16 x = scores(W::kSingle ? at.second : at.first);
      masked(n, x);
      return x;
    };
    walk.run(source, seen, use, [&](const Staged& at, f32x16& x) { add(x, W::kSingle ? at.first : at.second); });
  }
  if constexpr (SPLIT > 1) {
    // To the larger of both maxima, then the sums (l among them).
    float* const top = reinterpret_cast<float*>(smem) + wave * 64 + lane;
    __syncthreads();
    *top = m;
    __syncthreads();
    const float next = fmaxf(m, top[(walk.turn() ? -1 : 1) * W::kGroups * 64]), keep = exp2_(m - (next == -__builtin_inff() ? 0.f : next));
    f32x16 sum{};
    sum[0] = l * keep, m = next;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) o[b] *= keep;
    if (!walk.template join<DP / 32 + 1>([&](int b) -> f32x16& { return b == DP / 32 ? sum : o[b]; })) return;
    l = sum[0];
  }
  l += __shfl_xor(l, 32, 64);
  if (qi >= t.len) return;
  const float r = 1.f / l;
  const int64_t row = int64_t(t.start) + qi;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) store_block(a.out + (row * s.heads + head) * s.dim, o[b] * r, b, h, s.dim);
  if (a.lse && h == 0) a.lse[int64_t(head) * s.seqs.tokens + row] = (m + log2f(l)) * kLn2;
}

// ----------------------------------------------------------------- backward
struct BwdArgs {
  Shape s;
  const char *qp, *kp, *vp, *dp;
  const float* stats;
  float *dq, *dk, *dv;
  int parts;            // of a key head's query heads
  float *dk_p, *dv_p;  // [part][token][key head][dim] where there are several
  int block;             // of keys, 128 or 64
  int near, far_blocks;  // workgroups' blocks of keys, and of those that are seen past the window
  float* far;            // [chunk][block][key head][part][dk, dv][key of the block][dim]
};

// First tokens that stay visible are seen by every later query, other keys by a window's.
// So that their workgroup is not the last by far, the queries past the window of its block are
// dealt to workgroups of their own, chunks of 512 rows of a sequence, which start first and whose sums
// far_kernel adds in order (8 sequences of up to 2048, window 512, 4 first tokens, 12 heads of 80: a call
// for dk and dv 217 us, 286 with chunks of 1024 rows that start last; the kernel alone took 270 with those
// queries in the block's own workgroup, 243 with such chunks).
constexpr int kChunk = 512, kFarBlocks = 4;
__device__ __forceinline__ float* far_at(const BwdArgs& a, int chunk, int block, int kv_head, int part) {
  return a.far + (((int64_t(chunk) * a.far_blocks + block) * a.s.kv_heads + kv_head) * a.parts + part) * (2 * a.block * a.s.dim);
}
// The last row that the workgroup of the block at b0 takes: of its keys' window, or of the sequence
// where no other workgroup has what lies past it.
__device__ __forceinline__ int near_last(const BwdArgs& a, int b0, int len) {
  const Mask& m = a.s.mask;
  const bool all = m.window == 0 || (b0 < m.sinks && b0 >= a.far_blocks * a.block);
  return all ? len - 1 : min(len - 1, b0 + a.block - 1 + min(m.window, len) - 1);
}

// Three products of a tile, two of them computed again for dk and dv: the scores' gradients would be
// 4 bytes a pair in memory, written and read.  2 x 2048, 16 heads of 128: 280 us alone, 168 TFLOP/s, 1.0 PFLOP/s of pieces.
// (workgroup `index` of `count`)
template <int E, int SPLIT>
struct Dq {
  static constexpr int DP = blocked(E);
  using W = Walk<DP, 4, SPLIT, 0>;
  static constexpr int kBytes = W::kBytes;
  static __device__ void run(const BwdArgs a, char* smem, int index, int count);
};
template <int E, int SPLIT>
__device__ __forceinline__ void Dq<E, SPLIT>::run(const BwdArgs a, char* smem, int index, int count) {
  constexpr int kRows = W::kRows;
  const Shape& s = a.s;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int head = index % s.heads, block = count / s.heads - 1 - index / s.heads;
  SequenceTile t;
  if (!locate<kRows>(s.seqs, block, t) || t.index * kRows >= t.len) return;
  const int base32 = t.start / kTile + t.seq;
  const int64_t keys0 = tile_at<DP>(s, head / s.group, base32);
  const int b0 = t.index * kRows;
  const KeyTiles<> keys(s.mask, b0, min(b0 + kRows, t.len) - 1);
  const W walk{{lds_address(smem)}, wave, lane, keys.count};
  const auto source = [&](int n) {
    const int64_t at = keys0 + int64_t(keys.tile(n)) * kTileBytes<DP>;
    return Source{a.kp + at, a.vp + at};
  };
  walk.start(source);
  const int i0 = b0 + walk.rows(), i1 = min(i0 + kTile, t.len) - 1, row = tile_row(lane & 31), qi = i0 + row;
  // A wave past the sequence's end repeats its last tile, and stores nothing.
  const int mine = base32 + min(i0, t.len - 1) / kTile;
  Frag3 q[E / 16], g[E / 16];
  own_rows(q, a.qp + tile_at<DP>(s, head, mine), lane);
  own_rows(g, a.dp + tile_at<DP>(s, head, mine), lane);
  const float* const stat = a.stats + (int64_t(head) * s.tiles + mine) * 64 + row;
  const float lse = stat[0], delta = stat[32];
  f32x16 dq[DP / 32] = {};
  const uint32_t columns = column_base(lane);
  const auto seen = [&](int n) {
    const int j0 = keys.tile(n) * kTile;
    return i0 < t.len && !s.mask.none(i0, i1, j0, j0 + kTile - 1);
  };
  const auto use = [&](int n, const Staged& at) {
    const int j0 = keys.tile(n) * kTile;
    f32x16 x = product<3>(at.first, q, lane) - lse;
    if (!s.mask.all(i0, i1, j0, j0 + kTile - 1)) hide(x, [&](int r) { return s.mask.sees(qi, j0 + 16 * h + r); });
    const f32x16 dp = product<3>(at.second, g, lane);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = times(exp2_(x[r]), dp[r] - delta);
    return Halves{{split_half(x, 0), split_half(x, 1)}};
  };
  walk.run(source, seen, use, [&](const Staged& at, const Halves& ds) {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) dq[b] += product_columns(at.first + columns, b, ds.of);
  });
  if (!walk.template join<DP / 32>([&](int b) -> f32x16& { return dq[b]; }) || qi >= t.len) return;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
    store_block(a.dq + ((int64_t(t.start) + qi) * s.heads + head) * s.dim, dq[b] * s.scale, b, h, s.dim);
}

template <int E, int SPLIT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(SPLIT == 1 && E <= 64 ? 2 : 1))) void dq_kernel(const BwdArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[Dq<E, SPLIT>::kBytes];
  Dq<E, SPLIT>::run(a, smem, blockIdx.x, gridDim.x);
}

// Four products of a tile, the scores straight (a lane has 16 queries of a key), so that both sums run
// along what a lane holds.  380 us alone for 2 x 2048, 16 heads of 128: 165 TFLOP/s.
template <int E, int SPLIT>
struct Dkv {
  static constexpr int DP = blocked(E);
  using W = Walk<DP, 4, SPLIT, 1>;
  static constexpr int kAside = SPLIT == 1 && DP == 64 ? E / 16 : 0;  // steps whose values' smallest piece waits in LDS (two waves a SIMD)
  static constexpr int kBytes = W::kBytes + kAside * 4 * 1024;
  static __device__ void run(const BwdArgs a, char* smem, int number, int workgroups);
};
template <int E, int SPLIT>
__device__ __forceinline__ void Dkv<E, SPLIT>::run(const BwdArgs a, char* smem, int number, int workgroups) {
  constexpr int kRows = W::kRows;
  const Shape& s = a.s;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int across = s.kv_heads * a.parts, kv_head = number % across / a.parts, part = number % across % a.parts;
  // (those first, which have the most to do)
  const int index = number / across, block = index - (workgroups / across - a.near);
  const bool far = block < 0;
  const int chunk = far ? index / a.far_blocks : 0, far_block = far ? index % a.far_blocks : 0;
  SequenceTile t;
  if (far ? !locate<kChunk>(s.seqs, chunk, t) : !locate<kRows>(s.seqs, block, t)) return;
  const int b0 = (far ? far_block : t.index) * kRows;
  if (b0 >= t.len) return;
  const int base32 = t.start / kTile + t.seq;
  // The tiles of queries that see any of the workgroup's keys, of each head in turn.
  int from = b0 / kTile, to = near_last(a, b0, t.len) / kTile;
  if (far) {
    from = max(to + 1, t.index * (kChunk / kTile));
    to = min(t.len - 1, (t.index + 1) * kChunk - 1) / kTile;
  }
  const int tiles = to + 1 - from;
  if (tiles <= 0) return;
  const int heads = s.group / a.parts, head0 = kv_head * s.group + part * heads, count = heads * tiles;
  const W walk{{lds_address(smem)}, wave, lane, count};
  const auto source = [&](int n) {
    const int head = head0 + n / tiles, tile = base32 + from + n % tiles;
    const int64_t at = tile_at<DP>(s, head, tile);
    return Source{a.qp + at, a.dp + at, reinterpret_cast<const char*>(a.stats + (int64_t(head) * s.tiles + tile) * 64)};
  };
  walk.start(source);
  const int j0 = b0 + walk.rows(), j1 = j0 + kTile - 1, kj = j0 + tile_row(lane & 31);
  const int64_t mine = tile_at<DP>(s, kv_head, base32 + min(j0, t.len - 1) / kTile);
  Frag3 k[E / 16], v[E / 16];
  own_rows(k, a.kp + mine, lane);
  own_rows(v, a.vp + mine, lane);
  bf16x8* const aside_at = reinterpret_cast<bf16x8*>(smem + W::kBytes) + wave * kAside * 64 + lane;
#pragma unroll
  for (int i = 0; i < kAside; ++i) aside_at[i * 64] = v[i].lo;
  const auto low = [&](int i) { return i < kAside ? aside_at[i * 64] : v[i].lo; };
  f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
  const uint32_t columns = column_base(lane);
  const auto seen = [&](int n) {
    const int i0 = (from + n % tiles) * kTile;
    return j0 < t.len && !s.mask.none(i0, i0 + kTile - 1, j0, j1);
  };
  const auto use = [&](int n, const Staged& at) {
    const int i0 = (from + n % tiles) * kTile;
    f32x16 x = product<3>(at.first, k, lane), delta;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t stats = at.stats + (16 * h + 4 * i) * 4;
      const f32x4 lse = *pieces::lds_at<const f32x4>(stats), d = *pieces::lds_at<const f32x4>(stats + 128);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] -= lse[e], delta[4 * i + e] = d[e];
    }
    if (!s.mask.all(i0, i0 + kTile - 1, j0, j1)) hide(x, [&](int r) { return s.mask.sees(i0 + 16 * h + r, kj); });
    f32x16 dp = product<3>(at.second, v, lane, low);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = exp2_(x[r]);
      dp[r] = times(x[r], dp[r] - delta[r]);
    }
    const Frag3 p[2] = {split_half(x, 0), split_half(x, 1)};
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) dv[b] += product_columns(at.second + columns, b, p);
    return Halves{{split_half(dp, 0), split_half(dp, 1)}};
  };
  walk.run(source, seen, use, [&](const Staged& at, const Halves& ds) {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) dk[b] += product_columns(at.first + columns, b, ds.of);
  });
  if (!walk.template join<DP / 16>([&](int b) -> f32x16& { return b < DP / 32 ? dk[b] : dv[b - DP / 32]; })) return;
  if (kj >= t.len || (far && j0 >= s.mask.sinks)) return;
  float *to_k = a.dk, *to_v = a.dv;
  int64_t at = ((int64_t(t.start) + kj) * s.kv_heads + kv_head) * s.dim;
  if (far) {
    to_k = far_at(a, chunk, far_block, kv_head, part), to_v = to_k + kRows * s.dim;
    at = int64_t(kj - b0) * s.dim;
  } else if (a.parts > 1) {
    to_k = a.dk_p, to_v = a.dv_p;
    at += int64_t(part) * s.seqs.tokens * s.kv_heads * s.dim;
  }
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) {
    // q was packed times scale log2(e)
    if (a.dk) store_block(to_k + at, dk[b] * kLn2, b, h, s.dim);
    if (a.dv) store_block(to_v + at, dv[b], b, h, s.dim);
  }
}
template <int E, int SPLIT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(SPLIT == 1 && E <= 64 ? 2 : 1))) void dkv_kernel(const BwdArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[Dkv<E, SPLIT>::kBytes];
  Dkv<E, SPLIT>::run(a, smem, blockIdx.x, gridDim.x);
}
// Both, where workgroups are few: `first` of dk and dv, then those of dq, which fill the CUs that the others
// leave.  Calls with packing, in two launches and in one: 4 x 256, 12 heads of 64 46 and 38 us, 2048, 8 heads
// of 128 301 and 192, 2 x 2048, 16 heads of 128 716 and 711 (184 TFLOP/s without packing and the join, 1.1
// PFLOP/s of pieces).
template <int E>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(1))) void both_kernel(const BwdArgs a, int first) {
  __shared__ __attribute__((aligned(1024))) char smem[std::max(Dkv<E, 2>::kBytes, Dq<E, 2>::kBytes)];
  if (int(blockIdx.x) < first) Dkv<E, 2>::run(a, smem, blockIdx.x, first);
  else Dq<E, 2>::run(a, smem, blockIdx.x - first, gridDim.x - first);
}

// What queries past the window give first tokens' dk and dv, added to the rest: grid (blocks of
// keys times workgroups of a block, key heads, sequences or fewer).
__global__ __launch_bounds__(kThreads) void far_kernel(const BwdArgs a) {
  const Shape& s = a.s;
  const int per = gridDim.x / a.far_blocks, block = blockIdx.x / per, b0 = block * a.block;
  const int i = (blockIdx.x - block * per) * kThreads + threadIdx.x;
  for (int seq = blockIdx.z; seq < s.seqs.count; seq += gridDim.z) {
    const int start = s.seqs.start(seq), len = max(0, s.seqs.start(seq + 1) - start);
    if (b0 >= len || near_last(a, b0, len) / kTile == (len - 1) / kTile) continue;  // no queries past the window
    const int from = (near_last(a, b0, len) / kTile + 1) * kTile / kChunk, to = (len - 1) / kChunk, base = start / kChunk + seq;
    const int rows = min(min(a.block, len - b0), (s.mask.sinks - b0 + kTile - 1) / kTile * kTile);
    if (i >= rows * s.dim) continue;
    const int64_t at = ((int64_t(start) + b0 + i / s.dim) * s.kv_heads + blockIdx.y) * s.dim + i % s.dim;
    float k = a.dk ? a.dk[at] : 0.f, v = a.dv ? a.dv[at] : 0.f;
    // (eight sums on their way at a time; those of a gradient that is not wanted are not looked at)
    const int sums = (to - from + 1) * a.parts;
#pragma unroll 8
    for (int n = 0; n < sums; ++n) {
      const float* const sum = far_at(a, base + from + n / a.parts, block, blockIdx.y, n % a.parts) + i;
      k += sum[0];
      v += sum[a.block * s.dim];
    }
    if (a.dk) a.dk[at] = k;
    if (a.dv) a.dv[at] = v;
  }
}

// dk and dv: the parts' sums, in order, over the rows from the first sequence's start to the
// last one's end (14 us for four parts of 4096 x 4 x 128: 6 TB/s, in part from the cache).
__global__ __launch_bounds__(kThreads) void join_kernel(const BwdArgs a) {
  const Shape& s = a.s;
  const int64_t row = int64_t(s.kv_heads) * s.dim, step = s.seqs.tokens * row;
  const int64_t end = s.seqs.start(s.seqs.count) * row;
  const float* const from = blockIdx.y ? a.dv_p : a.dk_p;
  float* const to = blockIdx.y ? a.dv : a.dk;
  if (!to) return;
  for (int64_t i = s.seqs.start(0) * row + (int64_t(blockIdx.x) * kThreads + threadIdx.x) * 4; i < end;
       i += int64_t(gridDim.x) * kThreads * 4) {
    if (i + 4 <= end) {
      f32x4 v{};
#pragma unroll 4
      for (int p = 0; p < a.parts; ++p) v += *reinterpret_cast<const f32x4u*>(from + p * step + i);
      *reinterpret_cast<f32x4u*>(to + i) = v;
    } else {
      for (int64_t e = i; e < end; ++e) {
        float v = 0;
        for (int p = 0; p < a.parts; ++p) v += from[p * step + e];
        to[e] = v;
      }
    }
  }
}

// dk (y 0) and dv (y 1) of key heads without query heads: 0 in the sequences' rows, of `row` elements.
__global__ __launch_bounds__(kThreads) void no_heads_kernel(const Sequences seqs, int64_t row, float* dk, float* dv) {
  float* const to = blockIdx.y ? dv : dk;
  if (!to) return;
  const int64_t end = seqs.start(seqs.count) * row;
  for (int64_t i = seqs.start(0) * row + int64_t(blockIdx.x) * kThreads + threadIdx.x; i < end; i += int64_t(gridDim.x) * kThreads)
    to[i] = 0;
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
  // (a grid's work-items are counted in 32 bits; the largest has far blocks' chunks among its blocks)
  MX_REQUIRE(d->tokens <= (1 << 28) && d->sequences <= (1 << 21) && d->heads + d->kv_heads <= 65535 &&
                 (d->tokens / kBlock + d->sequences + kFarBlocks * (d->tokens / kChunk + d->sequences)) * d->heads < (1 << 24),
             MX_ERR_INVALID, who, ": size out of range");
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

int padded(int64_t dim) { return blocked(int(dim)); }

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
  char *qp, *kp, *vp, *dp;
  float *stats, *dk_p, *dv_p, *far;
};

// Blocks of keys that are seen past the window by workgroups of their own (of more first tokens
// the blocks behind have as much to do as each other), and chunks of queries.
int64_t far_blocks_of(const Shape& s, int block) {
  if (!s.mask.window || s.mask.window >= s.seqs.tokens) return 0;
  return std::min<int64_t>((std::min(s.mask.sinks, s.seqs.tokens) + block - 1) / block, kFarBlocks);
}
int64_t chunks_of(const Shape& s) { return sequence_tiles(s.seqs.tokens, s.seqs.count, kChunk); }

int64_t blocks_of(const Shape& s, int rows = kBlock) { return sequence_tiles(s.seqs.tokens, s.seqs.count, rows); }

// Parts that a key head's query heads are dealt into: as few as give every CU four
// workgroups of 128 keys (the first keys of a sequence have the most to do).
int parts_of(const Shape& s) {
  for (int p = 1; p <= s.group; ++p)
    if (s.group % p == 0 && blocks_of(s) * s.kv_heads * p >= int64_t(cu_count()) * 4) return p;
  return s.group;
}

// Whether workgroups of 128 rows, `blocks` in all, are so few that ones of 64 rows, which take two
// tiles at a time (one workgroup a CU for LDS), end sooner.  Four sequences of 256, 12 heads of 64: 28, 34 and 39 us
// for out, dq, and dk and dv with their packing, halved 23, 26 and 30; one of 2048, 8 heads of 128
// 160, 245 and 329, halved 108, 134 and 187.  From about three workgroups a CU on dq, dk and dv take
// as long either way (2 x 2048, 20 heads of 64: 222 and 299 us, halved 222 and 287; 4 x 2048, 14 of
// 96: 481 and 615, halved 512 and 643).  Forward walks gain less: two waves a SIMD, or for heads of 128
// scores ahead, go without (544 workgroups of 64 154 us, halved 144, 680 159 and 175; of 128, 320 68 and
// 68, 544 209 and 237); with a window, whose walks are alike, 272 of 64 36 and 40.
bool halved(const Shape& s, int64_t blocks, bool forward) {
  const bool alike = s.mask.window && s.mask.window < s.seqs.tokens;
  return blocks < int64_t(cu_count()) * (!forward ? 3 : alike || s.dim > 96 ? 1 : 2);
}
int key_block_of(const Shape& s) { return halved(s, blocks_of(s) * s.kv_heads * parts_of(s), false) ? kBlock / 2 : kBlock; }

Buffers carve(const Shape& s, bool backward, Carve& c) {
  const int64_t tile = padded(s.dim) / 16 * 3 * 1024, q = tile * s.tiles * s.heads, k = tile * s.tiles * s.kv_heads;
  Buffers b{};
  b.kp = c.take<char>(k);
  b.vp = c.take<char>(k);
  if (!backward) return b;
  const int parts = parts_of(s), block = key_block_of(s);
  b.qp = c.take<char>(q);
  b.dp = c.take<char>(q);
  b.stats = c.take<float>(int64_t(s.heads) * s.tiles * 256);
  if (parts > 1) {
    const int64_t part = (int64_t(parts) * s.seqs.tokens * s.kv_heads * s.dim * 4 + 255) / 256 * 256;
    b.dk_p = c.take<float>(part);
    b.dv_p = c.take<float>(part);
  }
  b.far = c.take<float>(chunks_of(s) * far_blocks_of(s, block) * s.kv_heads * parts * (2 * block * int64_t(s.dim) * 4));
  return b;
}

int64_t workspace_bytes_of(const mx_attention_desc* d, bool backward) {
  if (d->tokens == 0 || d->heads == 0) return 0;
  Carve c{nullptr};
  const Shape s = shape_of(d);
  carve(s, backward, c);
  return c.used;
}

// f with the head's elements padded to 16.
template <int E = 16, class F>
void with_dim(int dim, F&& f) {
  if (dim <= E) return f(std::integral_constant<int, E>{});
  if constexpr (E < kMaxDim) with_dim<E + 16>(dim, f);
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
  p.k = {k, d->k_token, d->k_head}, p.v = {v, d->v_token, d->v_head};
  p.kp = b.kp, p.vp = b.vp;
  const FwdArgs f{s, {q, d->q_token, d->q_head}, b.kp, b.vp, out, lse};
  with_dim(s.dim, [&](auto dp) {
    hipLaunchKernelGGL((pack_kernel<blocked(decltype(dp)::value)>), dim3(s.tiles, s.kv_heads), dim3(kThreads), 0, st, p);
  });
  MX_LAUNCHED();
  with_dim(s.dim, [&](auto dp) {
    constexpr int E = decltype(dp)::value;
    const int64_t wide = sequence_tiles(s.seqs.tokens, s.seqs.count, 8 * kTile) * s.heads;
    if (wide_blocks(wide)) {
      hipLaunchKernelGGL((fwd_kernel<E, 8, 1>), dim3(unsigned(wide)), dim3(512), 0, st, f);
      return;
    }
    if (halved(s, blocks_of(s) * s.heads, true)) {
      hipLaunchKernelGGL((fwd_kernel<E, 4, 2>), dim3(unsigned(blocks_of(s, kBlock / 2) * s.heads)), dim3(256), 0, st, f);
      return;
    }
    hipLaunchKernelGGL((fwd_kernel<E, 4, 1>), dim3(unsigned(blocks_of(s) * s.heads)), dim3(256), 0, st, f);
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
  if (d->tokens == 0 || (!dq && !dk && !dv)) return MX_OK;
  if (d->heads == 0) {
    const int64_t row = d->kv_heads * d->head_dim;
    if (row == 0 || (!dk && !dv)) return MX_OK;
    const unsigned blocks = unsigned(std::min<int64_t>((d->tokens * row + kThreads - 1) / kThreads, int64_t(cu_count()) * 8));
    hipLaunchKernelGGL(no_heads_kernel, dim3(blocks, 2), dim3(kThreads), 0, resolve_stream(stream),
                       Sequences{d->starts, int(d->tokens), int(d->sequences)}, row, dk, dv);
    MX_LAUNCHED();
    return MX_OK;
  }
  MX_REQUIRE(dout && q && k && v && out && lse, MX_ERR_INVALID, who, ": null buffer");
  const Shape s = shape_of(d);
  hipStream_t st = resolve_stream(stream);
  Workspace ws;
  MX_TRY(ws.take(who, workspace, workspace_bytes, workspace_bytes_of(d, true), st));
  Carve c{ws.as<char>()};
  const int parts = parts_of(s), block = key_block_of(s);
  const Buffers b = carve(s, true, c);
  PackArgs p{};
  p.s = s;
  p.q = {q, d->q_token, d->q_head}, p.k = {k, d->k_token, d->k_head}, p.v = {v, d->v_token, d->v_head};
  p.dout = {dout, d->heads * d->head_dim, d->head_dim}, p.out = {out, d->heads * d->head_dim, d->head_dim};
  p.lse = lse;
  p.qp = b.qp, p.kp = b.kp, p.vp = b.vp, p.dp = b.dp, p.stats = b.stats;
  const BwdArgs g{s, b.qp, b.kp, b.vp, b.dp, b.stats, dq, dk, dv, parts, b.dk_p, b.dv_p, block, int(blocks_of(s, block)), int(far_blocks_of(s, block)), b.far};
  with_dim(s.dim, [&](auto dp) {
    hipLaunchKernelGGL((pack_kernel<blocked(decltype(dp)::value)>), dim3(s.tiles, s.heads + s.kv_heads), dim3(kThreads), 0, st, p);
  });
  MX_LAUNCHED();
  const bool keys = dk || dv, key_halves = block < kBlock, query_halves = halved(s, blocks_of(s) * s.heads, false);
  const unsigned of_keys = unsigned((g.near + chunks_of(s) * g.far_blocks) * s.kv_heads * parts);
  const unsigned of_queries = unsigned(blocks_of(s, query_halves ? kBlock / 2 : kBlock) * s.heads);
  const bool both = dq && keys && key_halves && query_halves;
  if (both) {
    with_dim(s.dim, [&](auto dp) {
      hipLaunchKernelGGL((both_kernel<decltype(dp)::value>), dim3(of_keys + of_queries), dim3(kThreads), 0, st, g, int(of_keys));
    });
    MX_LAUNCHED();
  } else if (dq) {
    with_dim(s.dim, [&](auto dp) {
      constexpr int E = decltype(dp)::value;
      if (query_halves) hipLaunchKernelGGL((dq_kernel<E, 2>), dim3(of_queries), dim3(kThreads), 0, st, g);
      else hipLaunchKernelGGL((dq_kernel<E, 1>), dim3(of_queries), dim3(kThreads), 0, st, g);
    });
    MX_LAUNCHED();
  }
  if (keys) {
    if (!both) {
      with_dim(s.dim, [&](auto dp) {
        constexpr int E = decltype(dp)::value;
        if (key_halves) hipLaunchKernelGGL((dkv_kernel<E, 2>), dim3(of_keys), dim3(kThreads), 0, st, g);
        else hipLaunchKernelGGL((dkv_kernel<E, 1>), dim3(of_keys), dim3(kThreads), 0, st, g);
      });
      MX_LAUNCHED();
    }
    if (parts > 1) {
      const int64_t fours = (d->tokens * d->kv_heads * d->head_dim + 3) / 4;
      const unsigned blocks = unsigned(std::min<int64_t>((fours + kThreads - 1) / kThreads, int64_t(cu_count()) * 8));
      hipLaunchKernelGGL(join_kernel, dim3(blocks, 2), dim3(kThreads), 0, st, g);
      MX_LAUNCHED();
    }
    if (g.far_blocks) {
      const int rows = std::min(block, (std::min(s.mask.sinks, block) + kTile - 1) / kTile * kTile);
      const unsigned per = unsigned((rows * s.dim + kThreads - 1) / kThreads);
      hipLaunchKernelGGL(far_kernel, dim3(unsigned(g.far_blocks) * per, unsigned(s.kv_heads), unsigned(std::min(s.seqs.count, 4096))),
                         dim3(kThreads), 0, st, g);
      MX_LAUNCHED();
    }
  }
  return MX_OK;
  MX_ABI_END
}
