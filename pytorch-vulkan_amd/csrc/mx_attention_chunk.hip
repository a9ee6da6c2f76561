// Attention of chunks of many new tokens over a paged cache: the matrix instructions bound it,
// so what the chunk sees is packed once (gather_kernel) and the products read whole fragments
// through LDS, as in mx_attention.hip, for all rows of a sequence and key head.
//
// Keys are packed by row as there; values by element, which is how the cache holds them:
// lane l of block b and step t has element 32 b + l % 32 of keys 16 (l / 32) + 8 t + 0 .. 7, and
// needs no transposing read.  Bytes are one bf16 piece (three matrix instructions a product in
// place of six), and their scales go to the scores and the probabilities.  Keys without a page
// are marked; a row of an FP32 cache that is not finite has NaN keys and zero values.
#include <algorithm>
#include <cmath>

#include "mx_attention_paged.hpp"

namespace mx {
namespace {

using namespace attn;

constexpr int kStat = 128;  // floats of a tile: 32 key scales, 32 value scales, 32 marks of absent keys, any mark

struct ChunkArgs : Paged {
  int tiles, splits;  // tiles of keys, the most of a sequence; workgroups that share a row's keys
  char *kp, *vp;
  float* stats;
  float *part, *stat;  // of each split: [token][head][dim], [token][head] maxima and sums
};

// [key head][sequence][tile of what the sequence's new tokens see]
__device__ __forceinline__ int64_t tile_of(const ChunkArgs& a, int head, int seq, int n) {
  return (int64_t(head) * a.b.seqs.count + seq) * a.tiles + n;
}

// The tiles that a sequence's new tokens see, of which there may be more than were made room for
// only where a table is wider than the call's window and tokens reach: never.
__device__ __forceinline__ KeyTiles<> seen_by_all(const ChunkArgs& a, const RowTile<1>& rt) {
  return KeyTiles<>(a.mask, max(rt.first, 0), min(rt.first + rt.t.len / a.group - 1, rt.length - 1));
}

// grid (tiles, kv heads, sequences): 32 keys of one head and sequence.  (22 us for 4 sequences' 4608 keys of 4
// heads of 128, 57 MB: many short workgroups, each waiting for lengths, table and cache in turn.)
template <int DP, bool I8>
__global__ __launch_bounds__(256) void gather_kernel(const ChunkArgs a) {
  constexpr int P = I8 ? 1 : 3;
  using E = std::conditional_t<I8, int8_t, float>;
  __shared__ uint32_t bad[4];
  const kv::Cache& c = a.c;
  const int seq = blockIdx.z, head = blockIdx.y;
  RowTile<1> rt;
  rt.t.seq = seq, rt.t.start = a.b.seqs.start(seq), rt.t.len = max(0, a.b.seqs.start(seq + 1) - rt.t.start);
  if (rt.t.len == 0) return;
  rt.whole(a);
  const KeyTiles<> keys = seen_by_all(a, rt);
  if (int(blockIdx.x) >= keys.count) return;
  const int j0 = keys.tile(blockIdx.x) * kTile;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  int place[2], page[2];
  int64_t at[2];  // places' rows in the cache
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    page[g] = kv::page_of(c, a.b, seq, (j0 >> 4) + g, place[g]);
    at[g] = (int64_t(max(page[g], 0)) * c.heads + head) * c.page_size + place[g];
  }
  const int64_t tile = tile_of(a, head, seq, blockIdx.x);
  const auto there = [&](int r) { return page[r >> 4] >= 0 && j0 + r < rt.length; };
  // ---- values: block b's lane has 16 keys of one element
  uint32_t odd = 0;
  for (int b = wave; b < DP / 32; b += 4) {
    const int d = 32 * b + (lane & 31), g = h;
    Sixteen<I8> v{};
    if (d < c.dim && (g ? page[1] : page[0]) >= 0)
      v.load(static_cast<const E*>(c.v) + ((g ? at[1] - place[1] : at[0] - place[0])) * c.dim + int64_t(d) * c.page_size + (g ? place[1] : place[0]));
    if constexpr (!I8) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool fine = finite(v.raw[r >> 2][r & 3]), use = j0 + 16 * h + r < rt.length;
        if (!fine && use) odd |= 1u << r;
        if (!fine || !use) v.raw[r >> 2][r & 3] = 0;
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      bf16x8* const to = reinterpret_cast<bf16x8*>(a.vp + tile * kTileBytes<DP, P>) + (2 * b + t) * P * 64 + slot(lane);
      const Frag<P> f = v.half(t);
      if constexpr (I8) to[0] = f;
      else to[0] = f.hi, to[64] = f.mid, to[128] = f.lo;
    }
  }
  uint32_t bits = 0;
  if constexpr (!I8) {
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) odd |= __shfl_xor(int(odd), m, 64);
    const uint32_t low = __shfl(int(odd), 0, 64), high = __shfl(int(odd), 32, 64);
    if (lane == 0) bad[wave] = low | high << 16;
    __syncthreads();
    bits = bad[0] | bad[1] | bad[2] | bad[3];
  }
  // ---- keys: step s's lane has 8 elements of key tile_row(l % 32)
  const int r = tile_row(lane & 31);
  const bool here = there(r);
  for (int s = wave; s < DP / 16; s += 4) {
    const int e = 16 * s + 8 * h;
    Frag<P> f{};
    const bool has = here && e < c.dim;
    const E* const from = static_cast<const E*>(c.k) + ((r >> 4 ? at[1] : at[0]) + (r & 15)) * c.dim + e;
    bf16x8* const to = reinterpret_cast<bf16x8*>(a.kp + tile * kTileBytes<DP, P>) + s * P * 64 + slot(lane);
    if constexpr (I8) {
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      Sixteen<true> k{};
      if (has) {
        const i32x2 two = *reinterpret_cast<const i32x2*>(from);
        k.raw[0] = two[0], k.raw[1] = two[1];
      }
      to[0] = k.half(0);
    } else {
      f32x4 v[2] = {};
      if (has) v[0] = reinterpret_cast<const f32x4*>(from)[0], v[1] = reinterpret_cast<const f32x4*>(from)[1];
      if (bits >> r & 1) v[0] = v[1] = f32x4{1, 1, 1, 1} * __builtin_nanf("");
      f = split8(v[0], v[1]);
      to[0] = f.hi, to[64] = f.mid, to[128] = f.lo;
    }
  }
  // ---- scales and marks
  if (wave == 0 && h == 0) {
    const int n = lane;
    float* const to = a.stats + tile * kStat;
    const bool ok = there(n);
    if constexpr (I8) {
      const int64_t row = (n >> 4 ? at[1] : at[0]) + (n & 15);
      const float ks = ok ? c.ks[row] : 0.f, vs = ok ? c.vs[row] : 0.f;
      to[n] = fmaf(vs, 0.f, ks);  // a NaN value: NaN scores, whatever their probability
      to[32 + n] = vs;
    }
    to[64 + n] = ok ? 0.f : 1.f;
    const bool any = __ballot(!ok) & 0xFFFFFFFFu;
    if (n == 0) to[96] = any ? 1.f : 0.f;
  }
}

// 4 x 512 tokens, 16 heads of 128, 8-bit keys, window 4096: 199 us, 346 TFLOP/s, 1.04 PFLOP/s of pieces.
template <int DP, bool I8, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(I8 || DP <= 96 ? 2 : 1))) void chunk_kernel(
    const ChunkArgs a) {
  constexpr int P = I8 ? 1 : 3, kRows = WAVES * kTile;
  using St = Stages<DP, P, WAVES, 2>;
  constexpr int kAside = I8 && DP == 128 ? 4 : 0;  // steps whose queries' smallest piece waits in LDS
  __shared__ __attribute__((aligned(1024))) char smem[2 * St::kBytes + kAside * WAVES * 1024];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int head = blockIdx.x % a.c.heads, block = gridDim.x / a.c.heads - 1 - blockIdx.x / a.c.heads;
  RowTile<kRows> rt;
  if (!rt.find(a, block)) return;
  const SequenceTile& t = rt.t;
  RowTile<1> all;
  all.t = t;
  all.whole(a);
  const KeyTiles<> packed = seen_by_all(a, all), keys(a.mask, max(rt.i0, 0), rt.end);
  const int span = a.c.pages ? (keys.count + a.splits - 1) / a.splits : 0;
  const int begin = blockIdx.y * span, end = min(keys.count, begin + span);
  // The wave's rows, and the lane's.
  const int r0 = t.index * kRows + wave * kTile, row = r0 + tile_row(lane & 31);
  const int token = min(row, t.len - 1) / a.group, pos = rt.first + token;
  const int q_head = head * a.group + min(row, t.len - 1) - token * a.group;
  const int64_t flat = t.start / a.group + token;
  const int i0 = rt.first + min(r0, t.len - 1) / a.group, i1 = rt.first + (min(r0 + kTile, t.len) - 1) / a.group;
  const St st{lds_address(smem)};
  const auto fetch = [&](int n) {
    const int j = keys.tile(n);
    const int64_t tile = tile_of(a, head, t.seq, j < packed.sinks ? j : packed.sinks + j - packed.from);
    st.load(n & 1, a.kp + tile * kTileBytes<DP, P>, a.vp + tile * kTileBytes<DP, P>,
            reinterpret_cast<const char*>(a.stats + tile * kStat), wave, lane);
  };
  if (begin < end) fetch(begin);
  Frag3 q[DP / 16];
  {
    const float* const src = a.q + flat * a.q_token + q_head * a.q_head;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      f32x4 v[2];
      load8(src, s * 16 + h * 8, a.c.dim, v);
      q[s] = split8(v[0] * (a.scale * kLog2E), v[1] * (a.scale * kLog2E));
    }
  }
  bf16x8* const mine = reinterpret_cast<bf16x8*>(smem + 2 * St::kBytes) + wave * kAside * 64 + lane;
#pragma unroll
  for (int i = 0; i < kAside; ++i) mine[i * 64] = q[i].lo;
  const auto low = [&](int i) { return i < kAside ? mine[i * 64] : q[i].lo; };
  f32x16 o[DP / 32] = {};
  float m = -__builtin_inff(), l = 0;  // of the exponents
  for (int n = begin; n < end; ++n) {
    pieces::wait_loads<0>();
    pieces::barrier();
    if (n + 1 < end) fetch(n + 1);
    const int j0 = keys.tile(n) * kTile;
    if (r0 >= t.len || a.mask.none(i0, i1, j0, j0 + kTile - 1)) continue;
    const uint32_t tile = st.lds + (n & 1) * St::kBytes, stats = tile + St::kStats + 64 * h;
    f32x16 x = product<P>(tile, q, lane, low);
    const auto scaled = [&](int which, int i) { return *pieces::lds_at<const f32x4>(stats + 128 * which + 16 * i); };
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 ks = scaled(0, i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * i + e] *= ks[e];
      }
    }
    const bool absent = __builtin_amdgcn_readfirstlane(*pieces::lds_at<const int>(tile + St::kStats + 384)) != 0;
    if (absent || !a.mask.all(i0, i1, j0, j0 + kTile - 1)) {
      f32x16 marks;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 four = scaled(2, i);
#pragma unroll
        for (int e = 0; e < 4; ++e) marks[4 * i + e] = four[e];
      }
      hide(x, [&](int r) { return marks[r] == 0 && a.mask.sees(pos, j0 + 16 * h + r); });
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
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 vs = scaled(1, i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * i + e] = times(x[4 * i + e], vs[e]);
      }
    }
    const Frag3 p[2] = {split_half(x, 0), split_half(x, 1)};
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) {
      if (DP > 96 && (!I8 || b % 2 == 0)) __builtin_amdgcn_sched_barrier(0);  // one block's fragments at a time
      o[b] = o[b] * keep + product_halves(frag<P>(tile + St::kSecond, 2 * b, lane), frag<P>(tile + St::kSecond, 2 * b + 1, lane), p);
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (row >= t.len) return;
  const int64_t out_row = flat * a.heads + q_head;
  if (a.splits > 1) {
    const int64_t rows = int64_t(a.b.seqs.tokens) * a.heads, at = blockIdx.y * rows + out_row;
    if (h == 0) a.stat[2 * at] = m, a.stat[2 * at + 1] = l;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) store_block(a.part + at * a.c.dim, o[b], b, h, a.c.dim);
    return;
  }
  const float r = l == 0 ? 0.f : 1.f / l;  // a row that sees nothing
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) store_block(a.out + out_row * a.c.dim, o[b] * r, b, h, a.c.dim);
}

// The workgroups that shared a row's keys, in order: 32 lanes to a row of any sequence.
constexpr int kMaxSplits = 8;
__global__ __launch_bounds__(256) void chunk_join_kernel(const ChunkArgs a) {
  const int64_t rows = int64_t(a.b.seqs.tokens) * a.heads, first = int64_t(a.b.seqs.start(0) / a.group) * a.heads;
  const int64_t row = first + int64_t(blockIdx.x) * 8 + threadIdx.x / 32;
  if (row >= int64_t(a.b.seqs.start(a.b.seqs.count) / a.group) * a.heads) return;
  float m[kMaxSplits], l[kMaxSplits], all = -__builtin_inff(), total = 0;
#pragma unroll
  for (int i = 0; i < kMaxSplits; ++i) {
    m[i] = i < a.splits ? a.stat[2 * (i * rows + row)] : -__builtin_inff();
    l[i] = i < a.splits ? a.stat[2 * (i * rows + row) + 1] : 0.f;
    all = fmaxf(all, m[i]);
  }
  const float base = all == -__builtin_inff() ? 0.f : all;
#pragma unroll
  for (int i = 0; i < kMaxSplits; ++i) {
    m[i] = exp2_(m[i] - base);
    total = fmaf(l[i], m[i], total);
  }
  const float inv = total == 0 ? 0.f : 1.f / total;
  const int e = (threadIdx.x & 31) * 4;
  if (e >= a.c.dim) return;
  f32x4 v{};
#pragma unroll
  for (int i = 0; i < kMaxSplits; ++i)
    if (i < a.splits) v += *reinterpret_cast<const f32x4u*>(a.part + (i * rows + row) * a.c.dim + e) * m[i];
  *reinterpret_cast<f32x4u*>(a.out + row * a.c.dim + e) = v * inv;
}

int padded(int64_t dim) { return int((dim + 31) / 32 * 32); }

// The most tiles of 32 keys that a sequence's new tokens see.
int64_t tiles_of(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b) {
  const int64_t keys = b->table_width * c->page_size, most = (keys + kTile - 1) / kTile;
  if (!d->window) return most;
  const int64_t near = (std::min(d->window, keys) + b->tokens) / kTile + 2, sinks = (std::min(d->sinks, keys) + kTile - 1) / kTile;
  return std::min(most, near + sinks);
}

int64_t row_blocks(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b, int waves) {
  return sequence_tiles(b->tokens * (d->heads / c->heads), b->sequences, waves * kTile) * c->heads;
}

// How the call runs: waves of a workgroup, and how many workgroups share a row's keys, with eight
// tiles of keys at least to each: as many as give every CU what its registers and LDS hold (16 heads
// of 128, 4 x 512 tokens over 8-bit keys: 348 us unshared, 235 by two, 242 by four; heads of
// 64 225, 176 and 148; FP32 keys, heads of 128, one workgroup a CU: 456, 464 and 481).
struct Form {
  int waves, splits;
};
Form form_of(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b) {
  const bool i8 = c->type == MX_KV_I8;
  const int dim = padded(c->head_dim), per_cu = dim <= 64 ? 4 : i8 || dim <= 96 ? 2 : 1;
  if ((i8 || dim <= 96) && wide_blocks(row_blocks(d, c, b, 8))) return {8, 1};
  const int64_t blocks = std::max<int64_t>(1, row_blocks(d, c, b, 4)), want = (int64_t(cu_count()) * per_cu + blocks / 2) / blocks;
  return {4, int(std::max<int64_t>(1, std::min<int64_t>({want, tiles_of(d, c, b) / 8, kMaxSplits})))};
}

template <int DP, bool I8>
int launch(const ChunkArgs& a, int waves, int64_t blocks, hipStream_t s) {
  hipLaunchKernelGGL((gather_kernel<DP, I8>), dim3(unsigned(a.tiles), unsigned(a.c.heads), unsigned(a.b.seqs.count)), dim3(256), 0,
                     s, a);
  MX_LAUNCHED();
  const dim3 grid(unsigned(blocks), unsigned(a.splits));
  if constexpr (I8 || DP <= 96)
    if (waves == 8) {
      hipLaunchKernelGGL((chunk_kernel<DP, I8, 8>), grid, dim3(512), 0, s, a);
      MX_LAUNCHED();
      return MX_OK;
    }
  hipLaunchKernelGGL((chunk_kernel<DP, I8, 4>), grid, dim3(256), 0, s, a);
  MX_LAUNCHED();
  if (a.splits > 1) {
    hipLaunchKernelGGL(chunk_join_kernel, dim3(unsigned((int64_t(a.b.seqs.tokens) * a.heads + 7) / 8)), dim3(256), 0, s, a);
    MX_LAUNCHED();
  }
  return MX_OK;
}

// Bytes of the packed tiles, their scales and marks, and the parts.
struct Sizes {
  int64_t tiles, stats, part;
};
Sizes sizes_of(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b, int splits) {
  const int64_t all = tiles_of(d, c, b) * c->heads * b->sequences, rows = splits > 1 ? b->tokens * d->heads * splits : 0;
  return {all * (padded(c->head_dim) / 16 * 1024 * (c->type == MX_KV_I8 ? 1 : 3)), all * kStat * 4,
          (rows * c->head_dim * 4 + 15) / 16 * 16};
}

}  // namespace

// Rows of a sequence and key head from which packing is paid back.  Chunk's and token's form, us, 16
// heads of 128, contexts of 2048: 8 bits, 4 key heads, 16 sequences, 128 rows 89 and 68, 256
// 98 and 98, 512 165 and 162; FP32, 64 rows 146 and 138, 128 188 and 219, 512 333 and 607; 8 sequences of 16
// key heads, 128 rows 343 and 394.  (Scratch is held to 2 GiB, a bound that is not measured; past it the token's form runs:
// 4 x 512 tokens over 4096, 32 heads, 8 key heads of 128 577 us for 367 in 8 bits, 1846 for 805 in FP32.)
int64_t attn::chunk_workspace(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b) {
  const int64_t rows = b->tokens * (d->heads / c->heads);
  if (rows < (c->type == MX_KV_I8 ? 768 : 128) * b->sequences || b->sequences > 65535 || tiles_of(d, c, b) == 0) return 0;
  const int splits = form_of(d, c, b).splits;
  const Sizes z = sizes_of(d, c, b, splits);
  const int64_t bytes = 2 * z.tiles + z.stats + z.part + (splits > 1 ? b->tokens * d->heads * splits * 8 : 0);
  return bytes <= int64_t(1) << 31 ? bytes : 0;
}

int attn::chunk_attention(const Paged& p, const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b, char* workspace,
                          hipStream_t s) {
  ChunkArgs a{};
  static_cast<Paged&>(a) = p;
  const Form f = form_of(d, c, b);
  const Sizes z = sizes_of(d, c, b, f.splits);
  a.tiles = int(tiles_of(d, c, b)), a.splits = f.splits;
  a.kp = workspace, a.vp = a.kp + z.tiles, a.stats = reinterpret_cast<float*>(a.vp + z.tiles);
  a.part = a.stats + z.stats / 4, a.stat = a.part + z.part / 4;
  const bool i8 = c->type == MX_KV_I8;
  const int64_t blocks = row_blocks(d, c, b, f.waves);
  switch (padded(c->head_dim)) {
    case 32: return i8 ? launch<32, true>(a, f.waves, blocks, s) : launch<32, false>(a, f.waves, blocks, s);
    case 64: return i8 ? launch<64, true>(a, f.waves, blocks, s) : launch<64, false>(a, f.waves, blocks, s);
    case 96: return i8 ? launch<96, true>(a, f.waves, blocks, s) : launch<96, false>(a, f.waves, blocks, s);
    default: return i8 ? launch<128, true>(a, f.waves, blocks, s) : launch<128, false>(a, f.waves, blocks, s);
  }
}

}  // namespace mx
