// What the two forms of attention over a cache share: mx_attention_paged.hip reads the
// cache as it lies, for few rows; mx_attention_chunk.hip packs what a chunk sees.
#pragma once

#include "mx_attention.hpp"
#include "mx_kv_cache.hpp"

namespace mx {
namespace attn {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Rows of a sequence are its new tokens with the query heads that share a key head: row r is token
// r / group, head r % group of the key head's.
struct Paged {
  kv::Cache c;
  kv::Batch b;  // seqs.per is group
  const float* q;
  int64_t q_token, q_head;
  int heads, group;
  Mask mask;
  float scale;
  float* out;
};

// A tile of R rows: its sequence, whose tokens it has and at which positions.
template <int R>
struct RowTile {
  SequenceTile t;
  int length, first;  // tokens of the sequence that its table has room for, its first new one's position
  int i0, i1, end;    // the tile's positions, and the last of them within `length`
  __device__ __forceinline__ bool find(const Paged& a, int tile) {
    if (!locate<R>(a.b.seqs, tile, t) || t.index * R >= t.len) return false;
    whole(a);
    i0 = first + t.index * R / a.group;
    i1 = first + (min(t.len, (t.index + 1) * R) - 1) / a.group;
    end = min(i1, length - 1);
    return true;
  }
  __device__ __forceinline__ void whole(const Paged& a) {
    const int last = max(a.b.lengths[t.seq], -(1 << 30));
    length = int(min(int64_t(max(last, 0)), int64_t(a.b.width) * a.c.page_size));
    first = last - t.len / a.group;
  }
};

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
      w[2 * i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((mfma::f32x2{float(int8_t(x)), float(int8_t(x >> 8))}), mfma::bf16x2));
      w[2 * i + 1] =
          __builtin_bit_cast(uint32_t, __builtin_convertvector((mfma::f32x2{float(int8_t(x >> 16)), float(x >> 24)}), mfma::bf16x2));
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

// The chunk's form: bytes of workspace (0: it does not take such a call), and the call.
int64_t chunk_workspace(const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b);
int chunk_attention(const Paged& a, const mx_paged_desc* d, const mx_kv_cache* c, const mx_kv_batch* b, char* workspace,
                    hipStream_t s);

}  // namespace attn
}  // namespace mx
