// The paged cache as its kernels see it (mx_kv_cache.hip, mx_attention_paged.hip).
#pragma once

#include <type_traits>

#include "mx_internal.hpp"
#include "mx_sequences.hpp"

namespace mx {
namespace kv {

struct Cache {
  void *k, *v;
  float *ks, *vs;
  int pages, heads, page_size, dim;
};
struct Batch {
  Sequences seqs;
  const int32_t* lengths;
  const int32_t* table;
  int width;
};

// The page of places 16 group .. 16 group + 15 of a sequence (group >= 0) and the
// first one's place in it; -1 where the sequence has no such page in the cache.
__device__ __forceinline__ int page_of(const Cache& c, const Batch& b, int seq, int group, int& place) {
  const int per = c.page_size >> 4, entry = group / per;
  place = (group - entry * per) << 4;
  if (entry >= b.width) return -1;
  const int page = b.table[int64_t(seq) * b.width + entry];
  return page >= 0 && page < c.pages ? page : -1;
}

// Sizes, types and divisibility; then the pointers of a call that has work.
int check(const char* who, const mx_kv_cache* c, const mx_kv_batch* b);
int check_buffers(const char* who, const mx_kv_cache* c, const mx_kv_batch* b);
Cache cache_of(const mx_kv_cache* c);
Batch batch_of(const mx_kv_batch* b);

}  // namespace kv
}  // namespace mx
