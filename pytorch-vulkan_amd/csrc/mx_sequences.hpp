// Sequences packed behind each other, cut into tiles of U rows on the device.
//
// Only the host's grid needs a number of tiles, and the lengths are device data:
// sequence b's tiles start at base(b) = start(b) / U + EXTRA b (integer division),
// which leaves every sequence of n rows room for n / U + EXTRA of them and all of
// them within tokens / U + EXTRA sequences.  A workgroup finds its sequence from its
// tile's index by a search of 64 probes a step over base(), which ascends.
//
// Whatever `starts` holds, rows stay within 0 .. tokens and sequences within 0 ..
// count: entries that do not ascend give wrong rows, never an access out of range.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mx {

struct Sequences {
  const int32_t* starts;  // null: tokens / count rows each
  int tokens, count;
  int per = 1;  // rows a token

  __device__ __forceinline__ int start(int b) const {
    return (starts ? min(max(starts[b], 0), tokens) : int(int64_t(tokens) * b / count)) * per;
  }
};

struct SequenceTile {
  int seq, start, len;  // the sequence, its first row and its rows
  int base, index;      // its first tile, and this one's place among its tiles
};

// The most tiles that sequences of `tokens` rows have.
inline int64_t sequence_tiles(int64_t tokens, int64_t count, int unit, int extra = 1) {
  return tokens / unit + extra * count;
}

// The sequence of a tile, found by one wave (every lane gets it).  False where no
// sequence has this tile.
template <int U, int EXTRA = 1>
__device__ __forceinline__ bool locate(const Sequences& s, int tile, SequenceTile& t) {
  int lo = 0, n = s.count;
  const int lane = threadIdx.x & 63;
  while (n > 1) {
    const int step = (n + 63) >> 6, b = lo + lane * step;
    const bool below = lane * step < n && s.start(b) / U + EXTRA * b <= tile;
    const int c = max(1, __popcll(__ballot(below)));
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int first = s.start(lo), last = s.start(lo + 1);
  t.seq = lo;
  t.start = __builtin_amdgcn_readfirstlane(first);
  t.len = __builtin_amdgcn_readfirstlane(max(0, last - first));
  t.base = t.start / U + EXTRA * lo;
  t.index = tile - t.base;
  return t.index >= 0;
}

}  // namespace mx
