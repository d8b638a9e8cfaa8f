// The division of a sequence's keys and new tokens' rows for the key weights:
// blocks of kBlockKeys keys, and the rows that see a block in parts.  Counted
// on the host for the plan and on the device for the lengths that hold there.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

namespace klc {

constexpr int kBlockKeys = 256;  // of a workgroup
constexpr int kRowTile = 32;     // rows that it takes at once
constexpr int kLeastTiles = 8;   // of rows, for a part
constexpr int kPartRecord = 4;   // int32 of a part's record in the plan: sequence, part, parts, first joined one
// int32 of a listed workgroup, all that it needs but what may change between calls, so that it waits once for the plan:
// sequence, part, parts of the block, ListPlace, place of its sums, first new token's row of q, new tokens, least tiles of a part
constexpr int kListRecord = 8;

// Where a listed workgroup's block is: among the blocks with first tokens beside a window, or among the others that
// some row sees; `last` of them takes those behind it too.
struct ListPlace {
  bool head, last;
  int index;
  __host__ __device__ explicit ListPlace(int place) : head(place & 1), last(place & 2), index(place >> 2) {}
  static int32_t of(bool head, bool last, int64_t index) { return (int32_t)(index * 4 + (last ? 2 : 0) + (head ? 1 : 0)); }
};

// Of a sequence of n keys, the last `count` of them new (those below key 0 of a shorter one are none), groups of g heads.
struct KeyBlocks {
  int n, count, g, window, first;
  int base;         // the first new token's key
  int heads, low;   // blocks with first tokens, the first of the others that a row sees
  __host__ __device__ KeyBlocks(int n_, int count_, int g_, int window_, int first_)
      : n(n_), count(count_), g(g_), window(window_), first(first_), base(n_ - count_) {
    const int lowest = window > 0 && base >= window ? (base - window + 1) / kBlockKeys : 0;
    heads = window > 0 ? blocks(first < n ? first : n) : 0;
    low = lowest > heads ? lowest : heads;
  }
  static __host__ __device__ int blocks(int keys) { return (keys + kBlockKeys - 1) / kBlockKeys; }
  static __host__ __device__ int tiles(int rows) { return (rows + kRowTile - 1) / kRowTile; }
  __host__ __device__ int begin(bool head) const { return head ? 0 : low; }
  __host__ __device__ int end(bool head) const { return head ? heads : blocks(n); }
  // the rows that see one of a block's keys
  __host__ __device__ int row_begin(int block) const {
    const int tok = block * kBlockKeys - base;
    return (tok > 0 ? tok : 0) * g;
  }
  __host__ __device__ int row_end(int block) const {
    int last = count - 1;
    if (window > 0 && block >= heads) {  // its last key's last row
      const int key = block * kBlockKeys + kBlockKeys < n ? block * kBlockKeys + kBlockKeys - 1 : n - 1;
      const int64_t tok = (int64_t)key + window - 1 - base;
      if (tok < last) last = (int)tok;
    }
    return (last + 1) * g;
  }
  // a key that some row sees
  __host__ __device__ bool sees(int key) const { return window == 0 || key > base - window || key < first; }
  // the parts of a block's rows, of up to `most` with at least `least` tiles each, whatever the lengths are
  __host__ __device__ int parts(bool head, int most, int least) const {
    const int64_t reach = (int64_t)window + kBlockKeys - 1;
    const int tokens = window == 0 || head || count < reach ? count : (int)reach;
    const int p = (tiles(tokens * g) + least - 1) / least;
    return p < most ? p : most;
  }
  // rows of a part, in whole tiles if there are several
  static __host__ __device__ int per(int rows, int parts, int least) {
    if (parts == 1) return rows;
    const int share = (tiles(rows) + parts - 1) / parts;
    return (share > least ? share : least) * kRowTile;
  }
};

// The least tiles of rows of a part: in all eight workgroups a CU, if there are that many.  `starts` as the plan's.  A
// multiple of four, past which 18 tiles, 14 parts of 1,000 tokens over 4,000, take 69 us and 20, 13 parts, 67.
inline int least_tiles(const int32_t* starts, const int32_t* lengths, int64_t n_seq, int64_t g, int64_t n_kv, int64_t window,
                       int64_t first) {
  constexpr int kCus = 256;
  double work = 0.;
  for (int64_t s = 0; s < n_seq; ++s) {
    const int count = starts[s + 1] - starts[s];
    const KeyBlocks keys(lengths[s], count, (int)g, (int)window, (int)first);
    const double tiles = KeyBlocks::tiles((int)(count * g)), blocks = keys.end(false) - keys.low;
    // a row's blocks: behind a window its part of them and one more that it begins in; else the cached ones and half of the new
    const double past = keys.base / kBlockKeys;
    const double seen = window > 0 ? 1. + (double)window / kBlockKeys : past + (blocks - past + 1.) / 2.;
    work += std::max(tiles * std::min(seen, blocks), blocks) + tiles * keys.heads;
  }
  return std::max(kLeastTiles, 4 * (int)std::min(std::ceil(work * n_kv / (4 * 8 * kCus)), 1e8));
}

}  // namespace klc
