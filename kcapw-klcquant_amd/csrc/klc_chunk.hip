// Attention of chunks of new tokens over a paged KV cache (gfx950): of each
// sequence one new token or many, at the end of its keys, with a sliding
// window beside which some first tokens may stay visible.
//
//   out_i = sum_j 2^(c2 q_i . k_j - m) v_j / (sum_j 2^(c2 q_i . k_j - m) + 2^(s - m))
//
// over j <= i with j > i - window or j < first.  A row is (token, head of the
// group).  A plan made on the host, where the sizes are known, lists the
// workgroups' items, the longest first: up to 128 rows of one KV head of one
// sequence and a part of the keys that they see.
//   wide    more than 64 rows: 4 waves x 32 rows over one ring of tiles
//   pairs   33 to 64 rows, head sizes up to 64: the same of 2 pairs of waves,
//           of half the keys each, which join in LDS (past 64 wide has them)
//   narrow  up to 32 rows: each wave takes every fourth tile, K and V in turn
//           through LDS of its own, with no barrier, and the waves join there
// Rows whose keys are in parts leave float32 sums, which a second launch joins.
// As in the prompt's kernel a row with a NaN or infinity that may come from a
// value it must not see is computed again, token by token.
//
// What bounds it (64 heads over 8 of size 64 unless said): wide items by LDS
// reads, 96 bytes a clock of the 128 it has with three workgroups a CU, and
// the exponentials.  6,000 tokens over 2,000 beside 64 steps, 573 to 590 us by
// the card (0.84 PFLOP/s), 8,192 over none 631 (0.87; 64 rows a wave, half the
// reads at two waves a SIMD: 673 and 677 on one card), 2,000 over 16,000 of 32
// heads of size 128 576 to 588 (0.96).  Twelve suffixes of 50 to 100 over 2,000
// to 4,000 take 85, 464 items on 256 CUs, each waiting for itself.  Steps by
// HBM: 200 of a window of 1,024 and 4 first tokens 93 us (4.6 TB/s), 256 of
// 2,000 156 (5.1); eight of 700 keys take 12, the chain of item, length, page
// numbers and six tiles a wave.
#include <math.h>

#include <algorithm>
#include <queue>
#include <vector>

#include "klc_key_blocks.h"
#include "klc_paged_tiles.h"

namespace klc {
namespace {

constexpr int kWideRows = 32 * kWaves;
constexpr int kNarrowRows = 32;
// most rows of an item whose waves work in pairs; head sizes past 64 have no tiles of 64 keys for them
__host__ __device__ constexpr int pair_rows(int dim) { return dim <= 64 ? 64 : kNarrowRows; }
constexpr int kJoinRows = 16;    // of one workgroup
constexpr int kRecord = 8;       // int32 of an item and of a join
// LDS of a workgroup: three fit a CU, past head size 64 two (of size 64, with the loads of the time, 6,000 tokens over 2,000
// beside 64 steps took 700 us with two and 647 with three)
template <int DP>
constexpr int kChunkLds = (DP == 64 ? 48 : 64) * 1024;

struct ChunkArgs {
  const uint16_t* q;                  // bfloat16 [tokens] rows
  const uint16_t *k_pages, *v_pages;  // [n_pages][page][n_kv][d]
  const int32_t *tables, *lengths;    // [n_seq][width], [n_seq]
  const int32_t *items, *joins;
  const uint16_t* sinks;
  uint16_t* out;                      // [tokens][n_heads][d]
  float* lse;                         // [tokens][n_heads] or NULL
  float* part_o;                      // [n_kv][part_rows][d]
  float4* part_ml;                    // [n_kv][part_rows]: maximum, sum, sum of the unrounded
  int64_t q_stride, part_rows;
  int n_heads, n_kv, d, n_pages, page_log2, width, window, first;
  float c2;
};

// An item of the plan, the same for all threads of a workgroup.
struct ChunkItem {
  int seq, begin, count;  // the sequence, its first new token's row of q, its new tokens
  int row0, rows;         // of it
  int split, splits;      // part of the keys
  int part;               // row of the parts' arrays of the first part's first row
};

__device__ __forceinline__ bool sees(const ChunkArgs& a, int pos, int key) {
  return key <= pos && (a.window == 0 || key > pos - a.window || key < a.first);
}

// The keys that rows at positions p_lo..p_hi see, as a list of tiles of KT:
// those of the first tokens, then those of the window.  Both ranges are
// widened to whole pieces of 16 keys, which never span two pages.
template <int KT>
struct Span {
  int head_end, low, high;        // keys below head_end and from low to high
  int head_tiles, low_tile, tiles;
  __device__ __forceinline__ Span(const ChunkArgs& a, int p_lo, int p_hi) {
    low = a.window > 0 ? max(0, p_lo - a.window + 1) & ~15 : 0;
    head_end = (min(a.first, max(p_hi, 0)) + 15) & ~15;
    if (head_end >= low) head_end = low = 0;
    high = p_hi;
    head_tiles = (head_end + KT - 1) / KT;
    low_tile = max(low / KT, head_tiles);
    tiles = p_hi < 0 ? 0 : head_tiles + p_hi / KT + 1 - low_tile;
  }
  __device__ __forceinline__ int base(int j) const { return (j < head_tiles ? j : j - head_tiles + low_tile) * KT; }
  // of the tile behind the one at `tile`
  __device__ __forceinline__ int next(int tile) const { return tile + KT == head_tiles * KT ? low_tile * KT : tile + KT; }
  // the tile with key `high` or a lower one of a row
  __device__ __forceinline__ int tile_of(int key) const {
    const int t = key / KT;
    return t >= low_tile ? t - low_tile + head_tiles : t;
  }
  // all keys of the tile that starts at `tile` are in the ranges
  __device__ __forceinline__ bool whole(int tile) const {
    return tile < head_tiles * KT ? tile + KT <= head_end : tile >= low && tile + KT - 1 <= high;
  }
  // the key whose row stands for `key` of the tile that starts at `tile`
  __device__ __forceinline__ auto at(int tile) const {
    const int gap = tile < head_tiles * KT ? head_end - 1 : low, from = low, to = high, head = head_end;
    return [=](int key) { return key >= from ? min(key, to) : key < head ? key : gap; };
  }
};

// A lane's row: `from` + lane, or the item's last one.  Worked out where it is needed: held from the start to the end
// it would spill.
struct ChunkRow {
  int row, tok, head;
  int64_t out;  // of it, in out and lse
  __device__ __forceinline__ ChunkRow(const ChunkArgs& a, const ChunkItem& it, int kvh, int from) {
    int lane = threadIdx.x % 32;
    asm volatile("" : "+v"(lane));
    const int g = a.n_heads / a.n_kv;
    row = min(from + lane, it.row0 + it.rows - 1);
    tok = row / g;
    head = kvh * g + row - tok * g;
    out = (int64_t)(it.begin + tok) * a.n_heads + head;
  }
};

template <int DP, bool kF16, bool kFull, bool kLse>
struct ChunkRows {
  using F = AttnWave<DP, kF16, kFull, 1, kKeys>;
  static constexpr int kQuads = 4 * F::kDimBlocks;
  F f;
  float c2, plain;  // plain: this half's sum of the unrounded exponentials
  int pos;          // of the lane's row

  // rows `from` + lane on
  __device__ __forceinline__ void begin(const ChunkArgs& a, const ChunkItem& it, int kvh, int base, int from, lds_u8 ring) {
    const ChunkRow row(a, it, kvh, from);
    f.init(ring, a.d);
    plain = 0.f;
    pos = base + row.tok;
    load_query<F>(f.q[0], a.q + (it.begin + row.tok) * a.q_stride + (int64_t)row.head * a.d, a.d);
  }
  __device__ __forceinline__ void convert(const ChunkArgs& a) { c2 = a.c2 * convert_query<F, kF16>(f.q[0]); }
  __device__ __forceinline__ void mask(const ChunkArgs& a, int k0, f32x16_t (&s)[1][1]) const {
    // of the keys from the lane's first one on: up to its row in the window, or below the first tokens' end
    const int from = k0 + 4 * ((int)(threadIdx.x % kWave) / 32), rel = pos - from, head = min(a.first, pos + 1) - from;
    const uint32_t reach = a.window > 0 ? a.window : 0x7fffffffu;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int off = 8 * (e / 4) + e % 4;
      if (!((uint32_t)(rel - off) < reach || off < head)) s[0][0][e] = -INFINITY;
    }
  }
  __device__ __forceinline__ void raise(const f32x16_t (&s)[1]) {
    const float before = f.m[0];
    f.raise(0, s, c2);
    if constexpr (kLse) plain *= __builtin_amdgcn_exp2f(before == f.m[0] ? 0.f : before - f.m[0]);
  }
  __device__ __forceinline__ void weigh(const f32x16_t (&s)[1], u32x4_t (&p)[2]) {
    if constexpr (kLse)
      f.template weigh<true>(0, s, c2, p, &plain);
    else
      f.weigh(0, s, c2, p);
  }
  __device__ __forceinline__ bool odd() const {
    bool x = false;
#pragma unroll
    for (int db = 0; db < F::kDimBlocks; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) x |= !(fabsf(f.o[0][db][e]) < INFINITY);
    return x;
  }
};

// What a row's parts come to: the factor of its sums, and the log of its normaliser.
struct Norm {
  float inv, lse;
};
// m, l, plain: maximum, sum and unrounded sum of all its keys; none: it sees no key
__device__ __forceinline__ Norm normalise(const ChunkArgs& a, int head, float m, float l, float plain, bool none) {
  const float s = a.sinks != nullptr ? sink_log2(a.sinks[head]) : -INFINITY;
  const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
  const float x = __builtin_amdgcn_exp2f(m - base), y = __builtin_amdgcn_exp2f(s - base);
  // 0 / 0 where a row's scores and its sink are all -inf: NaN, as their softmax; without a key zeros
  return {none ? 0.f : x / fmaf(l, x, y), (base + __builtin_amdgcn_logf(fmaf(plain, x, y))) * 0.69314718055994530942f};
}

// Tile by tile for the rows of one token, with V cleared where that token does
// not see it, so that no NaN or infinity comes from there (0 * inf).  The
// wave works alone, in `lds`, on tiles from + i * step of the list, of each on
// the keys from `piece` on, 32 of every piece_step.
template <int DP, bool kF16, bool kFull, bool kLse, int KT>
__device__ __forceinline__ void careful_token(const ChunkArgs& a, const ChunkItem& it, ChunkRows<DP, kF16, kFull, kLse>& r,
                                              const Span<KT>& span, int kvh, int base, int row0, int tok, int from, int to,
                                              int step, int piece, int piece_step, lds_u8 lds) {
  using F = typename ChunkRows<DP, kF16, kFull, kLse>::F;
  typedef __attribute__((address_space(3))) u32x4_t* lds_u32x4;
  const int lane = threadIdx.x % kWave, pos = base + tok;
  const int32_t* table = a.tables + (int64_t)it.seq * a.width;
  r.begin(a, it, kvh, base, row0, lds);
  r.convert(a);
  PageLoads<ChunkArgs, F, kKeys, F::kDmas, 1> pages(a, 0, kvh);
  if (from < to) pages.hold(table, span.at(span.base(from))(span.base(from)) >> a.page_log2, a.width);
  for (int j = from; j < to; j += step)
    for (int k0 = span.base(j) + piece; k0 < span.base(j) + KT; k0 += piece_step) {
      if (k0 > pos) break;
      pages.load(k0, span.at(span.base(j)), lds, lds + F::kMatBytes);
      tile_wait<0, false>();
      for (int i = lane; i < kKeys * F::kChunks; i += kWave)
        if (!sees(a, pos, k0 + i / F::kChunks)) *(lds_u32x4)(lds + F::kMatBytes + i * 16) = u32x4_t{0, 0, 0, 0};
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      f32x16_t s[1][1];
      r.f.scores(0, s);
      r.mask(a, k0, s);
      r.raise(s[0]);
      u32x4_t p[1][2];
      r.weigh(s[0], p[0]);
      r.f.values(F::kMatBytes, p);
      tile_wait<63, false>();  // the tile has been read
    }
}

// Rows of an item in blocks of 32: a wave each, or with kSplit 2 a pair of
// waves each, of which one takes the tiles' first 32 keys and one the others.
template <int DP, bool kF16, bool kFull, bool kLse, int kSplit>
__device__ __forceinline__ void wide_part(const ChunkArgs& a, const ChunkItem& it, int kvh, int n, bool wrong, lds_u8 ring) {
  constexpr int KT = kSharedTile<DP>, kSub = KT / kKeys;
  using R = ChunkRows<DP, kF16, kFull, kLse>;
  using F = typename R::F;
  constexpr int kMat = kSub * F::kMatBytes, kStage = 2 * kMat, kRing = kChunkLds<DP> / kStage;
  constexpr int kDmas = kSub * F::kDmas / kWaves;  // of K, and of V, a wave and tile
  static_assert(kRing >= 3 && kSub * F::kDmas % kWaves == 0 && kSub >= kSplit, "");
  const int g = a.n_heads / a.n_kv, lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int base = n - it.count, last = it.row0 + it.rows - 1, w_row = it.row0 + 32 * (wave / kSplit), part = wave % kSplit;
  const bool w_live = w_row <= last;
  const Span<KT> span(a, base + it.row0 / g, base + last / g);
  const int per = (span.tiles + it.splits - 1) / it.splits, t0 = min(it.split * per, span.tiles), tiles = min(per, span.tiles - t0);
  // the wave's first and last position, its last tile, and whether it sees that tile's second half
  const int w_lo = base + min(w_row, last) / g, w_hi = base + min(w_row + 31, last) / g;
  const int w_last = w_live && w_hi >= 0 ? min(span.tile_of(w_hi) - t0, tiles - 1) : -1;
  const bool w_both = t0 + w_last < span.tile_of(w_hi) || w_hi % KT >= kKeys;
  // pieces of keys from `plain_from` to `plain_to` are seen by all of its rows
  const int plain_from = a.window > 0 ? w_hi - a.window + 1 : 0, plain_to = w_lo - kKeys + 1;
  const int32_t* table = a.tables + (int64_t)it.seq * a.width;
  R r;
  r.begin(a, it, kvh, base, w_row, ring);
  PageLoads<ChunkArgs, F, KT, kDmas, kWaves> pages(a, wave, kvh);
  pages.prepare_whole();
  if (tiles > 0) pages.hold(table, span.at(span.base(t0))(span.base(t0)) >> a.page_log2, a.width);
  settle_query<F>(r.f.q[0]);
  int load_key = span.base(t0);  // of the tile to be loaded next
  auto load = [&](int j, int slot) {
    if (j >= tiles) return;
    if (span.whole(load_key))
      pages.load_whole(load_key, ring + slot, ring + slot + kMat);
    else
      pages.load(load_key, span.at(load_key), ring + slot, ring + slot + kMat);
    load_key = span.next(load_key);
  };
#pragma unroll
  for (int j = 0; j < kRing - 1; ++j) load(j, j * kStage);
  r.convert(a);
  // tile j is there for all waves, `ahead` later ones may be in flight
  auto arrive = [&](int j, auto ahead) {
    if (j + decltype(ahead)::value < tiles)
      tile_wait<2 * kDmas * decltype(ahead)::value, true>();
    else
      tile_wait<0, true>();
  };
  auto settle = [&](int k0, f32x16_t (&s)[1][1]) {
    if (k0 < plain_from || k0 > plain_to) r.mask(a, k0, s);
    r.raise(s[0]);
  };
  // the values of the keys at `here`, whose settled scores are s, and the scores of those at `there`
  auto step = [&](int here, f32x16_t (&s)[1][1], int there, f32x16_t (&next)[1][1]) {
    u32x4_t p[1][2];
    r.f.scores(there, next);
    r.weigh(s[0], p[0]);
    r.f.values(here + kMat, p);
  };
  int j = 0, cur = 0, fill = (kRing - 1) * kStage, key = span.base(t0);
  auto behind = [&](int slot) { return slot + kStage == kRing * kStage ? 0 : slot + kStage; };
  // tile j + 1 is there from here on, every wave is done with tile j - 1
  auto advance = [&]() {
    arrive(j + 1, Count<kRing - 3>{});
    load(j + kRing - 1, fill);
    fill = cur;
  };
  f32x16_t sa[1][1], sb[1][1];
  arrive(0, Count<kRing - 2>{});
  if (w_last >= 0) {
    const int mine = part * F::kMatBytes, ahead = part * kKeys;  // of a pair's wave
    r.f.scores(mine, sa);
    settle(key + ahead, sa);
    if constexpr (kSub == 2 && kSplit == 1) {
      for (; j <= w_last; ++j) {
        const int here = cur, there = behind(cur), next_key = span.next(key);
        step(here, sa, here + F::kMatBytes, sb);
        const bool both = j < w_last || w_both;
        if (both) settle(key + kKeys, sb);
        advance();
        if (both) step(here + F::kMatBytes, sb, there, sa);  // past the last tile: scores of nothing, not used
        if (j < w_last) settle(next_key, sa);
        cur = there, key = next_key;
      }
    } else {
      auto tile = [&](f32x16_t (&s)[1][1], f32x16_t (&next)[1][1]) {
        const int here = cur, there = behind(cur);
        advance();
        step(here + mine, s, there + mine, next);
        key = span.next(key);
        if (j < w_last) settle(key + ahead, next);
        cur = there;
        ++j;
      };
      while (j <= w_last) {
        tile(sa, sb);
        if (j <= w_last) tile(sb, sa);
      }
    }
  }
  for (; j < tiles; ++j) {
    advance();
    cur = behind(cur);
  }

  const bool bad = __syncthreads_or(pages.bad) || wrong;
  const lds_u8 mine = ring + wave * (kChunkLds<DP> / kWaves);
  // all rows, or those of token `only`; of a pair every wave comes here
  auto finish = [&](int only) {
    if constexpr (kSplit == 2) {
      // the second wave's sums to the first, lane by lane: [pair][quad or (maximum, sums)][lane]
      typedef __attribute__((address_space(3))) f32x4_t* lds_f32x4;
      static_assert(kWaves / 2 * (R::kQuads + 1) * kWave * 16 <= kChunkLds<DP>, "");
      const lds_f32x4 sums = (lds_f32x4)ring + wave / 2 * (R::kQuads + 1) * kWave + lane;
      __syncthreads();
      if (part == 1) {
#pragma unroll
        for (int i = 0; i < R::kQuads; ++i) sums[i * kWave] = quad(r.f, i);
        sums[R::kQuads * kWave] = f32x4_t{r.f.m[0], r.f.l[0], r.plain, 0.f};
      }
      __syncthreads();
      if (part == 1) return;
      const f32x4_t other = sums[R::kQuads * kWave];
      const float top = fmaxf(r.f.m[0], other.x), ref = top == -INFINITY ? 0.f : top;
      const float x = __builtin_amdgcn_exp2f(r.f.m[0] - ref), y = __builtin_amdgcn_exp2f(other.x - ref);
      r.f.m[0] = top;
      r.f.l[0] = fmaf(r.f.l[0], x, other.y * y);
      r.plain = fmaf(r.plain, x, other.z * y);
#pragma unroll
      for (int i = 0; i < R::kQuads; ++i) {
        const f32x4_t o = sums[i * kWave];
#pragma unroll
        for (int e = 0; e < 4; ++e) r.f.o[0][i / 4][i % 4 * 4 + e] = fmaf(r.f.o[0][i / 4][i % 4 * 4 + e], x, o[e] * y);
      }
    }
    const ChunkRow row(a, it, kvh, w_row);
    const float sum = bad ? __uint_as_float(0x7fc00000u) : add_halves(r.f.l[0]), plain = kLse ? add_halves(r.plain) : 0.f;
    const bool live = w_row + lane % 32 <= last && (only < 0 || row.tok == only);
    if (it.splits > 1) {
      const int64_t at = (int64_t)kvh * a.part_rows + it.part + it.split * it.rows + (row.row - it.row0);
      if (live && lane < 32) a.part_ml[at] = make_float4(r.f.m[0], sum, plain, 0.f);
      // the wave's sums through LDS, so that they leave as whole rows: 16 bytes at (row, chunk ^ row) of [32][DP]
      typedef __attribute__((address_space(3))) f32x4_t* lds_f32x4;
      constexpr int kRowQuads = DP / 4;
      const lds_f32x4 out = (lds_f32x4)mine;
#pragma unroll
      for (int i = 0; i < R::kQuads; ++i) out[lane % 32 * kRowQuads + ((quad_dim(i) / 4) ^ (lane % 8))] = quad(r.f, i);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      float* dst = a.part_o + ((int64_t)kvh * a.part_rows + it.part + it.split * it.rows + (w_row - it.row0)) * a.d;
#pragma unroll 4
      for (int i = 0; i < 32 * kRowQuads / kWave; ++i) {
        const int x = (i * kWave + lane) / kRowQuads, c = lane % kRowQuads;
        if (w_row + x <= last && 4 * c < a.d && (only < 0 || (w_row + x) / g == only))
          *reinterpret_cast<f32x4_t*>(dst + x * a.d + 4 * c) = out[x * kRowQuads + (c ^ (x % 8))];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      return;
    }
    const Norm norm = normalise(a, row.head, r.f.m[0], sum, bad ? sum : plain, base + row.tok < 0 && !bad);
    if (kLse && live && lane < 32) a.lse[row.out] = norm.lse;
    uint16_t* dst = a.out + row.out * a.d + 8 * (lane / 32);
#pragma unroll
    for (int db = 0; db < F::kDimBlocks; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 8) {
        // the lane has dims 4 (lane / 32) + 0..3 and 8 more of 16; the halves trade, so that each has 8 in a row
        uint32_t w[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            w[i][x] = pack2<false>(r.f.o[0][db][e + 4 * i + 2 * x] * norm.inv, r.f.o[0][db][e + 4 * i + 2 * x + 1] * norm.inv);
        const auto lo = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        const int at = 32 * db + 2 * e;
        if (!live || (!kFull && at + 8 * (lane / 32) >= a.d)) continue;
        *reinterpret_cast<u32x4_t*>(dst + at) = u32x4_t{lo[0], hi[0], lo[1], hi[1]};
      }
  };
  // one `finish` for both: with two of them head size 128 spills
  const bool careful = __syncthreads_or(r.odd()) && !bad;
  if (kSplit == 1 && !w_live) return;
  const int tok0 = (kSplit == 2 ? it.row0 : w_row) / g, tok1 = (kSplit == 2 ? last : min(w_row + 31, last)) / g;
#pragma unroll 1
  for (int tok = careful ? tok0 : -1; tok <= (careful ? tok1 : -1); ++tok) {
    if (careful)
      careful_token<DP, kF16, kFull, kLse, KT>(a, it, r, span, kvh, base, w_row, tok, t0, t0 + tiles, 1, part * kKeys,
                                               kSplit * kKeys, mine);
    finish(tok);
    if (kSplit == 2 && careful) __syncthreads();  // the sums have been read
  }
}

template <int DP, bool kF16, bool kFull, bool kLse>
__device__ __forceinline__ void narrow_part(const ChunkArgs& a, const ChunkItem& it, int kvh, int n, bool wrong, lds_u8 lds,
                                            float4 (&wave_ml)[kWaves][kNarrowRows]) {
  using R = ChunkRows<DP, kF16, kFull, kLse>;
  using F = typename R::F;
  constexpr int KT = kKeys, kQuads = R::kQuads;
  static_assert(kChunkLds<DP> / kWaves / F::kStage == 1, "one tile a wave: K and V take turns");
  const int g = a.n_heads / a.n_kv, lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int base = n - it.count, last = it.row0 + it.rows - 1;
  const int p_lo = base + it.row0 / g, p_hi = base + last / g;
  const int32_t* table = a.tables + (int64_t)it.seq * a.width;
  const lds_u8 tile = lds + wave * F::kStage;
  R r;
  r.begin(a, it, kvh, base, it.row0, tile);
  PageLoads<ChunkArgs, F, KT, F::kDmas, 1> pages(a, 0, kvh);
  pages.prepare_whole();
  const Span<KT> span(a, p_lo, p_hi);
  const int per = (span.tiles + it.splits - 1) / it.splits, t0 = min(it.split * per, span.tiles), end = min(t0 + per, span.tiles);
  const int first = t0 + wave;
  if (first < end) pages.hold(table, span.at(span.base(first))(span.base(first)) >> a.page_log2, a.width);
  settle_query<F>(r.f.q[0]);
  auto load = [&](auto key, int j) {  // K of a tile, or V
    constexpr bool kKey = decltype(key)::value;
    const int at = span.base(j);
    if (span.whole(at))
      pages.template load_whole<kKey, !kKey>(at, tile, tile + F::kMatBytes);
    else
      pages.template load<kKey, !kKey>(at, span.at(at), tile, tile + F::kMatBytes);
  };
  if (first < end) {
    load(Count<true>{}, first);
    load(Count<false>{}, first);
  }
  r.convert(a);
  for (int j = first; j < end; j += kWaves) {
    const bool refill = j + kWaves < end;
    tile_wait<F::kDmas, false>();  // K is there, V may be in flight
    const int k0 = span.base(j);
    f32x16_t s[1][1];
    r.f.scores(0, s);
    if (refill) {
      tile_wait<63, false>();  // K has been read
      load(Count<true>{}, j + kWaves);
    }
    if (k0 + kKeys - 1 > p_lo || (a.window > 0 && k0 <= p_hi - a.window)) r.mask(a, k0, s);
    r.raise(s[0]);
    u32x4_t p[1][2];
    r.weigh(s[0], p[0]);
    if (refill)
      tile_wait<F::kDmas, false>();
    else
      tile_wait<0, false>();
    r.f.values(F::kMatBytes, p);
    if (refill) {
      tile_wait<63, false>();  // V has been read
      load(Count<false>{}, j + kWaves);
    }
  }

  const bool bad = __syncthreads_or(pages.bad) || wrong;
  // all rows, or those of token `only`; every wave comes here
  auto finish = [&](int only) {
    // the waves' sums, lane by lane: [wave][quad][lane]
    typedef __attribute__((address_space(3))) f32x4_t* lds_f32x4;
    const lds_f32x4 sums = (lds_f32x4)lds;
    const ChunkRow row(a, it, kvh, it.row0);
    const float sum = add_halves(r.f.l[0]), plain = kLse ? add_halves(r.plain) : 0.f;
    const bool live = lane % 32 < it.rows;
    __syncthreads();
    if (live) {
      if (lane < 32) wave_ml[wave][lane] = make_float4(r.f.m[0], sum, plain, 0.f);
#pragma unroll
      for (int i = 0; i < kQuads; ++i) sums[(wave * kQuads + i) * kWave + lane] = quad(r.f, i);
    }
    __syncthreads();
    if (live && (only < 0 || row.tok == only)) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_ml[w][lane % 32].x);
      const float ref = top == -INFINITY ? 0.f : top;
      float x[kWaves], l = bad ? __uint_as_float(0x7fc00000u) : 0.f, all = l;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float4 ml = wave_ml[w][lane % 32];
        x[w] = __builtin_amdgcn_exp2f(ml.x - ref);
        l = fmaf(x[w], ml.y, l);
        all = fmaf(x[w], ml.z, all);
      }
      const int64_t at = (int64_t)kvh * a.part_rows + it.part + it.split * it.rows + (row.row - it.row0);
      const Norm norm = normalise(a, row.head, top, l, all, base + row.tok < 0 && !bad);
      if (wave == 0 && lane < 32) {
        if (it.splits > 1)
          a.part_ml[at] = make_float4(top, l, all, 0.f);
        else if (kLse)
          a.lse[row.out] = norm.lse;
      }
#pragma unroll
      for (int n = 0; n < kQuads / kWaves; ++n) {
        const int i = wave + n * kWaves;
        f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) o += x[w] * sums[(w * kQuads + i) * kWave + lane];
        if (!kFull && quad_dim(i) >= a.d) continue;
        if (it.splits > 1)
          *reinterpret_cast<f32x4_t*>(a.part_o + at * a.d + quad_dim(i)) = o;
        else
          *reinterpret_cast<u32x2_t*>(a.out + row.out * a.d + quad_dim(i)) =
              u32x2_t{pack2<false>(o.x * norm.inv, o.y * norm.inv), pack2<false>(o.z * norm.inv, o.w * norm.inv)};
      }
    }
  };
  const bool careful = __syncthreads_or(r.odd()) && !bad;
#pragma unroll 1
  for (int tok = careful ? it.row0 / g : -1; tok <= (careful ? last / g : -1); ++tok) {
    if (careful) careful_token<DP, kF16, kFull, kLse, KT>(a, it, r, span, kvh, base, it.row0, tok, first, end, kWaves, 0,
                                                          kKeys, lds + wave * (kChunkLds<DP> / kWaves));
    finish(tok);
    __syncthreads();  // the sums have been read
  }
}

template <int DP, bool kF16, bool kFull, bool kLse>
__global__ __launch_bounds__(kWave * kWaves, DP == 64 ? 3 : 2) void chunk_attention_kernel(ChunkArgs a) {
  __shared__ __align__(1024) uint8_t lds[kChunkLds<DP>];
  __shared__ float4 wave_ml[kWaves][kNarrowRows];
  const int kvh = blockIdx.x % a.n_kv;
  const int32_t* rec = a.items + (int64_t)(blockIdx.x / a.n_kv) * kRecord;
  const ChunkItem it{table_at(rec, 0), table_at(rec, 1), table_at(rec, 2), table_at(rec, 3),
                     table_at(rec, 4), table_at(rec, 5), table_at(rec, 6), table_at(rec, 7)};
  const int asked = table_at(a.lengths, it.seq);
  const int64_t room = (int64_t)a.width << a.page_log2;
  const int n = (int)min((int64_t)max(asked, 0), room);
  if (it.rows > pair_rows(DP))
    wide_part<DP, kF16, kFull, kLse, 1>(a, it, kvh, n, asked > room, (lds_u8)lds);
  else if (DP == 64 && it.rows > kNarrowRows)
    wide_part<DP, kF16, kFull, kLse, DP == 64 ? 2 : 1>(a, it, kvh, n, asked > room, (lds_u8)lds);
  else
    narrow_part<DP, kF16, kFull, kLse>(a, it, kvh, n, asked > room, (lds_u8)lds, wave_ml);
}

// out[row] = sum over its parts: a workgroup has up to kJoinRows rows of a KV
// head, a wave every fourth of them; lanes take 4 dims each, and the groups of
// lanes that this leaves take parts in turn.
__global__ __launch_bounds__(kWave * kWaves) void chunk_join_kernel(ChunkArgs a) {
  const int kvh = blockIdx.x % a.n_kv, g = a.n_heads / a.n_kv;
  const int32_t* rec = a.joins + (int64_t)(blockIdx.x / a.n_kv) * kRecord;
  // sequence, its first new token's row of q, its new tokens, first row, rows, parts, first part's row, rows of a part
  const int seq = table_at(rec, 0), begin = table_at(rec, 1), count = table_at(rec, 2), row0 = table_at(rec, 3),
            rows = table_at(rec, 4), parts = table_at(rec, 5), part = table_at(rec, 6), stride = table_at(rec, 7);
  const int base = min(max(table_at(a.lengths, seq), 0), (int)min((int64_t)a.width << a.page_log2, (int64_t)0x7fffffff)) - count;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int lanes = a.d <= 32 ? 8 : a.d <= 64 ? 16 : 32, groups = kWave / lanes, grp = lane / lanes;
  const int dim = min(4 * (lane % lanes), a.d - 4);
  for (int i = wave; i < rows; i += kWaves) {
    const int row = row0 + i, tok = row / g, head = kvh * g + row - tok * g;
    const int64_t at = (int64_t)kvh * a.part_rows + part + i;
    float top = -INFINITY;
    for (int s = lane; s < parts; s += kWave) top = fmaxf(top, a.part_ml[at + (int64_t)s * stride].x);
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    const float ref = top == -INFINITY ? 0.f : top;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f, all = 0.f;
    constexpr int kAhead = 4;
    for (int s0 = grp; s0 < parts; s0 += kAhead * groups) {
      float4 y[kAhead], x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t p = at + (int64_t)min(s0 + k * groups, parts - 1) * stride;
        y[k] = *reinterpret_cast<const float4*>(a.part_o + p * a.d + dim);
        x[k] = a.part_ml[p];
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (s0 + k * groups >= parts) break;
        const float w = __builtin_amdgcn_exp2f(x[k].x - ref);
        l = fmaf(w, x[k].y, l);
        all = fmaf(w, x[k].z, all);
        o.x = fmaf(w, y[k].x, o.x), o.y = fmaf(w, y[k].y, o.y), o.z = fmaf(w, y[k].z, o.z), o.w = fmaf(w, y[k].w, o.w);
      }
    }
    for (int off = lanes; off < kWave; off <<= 1) {
      l += __shfl_xor(l, off), all += __shfl_xor(all, off);
      o.x += __shfl_xor(o.x, off), o.y += __shfl_xor(o.y, off), o.z += __shfl_xor(o.z, off), o.w += __shfl_xor(o.w, off);
    }
    const bool bad = l != l;
    const Norm norm = normalise(a, head, top, l, bad ? l : all, base + tok < 0 && !bad);
    const int64_t out = (int64_t)(begin + tok) * a.n_heads + head;
    if (lane == 0 && a.lse != nullptr) a.lse[out] = norm.lse;
    if (lane < a.d / 4)
      *reinterpret_cast<u32x2_t*>(a.out + out * a.d + dim) =
          u32x2_t{pack2<false>(o.x * norm.inv, o.y * norm.inv), pack2<false>(o.z * norm.inv, o.w * norm.inv)};
  }
}

// ---- the plan -------------------------------------------------------------------------

constexpr int kCus = 256;

// Rows of a sequence that share their tiles of keys, and the keys they see in
// tiles of kKeys.
struct RowTile {
  int seq, row0, rows, tiles, splits;
  // Microseconds, measured: of a workgroup by itself, and of what it takes from a CU that has others to run.  A wide
  // tile's throughput goes by its blocks of 32 rows, a narrow one's by its bytes from memory; a part's sums go out and
  // in (128 rows of size 64: 64 KB, 3.3 us of a CU's share).
  double alone(int64_t dim) const {
    const double tile = rows <= kNarrowRows ? .25 : dim <= 64 ? .62 : .75;
    return 4. + tile * ((tiles + splits - 1) / splits);
  }
  double shared(int64_t dim) const {
    const double tile = rows <= kNarrowRows ? .4 * dim / 64 : (dim <= 64 ? .33 : .55) * ((rows + 31) / 32) / 4;
    return 1.7 + tile * ((tiles + splits - 1) / splits) + (splits > 1 ? rows * dim / 2500. : 0.);
  }
};

// Of a sequence's rows the part that one workgroup of the key weights' kernel
// takes by a block of keys.
struct WeightPart {
  int seq, part, parts, offset;  // offset: of the first part among those that are joined
};

struct ChunkPlan {
  std::vector<int32_t> starts;
  std::vector<RowTile> tiles;
  int64_t items = 0, joins = 0, part_rows = 0;
  std::vector<WeightPart> weights;
  int64_t weight_joins = 0, weight_parts = 0;
};

int64_t span_tiles(int64_t p_lo, int64_t p_hi, int64_t window, int64_t first) {
  int64_t low = window > 0 ? std::max<int64_t>(0, p_lo - window + 1) & ~15 : 0, head = (std::min(first, std::max<int64_t>(p_hi, 0)) + 15) & ~15;
  if (head >= low) head = low = 0;
  const int64_t head_tiles = (head + kKeys - 1) / kKeys;
  return p_hi < 0 ? 0 : head_tiles + p_hi / kKeys + 1 - std::max(low / kKeys, head_tiles);
}

// When the last of `servers` is done, if the longest items go first.
double makespan(std::vector<double>& costs, int64_t servers) {
  std::sort(costs.begin(), costs.end(), std::greater<double>());
  std::priority_queue<double, std::vector<double>, std::greater<double>> ends;
  double last = 0.;
  for (double c : costs) {
    double at = 0.;
    if ((int64_t)ends.size() >= servers) at = ends.top(), ends.pop();
    ends.push(at + c);
    last = std::max(last, at + c);
  }
  return last;
}

// How long a plan takes, on one KV head's share of the chip.  It only has to tell cuts apart: two workgroups a CU count as
// side by side for every head size, and what the third of sizes up to 64 takes from them is in RowTile::shared.
double duration(const std::vector<RowTile>& tiles, int64_t n_kv, int64_t dim) {
  std::vector<double> alone, shared;
  bool joins = false;
  for (const RowTile& t : tiles) {
    alone.insert(alone.end(), t.splits, t.alone(dim));
    shared.insert(shared.end(), t.splits, t.shared(dim));
    joins |= t.splits > 1;
  }
  const int64_t cus = std::max<int64_t>(1, kCus / n_kv);
  return std::max(makespan(alone, 2 * cus), makespan(shared, cus)) + (joins ? 5. : 0.);  // the join's launch
}

// Tiles' keys in parts of about `most` tiles, or whole (0).
void split_tiles(std::vector<RowTile>& tiles, int64_t most) {
  for (RowTile& t : tiles) t.splits = most > 0 ? (int)std::max<int64_t>(1, (t.tiles + most / 2) / most) : 1;
}

ChunkPlan chunk_plan(const int32_t* counts, const int32_t* lengths, int64_t n_seq, int64_t n_heads, int64_t n_kv, int64_t dim,
                     int64_t window, int64_t first) {
  ChunkPlan p;
  const int64_t g = n_heads / n_kv;
  int64_t begin = 0, longest = 0;
  for (int64_t s = 0; s < n_seq; ++s) {
    p.starts.push_back((int32_t)begin);
    const int64_t rows = counts[s] * g, past = (int64_t)lengths[s] - counts[s];
    for (int64_t row0 = 0; row0 < rows; row0 += kWideRows) {
      const int64_t n = std::min<int64_t>(kWideRows, rows - row0);
      const int64_t tiles = span_tiles(past + row0 / g, past + (row0 + n - 1) / g, window, first);
      p.tiles.push_back({(int)s, (int)row0, (int)n, (int)tiles, 1});
      longest = std::max(longest, tiles);
    }
    begin += counts[s];
  }
  p.starts.push_back((int32_t)begin);
  // Keys in parts where that ends sooner: up to four workgroups a CU in all, or of many items the few longest (127 steps
  // of 200 to 1,000 keys and one of 32,000 take 258 us with that one whole and 60 with it in parts).
  auto count = [&] {
    int64_t n = 0;
    for (const RowTile& t : p.tiles) n += t.splits;
    return n * n_kv;
  };
  const int64_t whole = count();
  if (whole <= 16 * kCus) {
    double best = duration(p.tiles, n_kv, dim);
    int64_t most = 0;
    for (int64_t m = longest * 2 / 3; m >= 12; m = m * 3 / 4) {
      split_tiles(p.tiles, m);
      if (count() > std::max<int64_t>(4 * kCus, whole + whole / 4)) break;
      const double t = duration(p.tiles, n_kv, dim);
      if (t < best) best = t, most = m;
    }
    split_tiles(p.tiles, most);
  }
  std::stable_sort(p.tiles.begin(), p.tiles.end(), [dim](const RowTile& a, const RowTile& b) { return a.alone(dim) > b.alone(dim); });
  for (const RowTile& t : p.tiles) {
    p.items += t.splits;
    if (t.splits > 1) {
      p.joins += (t.rows + kJoinRows - 1) / kJoinRows;
      p.part_rows += (int64_t)t.rows * t.splits;
    }
  }
  // The key weights' rows in the parts of the block that most of them see.  Parts that are joined come first, the first of
  // each sequence at the very front.
  const int least = least_tiles(p.starts.data(), lengths, n_seq, g, n_kv, window, first);
  std::vector<WeightPart> rest, single;
  for (int64_t s = 0; s < n_seq; ++s) {
    const KeyBlocks keys(lengths[s], counts[s], (int)g, (int)window, (int)first);
    const int parts = keys.parts(keys.heads > 0, 1 << 30, least);
    if (parts == 1) {
      single.push_back({(int)s, 0, 1, 0});
      continue;
    }
    for (int i = 0; i < parts; ++i) (i == 0 ? p.weights : rest).push_back({(int)s, i, parts, (int)p.weight_parts});
    p.weight_parts += parts;
  }
  p.weight_joins = (int64_t)p.weights.size();
  p.weights.insert(p.weights.end(), rest.begin(), rest.end());
  p.weights.insert(p.weights.end(), single.begin(), single.end());
  return p;
}

template <int DP, bool kF16, bool kFull>
int launch_chunk(const ChunkArgs& a, int64_t wgs, hipStream_t st) {
  if (a.lse != nullptr)
    chunk_attention_kernel<DP, kF16, kFull, true><<<(unsigned)wgs, kWave * kWaves, 0, st>>>(a);
  else
    chunk_attention_kernel<DP, kF16, kFull, false><<<(unsigned)wgs, kWave * kWaves, 0, st>>>(a);
  return check_launch("chunk_attention_kernel");
}

int64_t part_bytes(int64_t part_rows, int64_t n_kv, int64_t d) { return part_rows * n_kv * (4 * d + 16); }

}  // namespace
}  // namespace klc

using namespace klc;

extern "C" int klc_attn_plan(const int32_t* counts, const int32_t* lengths, int64_t n_seq, int64_t n_heads, int64_t n_kv,
                             int64_t head_dim, int64_t window, int64_t first, int32_t* plan, int64_t capacity,
                             int64_t* sizes) {
  KLC_REQUIRE(counts && lengths && sizes && (plan || capacity == 0), KLC_ERR_ARGUMENT, "klc_attn_plan: null pointer");
  KLC_REQUIRE(n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && n_heads <= 4096 && head_dim >= 8 && head_dim % 8 == 0 &&
                  head_dim <= 128,
              KLC_ERR_SHAPE, "klc_attn_plan: heads %lld / %lld, head_dim %lld (8..128, multiple of 8)", (long long)n_heads,
              (long long)n_kv, (long long)head_dim);
  KLC_REQUIRE(n_seq > 0 && n_seq < ((int64_t)1 << 20) && window >= 0 && window < ((int64_t)1 << 30) && first >= 0 &&
                  first < ((int64_t)1 << 29) && (first == 0 || window > 0),
              KLC_ERR_ARGUMENT, "klc_attn_plan: %lld sequences, window %lld, %lld first tokens beside it", (long long)n_seq,
              (long long)window, (long long)first);
  int64_t tokens = 0;
  for (int64_t s = 0; s < n_seq; ++s) {
    KLC_REQUIRE(counts[s] > 0 && lengths[s] >= counts[s] && lengths[s] < (1 << 29), KLC_ERR_ARGUMENT,
                "klc_attn_plan: sequence %lld of %d new tokens among %d (at least one, below 2^29)", (long long)s, counts[s],
                lengths[s]);
    tokens += counts[s];
  }
  KLC_REQUIRE(tokens * (n_heads / n_kv) < ((int64_t)1 << 30), KLC_ERR_ARGUMENT,
              "klc_attn_plan: %lld tokens of groups of %lld heads (below 2^30 rows)", (long long)tokens,
              (long long)(n_heads / n_kv));
  try {
    const ChunkPlan p = chunk_plan(counts, lengths, n_seq, n_heads, n_kv, head_dim, window, first);
    const int64_t at_items = (n_seq + 1 + kRecord - 1) / kRecord * kRecord, at_joins = at_items + p.items * kRecord;
    KLC_REQUIRE(p.part_rows < ((int64_t)1 << 31) && p.items * n_kv < kMostBlocks && p.joins * n_kv < kMostBlocks,
                KLC_ERR_ARGUMENT, "klc_attn_plan: %lld tokens of %lld heads are too many", (long long)tokens, (long long)n_heads);
    const int64_t at_weights = at_joins + p.joins * kRecord;
    sizes[0] = at_weights + (int64_t)p.weights.size() * 4;
    sizes[1] = tokens;
    sizes[2] = at_items, sizes[3] = p.items;
    sizes[4] = at_joins, sizes[5] = p.joins;
    sizes[6] = p.part_rows, sizes[7] = part_bytes(p.part_rows, n_kv, head_dim);
    sizes[8] = at_weights, sizes[9] = (int64_t)p.weights.size(), sizes[10] = p.weight_joins, sizes[11] = p.weight_parts;
    if (sizes[0] > capacity) return KLC_OK;
    std::fill(plan, plan + at_items, 0);
    std::copy(p.starts.begin(), p.starts.end(), plan);
    int32_t *item = plan + at_items, *join = plan + at_joins;
    int64_t part = 0;
    for (const RowTile& t : p.tiles) {
      const int32_t begin = p.starts[t.seq], count = counts[t.seq];
      for (int s = 0; s < t.splits; ++s, item += kRecord) {
        const int32_t rec[kRecord] = {t.seq, begin, count, t.row0, t.rows, s, t.splits, t.splits > 1 ? (int32_t)part : 0};
        std::copy(rec, rec + kRecord, item);
      }
      if (t.splits == 1) continue;
      for (int r = 0; r < t.rows; r += kJoinRows, join += kRecord) {
        const int32_t rec[kRecord] = {t.seq, begin, count, t.row0 + r, std::min(kJoinRows, t.rows - r), t.splits, (int32_t)part + r, t.rows};
        std::copy(rec, rec + kRecord, join);
      }
      part += (int64_t)t.rows * t.splits;
    }
    int32_t* weight = plan + at_weights;
    for (const WeightPart& w : p.weights) {
      const int32_t rec[4] = {w.seq, w.part, w.parts, w.offset};
      weight = std::copy(rec, rec + 4, weight);
    }
  } catch (const std::exception& e) {
    return set_error(KLC_ERR_ARGUMENT, "klc_attn_plan: %s", e.what());
  }
  return KLC_OK;
}

extern "C" int klc_attn_chunk(const klc_attn_chunk_args* args, void* stream) {
  KLC_REQUIRE(args != nullptr, KLC_ERR_ARGUMENT, "klc_attn_chunk: null pointer");
  const klc_attn_chunk_args& x = *args;
  KLC_REQUIRE(x.q && x.k_pages && x.v_pages && x.lengths && x.plan && x.out && (x.tables || x.table_width == 0), KLC_ERR_ARGUMENT,
              "klc_attn_chunk: null pointer");
  const int64_t d = x.head_dim;
  KLC_REQUIRE(x.n_heads > 0 && x.n_kv > 0 && x.n_heads % x.n_kv == 0 && x.n_heads <= 4096 && d >= 8 && d % 8 == 0 && d <= 128,
              KLC_ERR_SHAPE, "klc_attn_chunk: heads %lld / %lld, head_dim %lld (8..128, multiple of 8)", (long long)x.n_heads,
              (long long)x.n_kv, (long long)d);
  KLC_REQUIRE(x.page_size >= 16 && x.page_size <= 4096 && (x.page_size & (x.page_size - 1)) == 0 && x.n_pages > 0 &&
                  x.n_pages < ((int64_t)1 << 31) && x.n_pages * x.page_size < ((int64_t)1 << 31) && x.table_width >= 0 &&
                  x.table_width < ((int64_t)1 << 25) && x.table_width * x.page_size < ((int64_t)1 << 29),
              KLC_ERR_SHAPE, "klc_attn_chunk: %lld pages of %lld tokens (a power of two, 16..4096), tables of %lld",
              (long long)x.n_pages, (long long)x.page_size, (long long)x.table_width);
  KLC_REQUIRE(x.page_size * x.n_kv * d < ((int64_t)1 << 30), KLC_ERR_SHAPE,
              "klc_attn_chunk: pages of %lld tokens of %lld x %lld (below 2 GiB)", (long long)x.page_size, (long long)x.n_kv,
              (long long)d);
  KLC_REQUIRE(x.q_stride >= x.n_heads * d && x.q_stride % 8 == 0, KLC_ERR_SHAPE,
              "klc_attn_chunk: q stride %lld (a multiple of 8, no overlap)", (long long)x.q_stride);
  KLC_REQUIRE(((uintptr_t)x.q | (uintptr_t)x.k_pages | (uintptr_t)x.v_pages | (uintptr_t)x.workspace | (uintptr_t)x.out) % 16 == 0 &&
                  ((uintptr_t)x.plan | (uintptr_t)x.lse) % 4 == 0,
              KLC_ERR_ARGUMENT, "klc_attn_chunk: q, pages, workspace and out must be 16-byte aligned");
  KLC_REQUIRE(x.window >= 0 && x.window < ((int64_t)1 << 30) && x.first >= 0 && x.first < ((int64_t)1 << 29) &&
                  (x.first == 0 || x.window > 0) && x.scale > 0 && (float)x.scale > 0.f && (float)(x.scale * kLog2e) < INFINITY,
              KLC_ERR_ARGUMENT, "klc_attn_chunk: window %lld, %lld first tokens, scale %g", (long long)x.window,
              (long long)x.first, x.scale);
  KLC_REQUIRE(x.kv_dtype == KLC_DTYPE_BF16 || x.kv_dtype == KLC_DTYPE_F16, KLC_ERR_UNSUPPORTED,
              "klc_attn_chunk: kv_dtype %lld (bfloat16 or float16)", (long long)x.kv_dtype);
  const int64_t need = part_bytes(x.part_rows, x.n_kv, d);
  KLC_REQUIRE(x.items > 0 && x.joins >= 0 && x.part_rows >= 0 && x.items * x.n_kv < kMostBlocks &&
                  x.joins * x.n_kv < kMostBlocks,
              KLC_ERR_ARGUMENT, "klc_attn_chunk: a plan of %lld items, %lld joins", (long long)x.items, (long long)x.joins);
  KLC_REQUIRE(need == 0 || (x.workspace && x.workspace_bytes >= need), KLC_ERR_ARGUMENT,
              "klc_attn_chunk: workspace of %lld bytes, need %lld", (long long)x.workspace_bytes, (long long)need);
  auto in = [](const void* v) { return static_cast<const uint16_t*>(v); };
  auto index = [](const void* v) { return static_cast<const int32_t*>(v); };
  int page_log2 = 0;
  while ((1 << page_log2) < x.page_size) ++page_log2;
  float* part_o = static_cast<float*>(x.workspace);
  const ChunkArgs a{in(x.q), in(x.k_pages), in(x.v_pages), index(x.tables), index(x.lengths), index(x.plan) + x.at_items,
                    index(x.plan) + x.at_joins, in(x.sinks), static_cast<uint16_t*>(x.out), static_cast<float*>(x.lse), part_o,
                    need > 0 ? reinterpret_cast<float4*>(part_o + x.part_rows * x.n_kv * d) : nullptr, x.q_stride, x.part_rows,
                    (int)x.n_heads, (int)x.n_kv, (int)d, (int)x.n_pages, page_log2, (int)x.table_width, (int)x.window,
                    (int)x.first, (float)(x.scale * kLog2e)};
  const hipStream_t st = as_stream(stream);
  const bool f16 = x.kv_dtype == KLC_DTYPE_F16;
  const int64_t wgs = x.items * x.n_kv;
  int rc;
  if (d == 64)
    rc = f16 ? launch_chunk<64, true, true>(a, wgs, st) : launch_chunk<64, false, true>(a, wgs, st);
  else if (d == 128)
    rc = f16 ? launch_chunk<128, true, true>(a, wgs, st) : launch_chunk<128, false, true>(a, wgs, st);
  else if (d < 64)
    rc = f16 ? launch_chunk<64, true, false>(a, wgs, st) : launch_chunk<64, false, false>(a, wgs, st);
  else
    rc = f16 ? launch_chunk<128, true, false>(a, wgs, st) : launch_chunk<128, false, false>(a, wgs, st);
  if (rc || x.joins == 0) return rc;
  chunk_join_kernel<<<(unsigned)(x.joins * x.n_kv), kWave * kWaves, 0, st>>>(a);
  return check_launch("chunk_join_kernel");
}
