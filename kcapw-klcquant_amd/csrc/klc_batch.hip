// Attention of a decode batch over a paged KV cache (gfx950): one token of
// each sequence, whose first tokens may be a prefix that all sequences share.
//
// One launch with two kinds of workgroups, so that the compute-bound prefix
// and the sequences' own keys, a stream from HBM, share the chip:
//   shared  a KV head, 128 query rows (sequence, head of the group) and a
//           range of the prefix: 4 waves x 32 rows over one ring of tiles
//   own     a KV head of one sequence and a range of its own keys (with a
//           window, or a prefix not worth the pass above, of all its keys):
//           1, 2 or 4 waves take its tiles in turn, each through a ring of its
//           own with no barrier
// Two workgroups fit a CU by LDS and registers.  Parts are float32 (sum,
// maximum, normaliser) and a second launch joins them; where a row has one
// part, the own workgroup writes the result itself:
//
//   out = sum_i 2^(m_i - m) o_i / (sum_i 2^(m_i - m) l_i + 2^(s - m)),  m = max(m_i, s)
//
// What bounds it (64 heads over 8 of size 64, float16 pages): 64 sequences
// with up to 700 own tokens behind a prefix of 8,192, 27 to 32 us of which the
// join is 4.5; the prefix's pass is the longer side, with one wave a SIMD 465
// ns for 32 rows by 32 keys where two waves would take 227 each.  More
// workgroups would write more parts; two waves that join theirs in LDS are not
// tried.  256 sequences of 2,000 tokens, 124 us: HBM at 4.8 TB/s.  200 on a
// window of 128, 13.6 us, and 8 behind 500 tokens, 9 us: the chain of length,
// page numbers, first tile.  32 of 900 behind 16,000, 32 heads of size 128,
// 29 to 37 us and a join of 5.5.  The plan goes by counts and the tables'
// width, not by the lengths: 127 sequences of 200 to 1,000 tokens take 44 us,
// and with one of 32,000 beside them 765, its keys being one wave's.
#include <math.h>

#include <algorithm>

#include "klc_paged_tiles.h"

namespace klc {
namespace {

constexpr int kBatchGroup = 32;   // most query heads of a KV head: the columns of a wave's matrix instruction
constexpr int kPrefixAlign = 64;  // own keys start at a multiple of this in a sequence's list of keys

struct BatchArgs {
  const uint16_t* q;                   // bfloat16 [n_seq] rows
  const uint16_t *k_pages, *v_pages;   // [n_pages][page][n_kv][d]
  const int32_t *tables, *lengths;     // [n_seq][width], [n_seq]
  const int32_t* prefix_table;         // [prefix pages]
  const uint16_t* sinks;
  uint16_t* out;
  float* part_o;                       // [n_seq * n_heads][splits][d]
  float2* part_ml;                     // [n_seq * n_heads][splits]
  int64_t q_stride;
  int n_seq, n_heads, n_kv, d, n_pages, page_log2, width, prefix, window;
  int shared_splits, shared_tiles, shared_wgs;  // parts of the prefix, tiles of one, workgroups
  int own_splits, own_waves;                    // parts of a sequence's keys, waves of one
  float c2;
};

// The prefix's part of 128 query rows: workgroup (KV head, split of the keys,
// tile of rows).  As in the prompt's kernel, the scores of the next 32 keys
// are multiplied while the exponentials of these are taken.
template <int DP, bool kF16, bool kFull>
__device__ __forceinline__ void shared_part(const BatchArgs& a, int wg, lds_u8 ring) {
  constexpr int KT = kSharedTile<DP>, kSub = KT / kKeys;
  using F = AttnWave<DP, kF16, kFull, 1, kKeys>;
  constexpr int kMat = kSub * F::kMatBytes, kStage = 2 * kMat, kRing = kTileLds / kStage;
  constexpr int kDmas = kSub * F::kDmas / kWaves;  // of K, and of V, a wave and tile
  constexpr int kQuads = 4 * F::kDimBlocks;
  static_assert(kRing >= 3 && kSub * F::kDmas % kWaves == 0, "");
  const int g = a.n_heads / a.n_kv, rows = a.n_seq * g;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int kvh = wg % a.n_kv, split = wg / a.n_kv % a.shared_splits, row_tile = wg / (a.n_kv * a.shared_splits);
  const int key0 = split * a.shared_tiles * KT, keys = min(a.shared_tiles * KT, a.prefix - key0);  // of this split
  const int tiles = (keys + KT - 1) / KT, steps = (keys + kKeys - 1) / kKeys;
  const int w_row = (row_tile * kWaves + wave) * 32;
  const bool w_live = w_row < rows;
  const int row = min(w_row + lane % 32, rows - 1), b = row / g, head = kvh * g + row - b * g;
  F f;
  f.init(ring, a.d);
  load_query<F>(f.q[0], a.q + b * a.q_stride + (int64_t)head * a.d, a.d);
  PageLoads<BatchArgs, F, KT, kDmas, kWaves> pages(a, wave, kvh);
  pages.hold(a.prefix_table, key0 >> a.page_log2, ((a.prefix - 1) >> a.page_log2) + 1);
  settle_query<F>(f.q[0]);
  auto stage = [&](int j) { return j % kRing * kStage; };
  auto load = [&](int j) {
    if (j < tiles) pages.load(key0 + j * KT, within(0, a.prefix - 1), ring + stage(j), ring + stage(j) + kMat);
  };
#pragma unroll
  for (int j = 0; j < kRing - 1; ++j) load(j);
  const float c2 = a.c2 * convert_query<F, kF16>(f.q[0]);
  // tile j is there for all waves, kAhead later ones may be in flight; a last tile's V is cleared behind its keys
  auto arrive = [&](int j, auto ahead) {
    if (j + decltype(ahead)::value < tiles)
      tile_wait<2 * kDmas * decltype(ahead)::value, true>();
    else
      tile_wait<0, true>();
    if ((j + 1) * KT > keys && j * KT < keys) {
      clear_values<F, KT>(ring + stage(j) + kMat, 0, keys - j * KT, threadIdx.x, kWave * kWaves);
      tile_wait<0, true>();
    }
  };
  auto settle = [&](int i, f32x16_t (&s)[1][1]) {
    if ((i + 1) * kKeys > keys) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (i * kKeys + 8 * (e / 4) + e % 4 + 4 * (lane / 32) >= keys) s[0][0][e] = -INFINITY;
    }
    f.raise(0, s[0], c2);
  };
  // the values of keys i, whose settled scores are s, and the scores of keys i + 1; `last`: of their tile
  auto step = [&](int i, auto last, f32x16_t (&s)[1][1], f32x16_t (&next)[1][1]) {
    const int j = i / kSub, here = stage(j) + i % kSub * F::kMatBytes;
    if constexpr (decltype(last)::value) {
      arrive(j + 1, Count<kRing - 3>{});  // every wave is done with tile j - 1
      load(j + kRing - 1);
    }
    if (!w_live) return;
    u32x4_t p[1][2];
    f.scores(stage((i + 1) / kSub) + (i + 1) % kSub * F::kMatBytes, next);  // past the last: of nothing, not used
    f.weigh(0, s[0], c2, p[0]);
    f.values(here + kMat, p);
    if (i + 1 < steps) settle(i + 1, next);
  };
  f32x16_t sa[1][1], sb[1][1];
  arrive(0, Count<kRing - 2>{});
  f.scores(0, sa);
  settle(0, sa);
  for (int i = 0; i < steps; i += 2) {
    step(i, Count<kSub == 1>{}, sa, sb);
    if (i + 1 < steps) step(i + 1, Count<1>{}, sb, sa);
  }

  const bool bad = __syncthreads_or(pages.bad);
  const float sum = add_halves(f.l[0]);
  const int splits = a.shared_splits + a.own_splits;
  if (lane < 32 && w_row + lane < rows)
    a.part_ml[((int64_t)b * a.n_heads + head) * splits + split] = make_float2(f.m[0], bad ? __uint_as_float(0x7fc00000u) : sum);
  // the wave's sums through LDS, so that they leave as whole rows: 16 bytes at (row, chunk ^ row) of [32][DP]
  typedef __attribute__((address_space(3))) f32x4_t* lds_f32x4;
  constexpr int kRowQuads = DP / 4;
  const lds_f32x4 out = (lds_f32x4)(ring + wave * 32 * DP * 4);
#pragma unroll
  for (int i = 0; i < kQuads; ++i) out[lane % 32 * kRowQuads + ((quad_dim(i) / 4) ^ (lane % 8))] = quad(f, i);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 4
  for (int i = 0; i < 32 * kRowQuads / kWave; ++i) {
    const int r = (i * kWave + lane) / kRowQuads, c = lane % kRowQuads, at_row = w_row + r;
    const int rb = at_row / g;
    if (at_row < rows && 4 * c < a.d)
      *reinterpret_cast<f32x4_t*>(a.part_o + (((int64_t)rb * a.n_heads + kvh * g + at_row - rb * g) * splits + split) * a.d + 4 * c) =
          out[r * kRowQuads + (c ^ (r % 8))];
  }
}

// A sequence's own part, and without a shared pass its part of the prefix:
// own_waves waves take item (KV head, split, sequence).  The keys are listed
// as [prefix, padded to kPrefixAlign][own].
template <int DP, bool kF16, bool kFull>
__device__ __forceinline__ void own_part(const BatchArgs& a, int wg, lds_u8 lds, float2 (&wave_ml)[kWaves][kBatchGroup]) {
  using F = AttnWave<DP, kF16, kFull, 1, kKeys>;
  constexpr int KT = kKeys, kRing = kTileLds / kWaves / F::kStage, kQuads = 4 * F::kDimBlocks;
  static_assert(kRing == 1 || kRing == 2, "");
  // With one tile a wave, K and V take turns: the next K comes while this V is multiplied, and the other way round
  // (64 sequences of 2,000 tokens, head size 128: 77.8 us by whole tiles, 69.7 so; with two tiles a wave the second
  // addressing costs more than it hides, 124 us against 128 for 256 sequences of head size 64).
  constexpr bool kHalves = kRing == 1;
  const int g = a.n_heads / a.n_kv, lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int team = a.own_waves, rank = wave % team;  // the item's waves, and which of them this is
  const int items = a.n_kv * a.own_splits * a.n_seq, item = min(wg * (kWaves / team) + wave / team, items - 1);
  const bool spare = wg * (kWaves / team) + wave / team >= items;  // past the last item: nothing to do but the barriers
  const int kvh = item % a.n_kv, split = item / a.n_kv % a.own_splits, b = item / (a.n_kv * a.own_splits);
  const int splits = a.shared_splits + a.own_splits;
  const int head = kvh * g + min(lane % 32, g - 1);
  F f;
  load_query<F>(f.q[0], a.q + b * a.q_stride + (int64_t)head * a.d, a.d);
  const int32_t* own_table = a.tables + (int64_t)b * a.width;
  PageLoads<BatchArgs, F, KT, F::kDmas, 1> pages(a, 0, kvh);
  int holds = a.width > 0 ? 1 : -1;  // 1 the own table, 0 the prefix's (which may be a row of `tables`)
  if (holds == 1) pages.hold(own_table, 0, a.width);  // while the length is on its way
  int n = table_at(a.lengths, b);
  const bool absent = n < 0;
  const int64_t room = (int64_t)a.width << a.page_log2;
  const int64_t n_asked = n;
  n = (int)min((int64_t)max(n, 0), room);
  const int pad = (a.prefix + kPrefixAlign - 1) / kPrefixAlign * kPrefixAlign;
  // the list's visible range: from `begin` on, up to the prefix's end in its tiles and `end` in the others
  const int seen = a.window > 0 ? min(a.window, a.prefix + n) : a.prefix + n, low = a.prefix + n - seen;
  const int begin = a.shared_splits > 0 || low >= a.prefix ? pad + max(0, low - a.prefix) : low;
  const int end = n > 0 ? pad + n : a.prefix;
  const int first_tile = begin / KT, n_tiles = begin < end && !spare && !absent ? (end - 1) / KT + 1 - first_tile : 0;
  const int per = (n_tiles + a.own_splits - 1) / a.own_splits;
  const int end_tile = first_tile + min((split + 1) * per, n_tiles), first = first_tile + split * per + rank;
  const lds_u8 ring = lds + wave * kRing * F::kStage;
  f.init(ring, a.d);
  pages.bad = n_asked > room;
  // tile j: of the prefix or of the sequence's own keys
  auto load = [&](auto key, auto value, int j, int slot) {
    const bool own = j * KT >= pad;
    const int base = own ? j * KT - pad : j * KT, from = own ? max(begin - pad, 0) : begin, last = own ? n - 1 : a.prefix - 1;
    if (holds != (int)own)
      pages.hold(own ? own_table : a.prefix_table, max(base, from) >> a.page_log2, (last >> a.page_log2) + 1);
    holds = own;
    pages.template load<decltype(key)::value, decltype(value)::value>(base, within(from, last), ring + slot * F::kStage,
                                                                      ring + slot * F::kStage + F::kMatBytes);
  };
  settle_query<F>(f.q[0]);
#pragma unroll
  for (int i = 0; i < kRing; ++i)
    if (first + i * team < end_tile) {
      if constexpr (kHalves) {
        load(Count<true>{}, Count<false>{}, first + i * team, i);
        load(Count<false>{}, Count<true>{}, first + i * team, i);
      } else {
        load(Count<true>{}, Count<true>{}, first + i * team, i);
      }
    }
  const float c2 = a.c2 * convert_query<F, kF16>(f.q[0]);
  int slot = 0;
  for (int j = first; j < end_tile; j += team) {
    // K is there, and V unless it comes by itself; the ring's other tile may be in flight
    const bool refill = j + kRing * team < end_tile;
    if (kHalves)
      tile_wait<F::kDmas, false>();
    else if (j + team < end_tile)
      tile_wait<2 * F::kDmas, false>();
    else
      tile_wait<0, false>();
    const int stage = slot * F::kStage;
    const int from = max(0, begin - j * KT), to = min(KT, (j * KT >= pad ? end : a.prefix) - j * KT);
    const bool part = from > 0 || to < KT;
    f32x16_t sc[1][1];
    f.scores(stage, sc);
    if (kHalves && refill) {
      tile_wait<63, false>();  // K has been read
      load(Count<true>{}, Count<false>{}, j + kRing * team, slot);
    }
    if (part) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = 8 * (e / 4) + e % 4 + 4 * (lane / 32);
        if (key < from || key >= to) sc[0][0][e] = -INFINITY;
      }
    }
    u32x4_t p[1][2];
    f.softmax(0, sc[0], c2, p[0]);
    if (kHalves && refill)
      tile_wait<F::kDmas, false>();
    else if (kHalves)
      tile_wait<0, false>();
    if (part) {
      clear_values<F, KT>(ring + stage + F::kMatBytes, from, to, lane, kWave);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    f.values(stage + F::kMatBytes, p);
    if (refill) {
      tile_wait<63, false>();  // the slot has been read
      load(Count<!kHalves>{}, Count<true>{}, j + kRing * team, slot);
    }
    slot = (slot + 1) % kRing;
  }

  // the team's sums, lane by lane: [wave][quad][lane]
  typedef __attribute__((address_space(3))) f32x4_t* lds_f32x4;
  const lds_f32x4 sums = (lds_f32x4)lds;
  const float sum = add_halves(f.l[0]);
  const bool live = lane % 32 < g;
  if (team > 1) {
    __syncthreads();
    if (live) {
      if (lane < 32) wave_ml[wave][lane] = make_float2(f.m[0], pages.bad ? __uint_as_float(0x7fc00000u) : sum);
#pragma unroll
      for (int i = 0; i < kQuads; ++i) sums[(wave * kQuads + i) * kWave + lane] = quad(f, i);
    }
    __syncthreads();
  }
  if (!live || spare) return;
  const int64_t row = (int64_t)b * a.n_heads + head, at = row * splits + a.shared_splits + split;
  float2 ml[kWaves];
  float sink = -INFINITY;
  if (splits == 1 && a.sinks != nullptr) sink = sink_log2(a.sinks[head]);
  float top = sink;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    ml[w] = make_float2(-INFINITY, 0.f);
    if (w < team) ml[w] = team > 1 ? wave_ml[wave - rank + w][lane % 32] : make_float2(f.m[0], pages.bad ? __uint_as_float(0x7fc00000u) : sum);
    top = fmaxf(top, ml[w].x);
  }
  const float base = top == -INFINITY ? 0.f : top;
  float x[kWaves], l = sink != -INFINITY ? __builtin_amdgcn_exp2f(sink - base) : 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    x[w] = __builtin_amdgcn_exp2f(ml[w].x - base);
    l = fmaf(x[w], ml[w].y, l);
  }
  // without a key zeros, else 1 / 0 and 0 times it for scores that are all -inf: NaN, as their softmax
  const float inv = absent || (l == 0.f && a.prefix + n == 0) ? 0.f : 1.f / l;
  auto put = [&](int i, f32x4_t o) {
    if (!kFull && quad_dim(i) >= a.d) return;
    if (splits == 1)
      *reinterpret_cast<u32x2_t*>(a.out + row * a.d + quad_dim(i)) = u32x2_t{pack2<false>(o.x * inv, o.y * inv), pack2<false>(o.z * inv, o.w * inv)};
    else
      *reinterpret_cast<f32x4_t*>(a.part_o + at * a.d + quad_dim(i)) = o;
  };
  if (team == 1) {
#pragma unroll
    for (int i = 0; i < kQuads; ++i) put(i, x[0] * quad(f, i));
  } else {
    for (int i = rank; i < kQuads; i += team) {
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        if (w < team) o += x[w] * sums[((wave - rank + w) * kQuads + i) * kWave + lane];
      put(i, o);
    }
  }
  if (splits > 1 && rank == 0 && lane < 32) a.part_ml[at] = make_float2(top, l);
}

template <int DP, bool kF16, bool kFull>
__global__ __launch_bounds__(kWave * kWaves, 2) void batch_attention_kernel(BatchArgs a) {
  __shared__ __align__(1024) uint8_t lds[kTileLds];
  __shared__ float2 wave_ml[kWaves][kBatchGroup];
  // the shared ones first, one a CU; the own ones take the CUs' other halves
  if ((int)blockIdx.x < a.shared_wgs)
    shared_part<DP, kF16, kFull>(a, blockIdx.x, (lds_u8)lds);
  else
    own_part<DP, kF16, kFull>(a, blockIdx.x - a.shared_wgs, (lds_u8)lds, wave_ml);
}

// out[row] = sum over the splits.  W waves a row; in a wave, lanes take 4 dims
// each and the groups of lanes that this leaves take splits in turn.
template <int W>
__global__ __launch_bounds__(256) void batch_join_kernel(BatchArgs a) {
  __shared__ float4 wave_o[4][32];
  __shared__ float wave_l[4];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t row = (int64_t)blockIdx.x * (4 / W) + wave / W, rows = (int64_t)a.n_seq * a.n_heads;
  const bool live = row < rows;
  const int64_t r = live ? row : rows - 1;
  const int splits = a.shared_splits + a.own_splits;
  const int lanes = a.d <= 32 ? 8 : a.d <= 64 ? 16 : 32, groups = kWave / lanes, grp = lane / lanes;
  const int dim = min(4 * (lane % lanes), a.d - 4);
  const int n = a.lengths[r / a.n_heads];
  const bool absent = n < 0;
  const float2* ml = a.part_ml + r * splits;
  const float sink = a.sinks != nullptr ? sink_log2(a.sinks[r % a.n_heads]) : -INFINITY;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  if (!absent) {
    float top = sink;
    for (int s = lane; s < splits; s += kWave) top = fmaxf(top, ml[s].x);
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    const float base = top == -INFINITY ? 0.f : top;
    constexpr int kAhead = 4;
    const int step = groups * W;
    for (int s0 = (wave % W) * groups + grp; s0 < splits; s0 += kAhead * step) {
      float4 y[kAhead];
      float2 x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int s = min(s0 + i * step, splits - 1);
        y[i] = *reinterpret_cast<const float4*>(a.part_o + (r * splits + s) * a.d + dim);
        x[i] = ml[s];
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (s0 + i * step >= splits) break;
        const float w = __builtin_amdgcn_exp2f(x[i].x - base);
        l = fmaf(w, x[i].y, l);
        o.x = fmaf(w, y[i].x, o.x), o.y = fmaf(w, y[i].y, o.y), o.z = fmaf(w, y[i].z, o.z), o.w = fmaf(w, y[i].w, o.w);
      }
    }
    for (int off = lanes; off < kWave; off <<= 1) {
      l += __shfl_xor(l, off);
      o.x += __shfl_xor(o.x, off), o.y += __shfl_xor(o.y, off), o.z += __shfl_xor(o.z, off), o.w += __shfl_xor(o.w, off);
    }
    if (wave % W == 0 && sink != -INFINITY) l += __builtin_amdgcn_exp2f(sink - base);
  }
  if constexpr (W > 1) {
    if (lane < lanes) wave_o[wave][lane] = o;
    if (lane == 0) wave_l[wave] = l;
    __syncthreads();
    if (wave % W != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float4 y = wave_o[wave + w][lane % lanes];
      l += wave_l[wave + w];
      o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
    }
  }
  const float inv = absent || (l == 0.f && a.prefix + n == 0) ? 0.f : 1.f / l;
  if (live && lane < a.d / 4)
    *reinterpret_cast<u32x2_t*>(a.out + row * a.d + dim) = u32x2_t{pack2<false>(o.x * inv, o.y * inv), pack2<false>(o.z * inv, o.w * inv)};
}

struct BatchPlan {
  int64_t shared_splits, shared_tiles, row_tiles, own_splits, own_waves;
  int64_t splits() const { return shared_splits + own_splits; }
};
BatchPlan batch_plan(int64_t n_seq, int64_t n_heads, int64_t n_kv, int64_t d, int64_t prefix, int64_t max_own, int64_t window) {
  BatchPlan p{};
  const int64_t rows = n_seq * (n_heads / n_kv), items = n_seq * n_kv;
  p.row_tiles = (rows + 32 * kWaves - 1) / (32 * kWaves);
  // 256 own workgroups, one a CU: 64 sequences of 8 KV heads (512 items) take 31.6 us with 2 waves an item, 34.7 with
  // 1 and 33.9 with 4; 128 sequences with 1,000 own tokens 49 us with 1 wave and 57 with 2 or 4.
  p.own_waves = items >= 1024 ? 1 : items >= 512 ? 2 : 4;
  // The prefix again for every sequence, mostly out of the caches, or one pass and a join (without a window only, also
  // where a window hides nothing: 200 x 1,000 with 500 own tokens 60 us, and 74 with a window of 4,096): 64 x 500 of head_dim 64 take
  // 16.8 us without the pass and 19.7 with it, 200 x 300 25.6 and 28.8, 64 x 1,000 23.2 and 20.3, 200 x 1,000 48.8 and 32.7.
  const bool shared = window == 0 && n_seq > 1 && (double)items * prefix * d >= 1 << 25;
  int64_t keys = max_own + (shared ? 0 : prefix);
  if (window > 0 && window < keys) keys = window;
  if (shared) {
    const int64_t tile = d <= 64 ? kSharedTile<64> : kSharedTile<128>, tiles = (prefix + tile - 1) / tile;
    const int64_t want = (256 + n_kv * p.row_tiles - 1) / (n_kv * p.row_tiles);
    p.shared_tiles = (tiles + want - 1) / want;
    p.shared_splits = (tiles + p.shared_tiles - 1) / p.shared_tiles;
  }
  // With few items also parts of their keys, if that is worth a join: of 20 tiles (8 sequences) one part takes 9.2 us,
  // and three 7.1 and the join's launch of 3.6 more.
  const int64_t tiles = keys / kKeys + 2, want = ((shared ? 256 : 512) + items - 1) / items;
  p.own_splits = p.own_waves < 4 || (!shared && tiles <= 8 * kWaves) ? 1 : std::min(want, (tiles + 2 * kWaves - 1) / (2 * kWaves));
  return p;
}

// a row of one part needs none
int64_t batch_bytes(const BatchPlan& p, int64_t n_seq, int64_t n_heads, int64_t d) {
  return p.splits() == 1 ? 0 : n_seq * n_heads * p.splits() * (4 * d + 8);
}

template <int DP, bool kF16, bool kFull>
int launch_batch(const BatchArgs& a, const BatchPlan& p, hipStream_t st) {
  const int64_t items = (int64_t)a.n_seq * a.n_kv * p.own_splits, teams = kWaves / p.own_waves;
  const int64_t wgs = a.shared_wgs + (items + teams - 1) / teams;
  batch_attention_kernel<DP, kF16, kFull><<<(unsigned)wgs, kWave * kWaves, 0, st>>>(a);
  const int rc = check_launch("batch_attention_kernel");
  if (rc || p.splits() == 1) return rc;
  const int64_t rows = (int64_t)a.n_seq * a.n_heads;
  if (p.splits() > 16)
    batch_join_kernel<4><<<(unsigned)rows, 256, 0, st>>>(a);
  else
    batch_join_kernel<1><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(a);
  return check_launch("batch_join_kernel");
}

int check_sizes(const char* name, int64_t n_seq, int64_t n_heads, int64_t n_kv, int64_t d, int64_t prefix,
                int64_t max_own, int64_t window) {
  KLC_REQUIRE(n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && n_heads / n_kv <= kBatchGroup && n_heads <= 4096 &&
                  d >= 8 && d % 8 == 0 && d <= 128,
              KLC_ERR_SHAPE, "%s: heads %lld / %lld (group <= %d), head_dim %lld (8..128, multiple of 8)", name,
              (long long)n_heads, (long long)n_kv, kBatchGroup, (long long)d);
  KLC_REQUIRE(n_seq > 0 && n_seq <= 65535 && prefix >= 0 && prefix < ((int64_t)1 << 29) && max_own >= 0 &&
                  max_own < ((int64_t)1 << 29) && window >= 0 && window < ((int64_t)1 << 30),
              KLC_ERR_ARGUMENT, "%s: %lld sequences, prefix %lld, own tokens up to %lld, window %lld", name,
              (long long)n_seq, (long long)prefix, (long long)max_own, (long long)window);
  return KLC_OK;
}

}  // namespace
}  // namespace klc

using namespace klc;

extern "C" int64_t klc_attn_batch_workspace_bytes(int64_t n_seq, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                                                  int64_t prefix_len, int64_t max_own, int64_t window) {
  const int rc = check_sizes("klc_attn_batch_workspace_bytes", n_seq, n_heads, n_kv, head_dim, prefix_len, max_own, window);
  if (rc) return rc;
  return batch_bytes(batch_plan(n_seq, n_heads, n_kv, head_dim, prefix_len, max_own, window), n_seq, n_heads, head_dim);
}

extern "C" int klc_attn_batch(const klc_attn_batch_args* args, void* stream) {
  KLC_REQUIRE(args != nullptr, KLC_ERR_ARGUMENT, "klc_attn_batch: null pointer");
  const klc_attn_batch_args& x = *args;
  KLC_REQUIRE(x.q && x.k_pages && x.v_pages && x.lengths && x.out, KLC_ERR_ARGUMENT, "klc_attn_batch: null pointer");
  KLC_REQUIRE((x.tables || x.table_width == 0) && (x.prefix_table || x.prefix_len == 0), KLC_ERR_ARGUMENT,
              "klc_attn_batch: null table");
  KLC_REQUIRE(x.page_size >= 16 && x.page_size <= 4096 && (x.page_size & (x.page_size - 1)) == 0 && x.n_pages > 0 &&
                  x.n_pages < ((int64_t)1 << 31) && x.n_pages * x.page_size < ((int64_t)1 << 31) && x.table_width >= 0 &&
                  x.table_width < ((int64_t)1 << 25),
              KLC_ERR_SHAPE, "klc_attn_batch: %lld pages of %lld tokens (a power of two, 16..4096), tables of %lld",
              (long long)x.n_pages, (long long)x.page_size, (long long)x.table_width);
  const int64_t max_own = x.table_width * x.page_size, d = x.head_dim, rows = x.n_seq * x.n_heads;
  int rc = check_sizes("klc_attn_batch", x.n_seq, x.n_heads, x.n_kv, d, x.prefix_len, max_own, x.window);
  if (rc) return rc;
  KLC_REQUIRE(x.page_size * x.n_kv * d < ((int64_t)1 << 30), KLC_ERR_SHAPE,
              "klc_attn_batch: pages of %lld tokens of %lld x %lld (below 2 GiB)", (long long)x.page_size,
              (long long)x.n_kv, (long long)d);
  KLC_REQUIRE(x.q_stride >= x.n_heads * d && x.q_stride % 8 == 0, KLC_ERR_SHAPE,
              "klc_attn_batch: q stride %lld (a multiple of 8, no overlap)", (long long)x.q_stride);
  KLC_REQUIRE(((uintptr_t)x.q | (uintptr_t)x.k_pages | (uintptr_t)x.v_pages | (uintptr_t)x.workspace | (uintptr_t)x.out) % 16 == 0,
              KLC_ERR_ARGUMENT, "klc_attn_batch: q, pages, workspace and out must be 16-byte aligned");
  KLC_REQUIRE(x.scale > 0 && (float)x.scale > 0.f && (float)(x.scale * kLog2e) < INFINITY, KLC_ERR_ARGUMENT,
              "klc_attn_batch: scale %g", x.scale);
  KLC_REQUIRE(x.kv_dtype == KLC_DTYPE_BF16 || x.kv_dtype == KLC_DTYPE_F16, KLC_ERR_UNSUPPORTED,
              "klc_attn_batch: kv_dtype %lld (bfloat16 or float16)", (long long)x.kv_dtype);
  const BatchPlan p = batch_plan(x.n_seq, x.n_heads, x.n_kv, d, x.prefix_len, max_own, x.window);
  const int64_t need = batch_bytes(p, x.n_seq, x.n_heads, d);
  KLC_REQUIRE(need == 0 || (x.workspace && x.workspace_bytes >= need), KLC_ERR_ARGUMENT,
              "klc_attn_batch: workspace of %lld bytes, need %lld", (long long)x.workspace_bytes, (long long)need);
  auto in = [](const void* v) { return static_cast<const uint16_t*>(v); };
  auto index = [](const void* v) { return static_cast<const int32_t*>(v); };
  int page_log2 = 0;
  while ((1 << page_log2) < x.page_size) ++page_log2;
  float* part_o = static_cast<float*>(x.workspace);
  float2* part_ml = need > 0 ? reinterpret_cast<float2*>(part_o + rows * p.splits() * d) : nullptr;
  const BatchArgs a{in(x.q), in(x.k_pages), in(x.v_pages), index(x.tables), index(x.lengths), index(x.prefix_table),
                    in(x.sinks), static_cast<uint16_t*>(x.out), part_o, part_ml, x.q_stride, (int)x.n_seq,
                    (int)x.n_heads, (int)x.n_kv, (int)d, (int)x.n_pages, page_log2, (int)x.table_width,
                    (int)x.prefix_len, (int)x.window, (int)p.shared_splits, (int)p.shared_tiles,
                    (int)(p.shared_splits * p.row_tiles * x.n_kv), (int)p.own_splits, (int)p.own_waves, (float)(x.scale * kLog2e)};
  const hipStream_t st = as_stream(stream);
  const bool f16 = x.kv_dtype == KLC_DTYPE_F16;
  if (d == 64) return f16 ? launch_batch<64, true, true>(a, p, st) : launch_batch<64, false, true>(a, p, st);
  if (d == 128) return f16 ? launch_batch<128, true, true>(a, p, st) : launch_batch<128, false, true>(a, p, st);
  if (d < 64) return f16 ? launch_batch<64, true, false>(a, p, st) : launch_batch<64, false, false>(a, p, st);
  return f16 ? launch_batch<128, true, false>(a, p, st) : launch_batch<128, false, false>(a, p, st);
}
