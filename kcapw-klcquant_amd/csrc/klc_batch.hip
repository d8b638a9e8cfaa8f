// Attention of a decode batch over a paged KV cache (gfx950): one token of
// each sequence, whose first tokens may be a prefix that all sequences share.
//
// One launch with two kinds of workgroups, so that the compute-bound prefix
// and the sequences' own keys, a stream from HBM, share the chip:
//   shared  a KV head, 128 query rows (sequence, head of the group) and a
//           range of the prefix: 4 waves x 32 rows over one ring of tiles, the
//           prefix's keys read once for the batch
//   own     a KV head of one sequence and a range of its own keys (with a
//           window, or a prefix not worth the pass above, of all its keys):
//           its waves take tiles in turn, each through a ring of its own with
//           no barrier, and join their sums in LDS
// Parts are float32 (sum, maximum, normaliser) and a second launch joins
// them; where a row has one part, the own workgroup writes the result itself.
#include <math.h>

#include "klc_flash.h"

namespace klc {
namespace {

constexpr int kWaves = 4;
constexpr int kOwnTile = 32;      // keys of a tile of an own wave
constexpr int kOwnRing = 2;
constexpr int kBatchGroup = 32;   // most query heads of a KV head: the columns of a wave's matrix instruction
constexpr int kPrefixAlign = 64;  // own keys start at a multiple of this in a sequence's list of keys
// a shared tile is 16 KB of K and V, four of them the LDS of a head size of 64
template <int DP>
constexpr int kSharedTile = DP == 64 ? 64 : 32;
template <int DP>
constexpr int kBatchLds = kWaves * kOwnRing * 2 * kOwnTile * 2 * DP;

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
  int n_seq, n_heads, n_kv, d, n_pages, page_log2, width, prefix, window, shared_splits, own_splits, shared_tiles, shared_wgs;
  float c2;
};

typedef const __attribute__((address_space(4))) int32_t* const_i32;
// a uniform element of a table, by a scalar load: vector loads would wait behind the tiles in flight
__device__ __forceinline__ int32_t table_at(const int32_t* t, int64_t i) {
  return reinterpret_cast<const_i32>(reinterpret_cast<uintptr_t>(t))[i];
}

// Chunk c of a bfloat16 query row for each of the wave's steps, in the
// cache's type.  A float16 cache takes the row times a power of two that
// brings its largest value to [1, 2), which every float16 represents as well
// as bfloat16 does (what it rounds off lies 2^-24 below that value); the
// returned factor puts it back.
template <class F, bool kF16>
__device__ __forceinline__ float load_query(u32x4_t (&q)[F::kSteps], const uint16_t* src, int d) {
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int st = 0; st < F::kSteps; ++st) {
    const int c = 2 * st + lane / 32;
    q[st] = u32x4_t{0, 0, 0, 0};
    if (8 * c < d) q[st] = *reinterpret_cast<const u32x4_t*>(src + 8 * c);
  }
  if constexpr (!kF16) return 1.f;
  float most = 0.f;
#pragma unroll
  for (int st = 0; st < F::kSteps; ++st)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      most = fmaxf(most, fmaxf(fabsf(__uint_as_float(q[st][e] << 16)), fabsf(__uint_as_float(q[st][e] & 0xffff0000u))));
  most = max_halves(most);
  const int ex = most > 0.f && most < INFINITY ? ilogbf(most) : 0;
#pragma unroll
  for (int st = 0; st < F::kSteps; ++st)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      q[st][e] = pack2<true>(ldexpf(__uint_as_float(q[st][e] << 16), -ex), ldexpf(__uint_as_float(q[st][e] & 0xffff0000u), -ex));
  return ldexpf(1.f, ex);
}

// A lane's source row of a load instruction: `key` is the instruction's first
// key (its rows lie in one page).  Keys outside the visible first..last take
// the nearest visible one's row, so that only its pages are asked for.
struct PageRow {
  int64_t row;  // of [n_pages * page]
  bool bad;
};
__device__ __forceinline__ PageRow page_row(const int32_t* table, int key, int lane_key, int first, int last,
                                            int page_log2, int n_pages) {
  const int page = table_at(table, __builtin_amdgcn_readfirstlane(min(max(key, first), last) >> page_log2));
  const bool bad = (unsigned)page >= (unsigned)n_pages;
  return {((int64_t)(bad ? 0 : page) << page_log2) + (min(max(lane_key, first), last) & ((1 << page_log2) - 1)), bad};
}

// The tile's loads have landed: of the wave's own, or with kBarrier of every
// wave of the workgroup, each of which is then done with the tile before.
template <int kOutstanding, bool kBarrier>
__device__ __forceinline__ void tile_wait() {
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(kOutstanding));
  if constexpr (kBarrier) __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// Clears the V rows of a tile outside [from, to), whose values no query sees
// (0 * inf would make NaN of them); the caller orders it.
template <class F, int KT>
__device__ __forceinline__ void clear_values(lds_u8 stage, int from, int to, int thread, int threads) {
  for (int i = thread; i < KT * F::kChunks; i += threads) {
    const int r = i / F::kChunks;
    if (r < from || r >= to)
      *reinterpret_cast<__attribute__((address_space(3))) u32x4_t*>(stage + F::kMatBytes + i * 16) = u32x4_t{0, 0, 0, 0};
  }
}

// The prefix's part of 128 query rows: workgroup (KV head, tile of rows,
// split of the keys).
template <int DP, bool kF16, bool kFull>
__device__ __forceinline__ void shared_part(const BatchArgs& a, int wg, lds_u8 ring) {
  constexpr int KT = kSharedTile<DP>, W = kWaves;
  using F = Flash<DP, kF16, kFull, 1, KT>;
  constexpr int kRing = kBatchLds<DP> / F::kStage, kLoads = 2 * F::kDmas / W;
  static_assert(F::kDmas % W == 0 && kRing >= 3, "the tile's loads split evenly over the waves");
  const int g = a.n_heads / a.n_kv, rows = a.n_seq * g;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int kvh = wg % a.n_kv, split = wg / a.n_kv % a.shared_splits, row_tile = wg / (a.n_kv * a.shared_splits);
  const int first = split * a.shared_tiles, end_tile = min(first + a.shared_tiles, (a.prefix + KT - 1) / KT);
  const int w_row = (row_tile * W + wave) * 32;
  const bool w_live = w_row < rows;
  const int row = min(w_row + lane % 32, rows - 1), b = row / g, head = kvh * g + row - b * g;
  F f;
  f.init(ring, a.d);
  const float c2 = a.c2 * load_query<F, kF16>(f.q[0], a.q + b * a.q_stride + (int64_t)head * a.d, a.d);
  const int64_t kv_stride = (int64_t)a.n_kv * a.d;
  bool bad = false;
  auto load = [&](int j) {
    const lds_u8 stage = ring + ((j - first) % kRing) * F::kStage;
#pragma unroll
    for (int i = 0; i < F::kDmas / W; ++i) {
      const int n = wave + i * W, r = F::dma_row(n);
      const PageRow p = page_row(a.prefix_table, j * KT + n * F::kRowsPerDma, j * KT + r, 0, a.prefix - 1, a.page_log2, a.n_pages);
      bad |= p.bad;
      const int64_t at = p.row * kv_stride + (int64_t)kvh * a.d + 8 * F::dma_chunk(r, a.d);
      load_to_lds(a.k_pages + at, stage + n * 1024);
      load_to_lds(a.v_pages + at, stage + F::kMatBytes + n * 1024);
    }
  };
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i)
    if (first + i < end_tile) load(first + i);
  for (int j = first; j < end_tile; ++j) {
    if (j + kRing - 2 < end_tile)
      tile_wait<kLoads*(kRing - 2), true>();
    else
      tile_wait<0, true>();
    if (j + kRing - 1 < end_tile) load(j + kRing - 1);
    const int stage = ((j - first) % kRing) * F::kStage;
    const int left = a.prefix - j * KT;
    if (left < KT) {
      clear_values<F, KT>(ring + stage, 0, left, threadIdx.x, 64 * W);
      tile_wait<0, true>();
    }
    if (!w_live) continue;
    f32x16_t sc[1][KT / 32];
    f.scores(stage, sc);
    if (left < KT) {
#pragma unroll
      for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * kb + 8 * (e / 4) + e % 4 + 4 * (lane / 32) >= left) sc[0][kb][e] = -INFINITY;
    }
    u32x4_t p[1][KT / 16];
    f.softmax(0, sc[0], c2, p[0]);
    f.values(stage, p);
  }
  bad = __syncthreads_or(bad);
  const float sum = add_halves(f.l[0]);
  if (w_row + lane % 32 >= rows) return;
  const int64_t at = ((int64_t)b * a.n_heads + head) * (a.shared_splits + a.own_splits) + split;
  if (lane < 32) a.part_ml[at] = make_float2(f.m[0], bad ? __uint_as_float(0x7fc00000u) : sum);
  float* dst = a.part_o + at * a.d + 4 * (lane / 32);
#pragma unroll
  for (int db = 0; db < F::kDimBlocks; ++db)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int dim = 32 * db + 2 * e;
      if (!kFull && dim + 4 * (lane / 32) >= a.d) continue;
      *reinterpret_cast<float4*>(dst + dim) = make_float4(f.o[0][db][e], f.o[0][db][e + 1], f.o[0][db][e + 2], f.o[0][db][e + 3]);
    }
}

// A sequence's own part, and without a shared pass its part of the prefix.
// The keys are listed as [prefix, padded to kPrefixAlign][own].
template <int DP, bool kF16, bool kFull>
__device__ __forceinline__ void own_part(const BatchArgs& a, int wg, lds_u8 lds, float2 (&wave_ml)[kWaves][kBatchGroup]) {
  using F = Flash<DP, kF16, kFull, 1, kOwnTile>;
  constexpr int KT = kOwnTile, kLoads = 2 * F::kDmas;
  const int g = a.n_heads / a.n_kv, lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int kvh = wg % a.n_kv, split = wg / a.n_kv % a.own_splits, b = wg / (a.n_kv * a.own_splits);
  const int splits = a.shared_splits + a.own_splits;
  int n = table_at(a.lengths, b);
  if (n < 0) {  // no sequence: zeros, here or from the join
    if (splits == 1)
      for (int i = threadIdx.x; i < g * a.d; i += kWaves * kWave) a.out[((int64_t)b * a.n_heads + kvh * g) * a.d + i] = 0;
    return;
  }
  const lds_u8 ring = lds + wave * kOwnRing * F::kStage;
  const int64_t room = (int64_t)a.width << a.page_log2;
  bool bad = n > room;
  n = (int)min((int64_t)n, room);
  const int pad = (a.prefix + kPrefixAlign - 1) / kPrefixAlign * kPrefixAlign;
  // the list's visible range: from `begin` on, up to the prefix's end in its tiles and `end` in the others
  const int seen = a.window > 0 ? min(a.window, a.prefix + n) : a.prefix + n, low = a.prefix + n - seen;
  const int begin = a.shared_splits > 0 || low >= a.prefix ? pad + max(0, low - a.prefix) : low;
  const int end = n > 0 ? pad + n : a.prefix;
  const int first_tile = begin / KT, n_tiles = begin < end ? (end - 1) / KT + 1 - first_tile : 0;
  const int per = (n_tiles + a.own_splits - 1) / a.own_splits;
  const int end_tile = first_tile + min((split + 1) * per, n_tiles), first = first_tile + split * per + wave;
  const int col = min(lane % 32, g - 1), head = kvh * g + col;
  F f;
  f.init(ring, a.d);
  const float c2 = a.c2 * load_query<F, kF16>(f.q[0], a.q + b * a.q_stride + (int64_t)head * a.d, a.d);
  const int64_t kv_stride = (int64_t)a.n_kv * a.d;
  const int32_t* own_table = a.tables + (int64_t)b * a.width;
  auto load = [&](int j, int slot) {
    const lds_u8 stage = ring + slot * F::kStage;
    const bool own = j * KT >= pad;
    const int base = own ? j * KT - pad : j * KT, last = own ? n - 1 : a.prefix - 1;
    const int visible = own ? max(begin - pad, 0) : begin;
#pragma unroll
    for (int i = 0; i < F::kDmas; ++i) {
      const int r = F::dma_row(i);
      const PageRow p = page_row(own ? own_table : a.prefix_table, base + i * F::kRowsPerDma, base + r, visible, last, a.page_log2, a.n_pages);
      bad |= p.bad;
      const int64_t at = p.row * kv_stride + (int64_t)kvh * a.d + 8 * F::dma_chunk(r, a.d);
      load_to_lds(a.k_pages + at, stage + i * 1024);
      load_to_lds(a.v_pages + at, stage + F::kMatBytes + i * 1024);
    }
  };
  if (first < end_tile) load(first, 0);
  if (first + kWaves < end_tile) load(first + kWaves, 1);
  int slot = 0;
  for (int j = first; j < end_tile; j += kWaves) {
    if (j + kWaves < end_tile)
      tile_wait<kLoads, false>();
    else
      tile_wait<0, false>();
    const int stage = slot * F::kStage;
    const int from = max(0, begin - j * KT), to = min(KT, (j * KT >= pad ? end : a.prefix) - j * KT);
    const bool part = from > 0 || to < KT;
    if (part) {
      clear_values<F, KT>(ring + stage, from, to, lane, kWave);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    f32x16_t sc[1][KT / 32];
    f.scores(stage, sc);
    if (part) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = 8 * (e / 4) + e % 4 + 4 * (lane / 32);
        if (key < from || key >= to) sc[0][0][e] = -INFINITY;
      }
    }
    u32x4_t p[1][KT / 16];
    f.softmax(0, sc[0], c2, p[0]);
    f.values(stage, p);
    if (j + 2 * kWaves < end_tile) {
      tile_wait<63, false>();  // the slot's reads are done
      load(j + 2 * kWaves, slot);
    }
    slot ^= 1;
  }

  // the waves' sums: [wave][head of the group][d], rows 16 bytes apart from a multiple of the banks
  __syncthreads();
  const int stride = a.d + 4;
  typedef __attribute__((address_space(3))) float* lds_f32;
  typedef __attribute__((address_space(3))) f32x4_t* lds_f32x4;
  const lds_f32 sums = (lds_f32)lds;
  const float sum = add_halves(f.l[0]);
  if (lane % 32 < g) {
    if (lane < 32) wave_ml[wave][lane] = make_float2(f.m[0], bad ? __uint_as_float(0x7fc00000u) : sum);
    const lds_f32 dst = sums + (wave * g + lane % 32) * stride + 4 * (lane / 32);
#pragma unroll
    for (int db = 0; db < F::kDimBlocks; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int dim = 32 * db + 2 * e;
        if (!kFull && dim + 4 * (lane / 32) >= a.d) continue;
        *(lds_f32x4)(dst + dim) = f32x4_t{f.o[0][db][e], f.o[0][db][e + 1], f.o[0][db][e + 2], f.o[0][db][e + 3]};
      }
  }
  __syncthreads();
  const int quads = a.d / 4;
  for (int i = threadIdx.x; i < g * quads; i += kWaves * kWave) {
    const int h = i / quads, dim = 4 * (i - h * quads);
    float2 ml[kWaves];
    float top = -INFINITY, sink = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      ml[w] = wave_ml[w][h];
      top = fmaxf(top, ml[w].x);
    }
    if (splits == 1 && a.sinks != nullptr) top = fmaxf(top, sink = sink_log2(a.sinks[kvh * g + h]));
    const float base = top == -INFINITY ? 0.f : top;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float x = __builtin_amdgcn_exp2f(ml[w].x - base);
      const f32x4_t y = *(lds_f32x4)(sums + (w * g + h) * stride + dim);
      l = fmaf(x, ml[w].y, l);
      o.x = fmaf(x, y.x, o.x), o.y = fmaf(x, y.y, o.y), o.z = fmaf(x, y.z, o.z), o.w = fmaf(x, y.w, o.w);
    }
    const int64_t row = (int64_t)b * a.n_heads + kvh * g + h;
    if (splits == 1) {
      if (sink != -INFINITY) l += __builtin_amdgcn_exp2f(sink - base);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      *reinterpret_cast<u32x2_t*>(a.out + row * a.d + dim) = u32x2_t{pack2<false>(o.x * inv, o.y * inv), pack2<false>(o.z * inv, o.w * inv)};
    } else {
      const int64_t at = row * splits + a.shared_splits + split;
      *reinterpret_cast<float4*>(a.part_o + at * a.d + dim) = o;
      if (dim == 0) a.part_ml[at] = make_float2(top, l);
    }
  }
}

template <int DP, bool kF16, bool kFull>
__global__ __launch_bounds__(kWave * kWaves, DP == 64 ? 2 : 1) void batch_attention_kernel(BatchArgs a) {
  __shared__ __align__(1024) uint8_t lds[kBatchLds<DP>];
  __shared__ float2 wave_ml[kWaves][kBatchGroup];
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
  const bool absent = a.lengths[r / a.n_heads] < 0;
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
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (live && lane < a.d / 4)
    *reinterpret_cast<u32x2_t*>(a.out + row * a.d + dim) = u32x2_t{pack2<false>(o.x * inv, o.y * inv), pack2<false>(o.z * inv, o.w * inv)};
}

struct BatchPlan {
  int64_t shared_splits, shared_tiles, row_tiles, own_splits;
  int64_t splits() const { return shared_splits + own_splits; }
};
BatchPlan batch_plan(int64_t n_seq, int64_t n_heads, int64_t n_kv, int64_t d, int64_t prefix, int64_t max_own, int64_t window) {
  BatchPlan p{};
  const int64_t rows = n_seq * (n_heads / n_kv);
  p.row_tiles = (rows + 32 * kWaves - 1) / (32 * kWaves);
  const bool shared = prefix > 0 && window == 0 && n_seq > 1;
  int64_t keys = max_own + (shared ? 0 : prefix);
  if (window > 0 && window < keys) keys = window;
  if (shared) {
    const int64_t tile = d <= 64 ? kSharedTile<64> : kSharedTile<128>;
    const int64_t tiles = (prefix + tile - 1) / tile;
    const int64_t want = (256 + n_kv * p.row_tiles - 1) / (n_kv * p.row_tiles);
    p.shared_tiles = (tiles + want - 1) / want;
    p.shared_splits = (tiles + p.shared_tiles - 1) / p.shared_tiles;
  }
  const int64_t own_tiles = keys / kOwnTile + 2;
  const int64_t want = (512 + n_seq * n_kv - 1) / (n_seq * n_kv), most = (own_tiles + 2 * kWaves - 1) / (2 * kWaves);
  p.own_splits = want < most ? want : most;
  return p;
}

// a row of one part needs none
int64_t batch_bytes(const BatchPlan& p, int64_t n_seq, int64_t n_heads, int64_t d) {
  return p.splits() == 1 ? 0 : n_seq * n_heads * p.splits() * (4 * d + 8);
}

template <int DP, bool kF16, bool kFull>
int launch_batch(const BatchArgs& a, const BatchPlan& p, hipStream_t st) {
  const int64_t wgs = a.shared_wgs + (int64_t)a.n_seq * a.n_kv * p.own_splits;
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
  KLC_REQUIRE(x.q_stride >= x.n_heads * d && x.q_stride % 8 == 0, KLC_ERR_SHAPE,
              "klc_attn_batch: q stride %lld (a multiple of 8, no overlap)", (long long)x.q_stride);
  KLC_REQUIRE(((uintptr_t)x.q | (uintptr_t)x.k_pages | (uintptr_t)x.v_pages | (uintptr_t)x.workspace | (uintptr_t)x.out) % 16 == 0,
              KLC_ERR_ARGUMENT, "klc_attn_batch: q, pages, workspace and out must be 16-byte aligned");
  KLC_REQUIRE(x.scale > 0 && (float)x.scale > 0.f && (float)x.scale < INFINITY, KLC_ERR_ARGUMENT,
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
                    (int)x.prefix_len, (int)x.window, (int)p.shared_splits, (int)p.own_splits, (int)p.shared_tiles,
                    (int)(p.shared_splits * p.row_tiles * x.n_kv), (float)(x.scale * kLog2e)};
  const hipStream_t st = as_stream(stream);
  const bool f16 = x.kv_dtype == KLC_DTYPE_F16;
  if (d == 64) return f16 ? launch_batch<64, true, true>(a, p, st) : launch_batch<64, false, true>(a, p, st);
  if (d == 128) return f16 ? launch_batch<128, true, true>(a, p, st) : launch_batch<128, false, true>(a, p, st);
  if (d < 64) return f16 ? launch_batch<64, true, false>(a, p, st) : launch_batch<64, false, false>(a, p, st);
  return f16 ? launch_batch<128, true, false>(a, p, st) : launch_batch<128, false, false>(a, p, st);
}
