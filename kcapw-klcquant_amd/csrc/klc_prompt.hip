// Attention of whole prompts (gfx950): causal, grouped heads, sequences of
// different lengths packed one behind the other.
//
//   out_i = sum_j p_j v_j / (sum_j p_j + 2^(s - m)),  p_j = 2^(c2 q_i . k_j - m)
//
// over the visible j <= i in one pass over the keys, with the running maximum
// m and sum of klc_attn_wave.h.  The sink s joins at the end: m is the keys'
// own, as p_j is rounded to 16 bits and float16 holds nothing 2^-24 below 1
// (a sink 18 above 2,000 ordinary scores, taken into m, cost a quarter of the
// result).  A row is (token, head of the group), so that the
// heads of a group share every K and V tile and 128 or 256 rows span few
// tokens: little of the diagonal is multiplied in vain.
//
// What bounds it: long prompts by the matrix instructions and the
// exponentials beside them.  8,192 tokens of 64 heads over 8 of size 64 take
// 550 to 588 us, 550 GFLOP at 0.94 to 1.0 PFLOP/s; a loop of the same
// instructions on registers alone takes 466 to 490 us whatever its order and
// wave count.  6,778 tokens of 32 heads of size 128 take 205 to 218 us (0.89
// PFLOP/s), of which that size's loop on registers is 138 (388 ns for 32 rows
// by 32 keys).  Short prompts and windows by the start and end of a workgroup:
// 6,001 tokens in twelve with a window of 128 take 40 to 47 us for 22 us of
// bytes, and two thirds of that without any compute.
#include <math.h>

#include "klc_attn_wave.h"

namespace klc {
namespace {

struct PromptArgs {
  const uint16_t *q, *k, *v;
  const uint16_t* sinks;        // bfloat16 [n_heads] or NULL
  const int32_t* starts;        // [n_seq + 1]
  uint16_t* out;                // [tokens][n_heads][d]
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  int tokens, n_seq, n_heads, n_kv, d, window;
  float c2;                     // scale * log2(e)
};

// What a workgroup works on, the same for all its threads.
struct PromptTile {
  int begin, len;   // the sequence
  int row0, last;   // its rows (token, query head of the group) here, first and last
  int kvh, g;
};

// 64 keys a tile in LDS, of which a wave takes 32 at a time.
constexpr int kKeys = 32;
constexpr int kTileKeys = 64;

template <int DP, bool kF16, bool kFull, int RB>
struct Rows {
  using F = AttnWave<DP, kF16, kFull, RB, kKeys>;
  static constexpr int kStage = 2 * F::kStage;  // K of the tile, then V
  static constexpr int kV = 2 * F::kMatBytes;

  F f;
  int tok[RB];
  uint32_t sink[RB];  // bfloat16, of the row's head

  // the wave's rows from w_row on
  __device__ __forceinline__ void begin(const PromptArgs& a, const PromptTile& t, int w_row, lds_u8 ring) {
    const int lane = threadIdx.x % kWave;
    f.init(ring, a.d);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int row = min(w_row + 32 * rb + lane % 32, t.last);
      tok[rb] = row / t.g;
      const int head = t.kvh * t.g + row - tok[rb] * t.g;
      const uint16_t* src = a.q + (t.begin + tok[rb]) * a.q_stride + (int64_t)head * a.d;
#pragma unroll
      for (int st = 0; st < F::kSteps; ++st) {
        const int c = 2 * st + lane / 32;
        f.q[rb][st] = u32x4_t{0, 0, 0, 0};
        if (kFull || 8 * c < a.d) f.q[rb][st] = *reinterpret_cast<const u32x4_t*>(src + 8 * c);
      }
      asm volatile("" : "+v"(f.m[rb]), "+v"(f.l[rb]));  // not the constants they are: what follows from them spills
    }
  }
  // their sinks (-inf: none), asked for behind the keys: held from the start they would spill, and so would the
  // lane's rows and heads, which are worked out again from here on
  __device__ __forceinline__ void load_sinks(const PromptArgs& a, const PromptTile& t, int w_row) {
    int lane = threadIdx.x % kWave;
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int head = t.kvh * t.g + min(w_row + 32 * rb + lane % 32, t.last) - tok[rb] * t.g;
      sink[rb] = 0xff80u;
      if (a.sinks != nullptr) sink[rb] = a.sinks[head];
    }
  }

  // key k0 + 4 (lane / 32) + off is visible for low < off <= rel
  __device__ __forceinline__ int rel(int rb, int k0) const { return tok[rb] - k0 - 4 * ((int)(threadIdx.x % kWave) / 32); }
  __device__ __forceinline__ int low(const PromptArgs& a, int rb, int k0) const {
    return a.window > 0 ? rel(rb, k0) - a.window : -0x40000000;
  }
  __device__ __forceinline__ void mask(const PromptArgs& a, int k0, f32x16_t (&s)[RB][1]) const {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int off = 8 * (e / 4) + e % 4;
        s[rb][0][e] = off <= rel(rb, k0) && off > low(a, rb, k0) ? s[rb][0][e] : -INFINITY;
      }
  }

  // all rows, or those of token `only`
  __device__ __forceinline__ void store(const PromptArgs& a, const PromptTile& t, int w_row, int only = -1) const {
    int lane = threadIdx.x % kWave;
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const float s = sink_log2((uint16_t)sink[rb]), top = fmaxf(f.m[rb], s), base = top == -INFINITY ? 0.f : top;
      const float x = __builtin_amdgcn_exp2f(f.m[rb] - base), sum = fmaf(add_halves(f.l[rb]), x, __builtin_amdgcn_exp2f(s - base));
      const float inv = x / sum;  // 0 / 0 where a row's scores and its sink are all -inf: NaN, as their softmax
      const int row = w_row + 32 * rb + lane % 32, head = t.kvh * t.g + row - tok[rb] * t.g;
      const bool live = row <= t.last && (only < 0 || tok[rb] == only);
      uint16_t* dst = a.out + ((int64_t)(t.begin + tok[rb]) * a.n_heads + head) * a.d + 8 * (lane / 32);
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
              w[i][x] = pack2<kF16>(f.o[rb][db][e + 4 * i + 2 * x] * inv, f.o[rb][db][e + 4 * i + 2 * x + 1] * inv);
          const auto lo = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
          const auto hi = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
          const int at = 32 * db + 2 * e;
          if (!live || (!kFull && at + 8 * (lane / 32) >= a.d)) continue;
          *reinterpret_cast<u32x4_t*>(dst + at) = u32x4_t{lo[0], hi[0], lo[1], hi[1]};
        }
    }
  }
};

// The tiles of keys that a row of the workgroup sees, through a ring of
// kRing of them in LDS that its W waves fill together.
template <class R, int W, int kRing>
struct Tiles {
  using F = typename R::F;
  static constexpr int kDmas = 2 * F::kDmas / W;  // load instructions of K, and of V, a wave and tile
  static_assert(2 * F::kDmas % W == 0, "the tile's loads split evenly over the waves");
  const PromptArgs& a;
  const PromptTile& t;
  lds_u8 ring;
  const uint16_t *k, *v;  // of the first key
  int wave, first, count, whole;
  uint32_t k_off[kDmas], v_off[kDmas];

  __device__ __forceinline__ Tiles(const PromptArgs& args, const PromptTile& tile, lds_u8 lds) : a(args), t(tile), ring(lds) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    first = a.window > 0 ? max(0, t.row0 / t.g - a.window + 1) : 0;
    count = (t.last / t.g - first) / kTileKeys + 1;
    k = a.k + (t.begin + first) * a.k_stride + (int64_t)t.kvh * a.d;
    v = a.v + (t.begin + first) * a.v_stride + (int64_t)t.kvh * a.d;
    // tiles whose rows all exist, and whose offsets fit a load's 32 bits: no address arithmetic in vector registers
    whole = max(a.k_stride, a.v_stride) <= 0x7fffffff / (2 * kTileKeys) ? (t.len - first) / kTileKeys : 0;
#pragma unroll
    for (int i = 0; i < kDmas; ++i) {
      const int r = F::dma_row(wave + i * W), c = 8 * F::dma_chunk(r, a.d);
      k_off[i] = 2 * (uint32_t)(r * a.k_stride + c);
      v_off[i] = 2 * (uint32_t)(r * a.v_stride + c);
    }
  }
  __device__ __forceinline__ int stage(int j) const { return j % kRing * R::kStage; }
  __device__ __forceinline__ void load(int j) const {
    if (j >= count) return;
    const lds_u8 dst = ring + stage(j) + wave * 1024;
    const uint16_t *kj = k + (int64_t)j * kTileKeys * a.k_stride, *vj = v + (int64_t)j * kTileKeys * a.v_stride;
    if (j < whole) {
#pragma unroll
      for (int i = 0; i < kDmas; ++i) {
        load_to_lds(kj, k_off[i], dst + i * W * 1024);
        load_to_lds(vj, v_off[i], dst + i * W * 1024 + R::kV);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kDmas; ++i) {
        const int r = F::dma_row(wave + i * W), c = 8 * F::dma_chunk(r, a.d);
        const int64_t key = min(first + j * kTileKeys + r, t.len - 1) - (first + j * kTileKeys);
        load_to_lds(kj + key * a.k_stride + c, dst + i * W * 1024);
        load_to_lds(vj + key * a.v_stride + c, dst + i * W * 1024 + R::kV);
      }
    }
  }
  // Tile j has landed for every wave, and every wave is done with the tiles before j - 1; kAhead later tiles may
  // be in flight.
  template <int kAhead>
  __device__ __forceinline__ void arrive(int j) const {
    if (j + kAhead < count)
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * kDmas * kAhead));
    else
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  }
};

// The rows of one wave from w_row on, 32 RB of them.  Stores them, or returns
// true and stores nothing if a row of the workgroup has a NaN or infinity
// that may come from a value it must not see (0 * inf in the matrix
// instruction).
//
// The scores of the next 32 keys are multiplied while the exponentials of
// these are taken: the matrix instructions of a wave run beside its own
// vector instructions, and not only beside another wave's.
//
// With kSplit 2 two waves take the same rows, each every other 32 keys, and
// join at the end; the first of them stores.
template <int DP, bool kF16, bool kFull, int RB, int W, int kSplit, int kRing>
__device__ __forceinline__ bool prompt_rows(const PromptArgs& a, const PromptTile& t, int w_row, lds_u8 ring) {
  using R = Rows<DP, kF16, kFull, RB>;
  using F = typename R::F;
  R r;
  r.begin(a, t, w_row, ring);
  const Tiles<R, W, kRing> tiles(a, t, ring);
  // the wave's tokens, and the first and last tile that one of them sees
  const int w_lo = min(w_row, t.last) / t.g, w_hi = min(w_row + 32 * RB - 1, t.last) / t.g;
  const int from = a.window > 0 ? max(0, w_lo - a.window + 1 - tiles.first) / kTileKeys : 0;
  const int to = w_row <= t.last ? (w_hi - tiles.first) / kTileKeys : from - 1;
#pragma unroll
  for (int j = 0; j < kRing - 1; ++j) tiles.load(j);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), part = wave % kSplit;

  // what follows the scores of keys i: the mask and the maximum
  auto settle = [&](int i, f32x16_t (&s)[RB][1]) {
    const int k0 = tiles.first + i * kKeys;
    if (k0 + kKeys - 1 > w_lo || (a.window > 0 && k0 <= w_hi - a.window)) r.mask(a, k0, s);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) r.f.raise(rb, s[rb], a.c2);
  };
  f32x16_t sa[RB][1], sb[RB][1];
  // the values of the keys at `here`, whose settled scores are s, and the scores of those at `there`
  auto step = [&](int here, f32x16_t (&s)[RB][1], int there, f32x16_t (&next)[RB][1]) {
    u32x4_t p[RB][2];
    r.f.scores(there, next);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) r.f.weigh(rb, s[rb], a.c2, p[rb]);
    r.f.values(here + R::kV, p);
  };
  // tile j + 1 is there from here on, every wave is done with tile j - 1
  auto advance = [&](int j) {
    tiles.template arrive<kRing - 3>(j + 1);
    tiles.load(j + kRing - 1);
  };
  tiles.template arrive<kRing - 2>(0);
  int j = 0;
  for (; j < min(from, tiles.count); ++j) advance(j);
  if constexpr (kSplit == 2) {
    if (from <= to) {
      const int mine = part * F::kMatBytes;
      r.f.scores(tiles.stage(j) + mine, sa);
      settle(2 * j + part, sa);
      for (; j <= to; ++j) {
        advance(j);
        step(tiles.stage(j) + mine, sa, tiles.stage(j + 1) + mine, sb);  // past the last tile: scores of nothing, not used
        if (++j > to) break;
        settle(2 * j + part, sb);
        advance(j);
        step(tiles.stage(j) + mine, sb, tiles.stage(j + 1) + mine, sa);
        if (j < to) settle(2 * j + 2 + part, sa);
      }
    }
  } else if (from <= to) {
    r.f.scores(tiles.stage(j), sa);
    settle(2 * j, sa);
    for (; j <= to; ++j) {
      const int here = tiles.stage(j);
      step(here, sa, here + F::kMatBytes, sb);
      const bool both = j < to || tiles.first + (2 * j + 1) * kKeys <= w_hi;  // else no row sees the second half
      if (both) settle(2 * j + 1, sb);
      advance(j);
      if (!both) continue;
      step(here + F::kMatBytes, sb, tiles.stage(j + 1), sa);  // past the last tile: scores of nothing, not used
      if (j < to) settle(2 * j + 2, sa);
    }
  }
  for (; j < tiles.count; ++j) advance(j);

  r.load_sinks(a, t, w_row);
  bool odd = false;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int db = 0; db < F::kDimBlocks; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) odd |= !(fabsf(r.f.o[rb][db][e]) < INFINITY);
  if (__syncthreads_or(odd)) return true;
  if constexpr (kSplit == 2) {
    // the second wave's sums to the first, lane by lane: [pair][4 dims or (maximum, sum)][lane]
    constexpr int kQuads = 4 * F::kDimBlocks;
    static_assert(RB == 1 && W / 2 * (kQuads + 1) * kWave * 16 <= kRing * R::kStage, "");
    typedef __attribute__((address_space(3))) f32x4_t* lds_f32x4;
    const lds_f32x4 sums = (lds_f32x4)ring + wave / 2 * (kQuads + 1) * kWave + threadIdx.x % kWave;
    if (part == 1) {
#pragma unroll
      for (int i = 0; i < kQuads; ++i) {
        const f32x16_t& o = r.f.o[0][i / 4];
        sums[i * kWave] = f32x4_t{o[i % 4 * 4], o[i % 4 * 4 + 1], o[i % 4 * 4 + 2], o[i % 4 * 4 + 3]};
      }
      sums[kQuads * kWave] = f32x4_t{r.f.m[0], r.f.l[0], 0.f, 0.f};
    }
    __syncthreads();
    if (part == 1) return false;
    const f32x4_t other = sums[kQuads * kWave];
    const float top = fmaxf(r.f.m[0], other.x), base = top == -INFINITY ? 0.f : top;
    const float x = __builtin_amdgcn_exp2f(r.f.m[0] - base), y = __builtin_amdgcn_exp2f(other.x - base);
    r.f.m[0] = top;
    r.f.l[0] = fmaf(r.f.l[0], x, other.y * y);
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const f32x4_t o = sums[i * kWave];
#pragma unroll
      for (int e = 0; e < 4; ++e) r.f.o[0][i / 4][i % 4 * 4 + e] = fmaf(r.f.o[0][i / 4][i % 4 * 4 + e], x, o[e] * y);
    }
  }
  r.store(a, t, w_row);
  return false;
}

// The same for 32 rows, with NaN and infinities kept out of the rows that do
// not see them: one token's rows at a time, all of which see the same keys,
// with V cleared behind them.  The wave works alone, in `tile`.
template <int DP, bool kF16, bool kFull>
__device__ __forceinline__ void prompt_rows_careful(const PromptArgs& a, const PromptTile& t, int w_row, lds_u8 tile) {
  using R = Rows<DP, kF16, kFull, 1>;
  using F = typename R::F;
  const int last_tok = min(w_row + 31, t.last) / t.g;
  const uint16_t* k = a.k + t.begin * a.k_stride + (int64_t)t.kvh * a.d;
  const uint16_t* v = a.v + t.begin * a.v_stride + (int64_t)t.kvh * a.d;
  for (int tok = w_row / t.g; tok <= last_tok && w_row <= t.last; ++tok) {
    R r;
    r.begin(a, t, w_row, tile);
    for (int k0 = a.window > 0 ? max(0, tok - a.window + 1) : 0; k0 <= tok; k0 += kKeys) {
#pragma unroll
      for (int n = 0; n < F::kDmas; ++n) {
        const int row = F::dma_row(n), c = 8 * F::dma_chunk(row, a.d);
        const int64_t key = min(k0 + row, tok);
        load_to_lds(k + key * a.k_stride + c, tile + n * 1024);
        load_to_lds(v + key * a.v_stride + c, tile + F::kMatBytes + n * 1024);
      }
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
      clear_values<F, kKeys>(tile + F::kMatBytes, 0, tok - k0 + 1, threadIdx.x % kWave, kWave);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      f32x16_t s[1][1];
      r.f.scores(0, s);
      r.mask(a, k0, s);
      u32x4_t p[1][2];
      r.f.softmax(0, s[0], a.c2, p[0]);
      r.f.values(F::kMatBytes, p);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(63));  // the tile's reads are done
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    }
    r.load_sinks(a, t, w_row);
    r.store(a, t, w_row, tok);
  }
}

// Workgroup: W / kSplit times 32 RB rows of one KV head, a row being (token, query
// head of the group), so that a group's heads share every K and V tile and a
// tile of rows covers few tokens (little of the diagonal is wasted).
template <int DP, bool kF16, bool kFull, int RB, int W, int kSplit, int kRing, int kPerSimd>
__global__ __launch_bounds__(64 * W, kPerSimd) void prompt_attention_kernel(PromptArgs a) {
  constexpr int kRows = 32 * RB * W / kSplit;
  __shared__ __align__(1024) uint8_t ring[kRing * Rows<DP, kF16, kFull, RB>::kStage];
  PromptTile t;
  t.g = a.n_heads / a.n_kv;
  t.kvh = blockIdx.x % a.n_kv;
  // Tile i belongs to the last sequence s with start_s * g / kRows + s <= i: each sequence owns at least as many
  // tiles as its rows need, and the list needs no pass over the lengths.  Late tiles, the longest of a
  // sequence, go first.
  const int i = (int)(gridDim.x / a.n_kv) - 1 - (int)(blockIdx.x / a.n_kv);
  auto tile_at = [&](int begin, int s) { return (int)((int64_t)begin * t.g / kRows) + s; };
  // 64 sequences a look: the last one that starts at or before i (the first is taken to)
  int s = 0, span = a.n_seq, stride, start, found;  // it is among s .. s + span - 1
  do {
    stride = (span + kWave - 1) / kWave;
    const int at = min(s + stride * (int)(threadIdx.x % kWave), a.n_seq);
    start = min(max(a.starts[at], 0), a.tokens);
    found = __popcll(__ballot(at == s || (at < s + span && tile_at(start, at) <= i))) - 1;
    span = min(stride, span - found * stride);
    s += found * stride;
  } while (stride > 1);
  s = __builtin_amdgcn_readfirstlane(s);
  found = __builtin_amdgcn_readfirstlane(found);
  t.begin = __builtin_amdgcn_readlane(start, found);
  const int end = found + 1 < kWave ? __builtin_amdgcn_readlane(start, found + 1) : min(max(a.starts[s + 1], 0), a.tokens);
  t.len = __builtin_amdgcn_readfirstlane(end) - t.begin;
  const int64_t row0 = (int64_t)(i - tile_at(t.begin, s)) * kRows, seq_rows = (int64_t)t.len * t.g;
  if (row0 < 0 || row0 >= seq_rows) return;  // no tile of an (empty) sequence
  t.row0 = (int)row0;
  t.last = (int)(min(row0 + kRows, seq_rows) - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), w_row = t.row0 + wave / kSplit * 32 * RB;
  if (prompt_rows<DP, kF16, kFull, RB, W, kSplit, kRing>(a, t, w_row, (lds_u8)ring) && wave % kSplit == 0)
#pragma unroll 1
    for (int rb = 0; rb < RB; ++rb)
      prompt_rows_careful<DP, kF16, kFull>(a, t, w_row + 32 * rb, (lds_u8)ring + wave * 2 * 2 * kKeys * DP);
}

template <int kValue>
struct Count {
  static constexpr int value = kValue;
};

template <int DP, bool kF16, bool kFull>
int launch_prompt(const PromptArgs& a, hipStream_t st) {
  const int64_t g = a.n_heads / a.n_kv;
  // Head sizes up to 64: 64 rows a wave share the K and V reads of a long sequence, 32 a wave give three workgroups a
  // CU, whose starts and ends hide each other, and fill the chip sooner.  64 heads over 8: one sequence of 512 tokens
  // takes 13.4 us with 32 rows and 19.8 with 64, of 1,000 22 and 31, of 3,000 95 and 99, of 8,192 615 and 587; 400 of
  // 125 tokens 299 and 320, 7 of 2,857 762 and 748.  Past 64 a wave's registers take 32 rows, and eight waves share them.
  const bool short_rows = a.tokens * g * a.n_kv < 1024 * 256 || a.tokens / a.n_seq < 2048;
  // Where all rows are there at once, the longest set the time: a pair of waves a row, of half the keys each.  Size 64
  // (three workgroups of 64 rows a CU): 513 tokens 13.9 -> 12.2 us, 750 18.7 -> 15.6, but 1,000 23.4 -> 24.2, 20 of 22
  // tokens 7.2 -> 8.6, a window of 128 over 500 9.2 -> 10.1; other sizes below it would spill.  Size 128, 32 heads (one
  // of 128 rows): 600 tokens 22.6 -> 17.8, 1,500 in two rounds 46.8 -> 36.2, but five of 360 21.5 -> 27.8, a window of
  // 256 over 1,200 18.0 -> 25.4.
  const int64_t mean = a.tokens / a.n_seq, seen = a.window > 0 && a.window < mean ? a.window : mean;
  const int64_t split_wgs = (a.tokens * g / (DP == 64 ? 64 : 128) + a.n_seq) * a.n_kv;
  const bool few_rows = DP == 64 ? kFull && split_wgs <= 768 && seen >= 256
                                 : seen >= 256 && split_wgs <= (seen >= 768 ? 512 : 256);
  auto run = [&](auto rb, auto w, auto split, auto ring, auto per_simd) {
    constexpr int RB = decltype(rb)::value, W = decltype(w)::value, kSplit = decltype(split)::value;
    const int64_t tiles = a.tokens * g / (32 * RB * W / kSplit) + a.n_seq;
    prompt_attention_kernel<DP, kF16, kFull, RB, W, kSplit, decltype(ring)::value, decltype(per_simd)::value>
        <<<(unsigned)(tiles * a.n_kv), 64 * W, 0, st>>>(a);
  };
  if constexpr (DP == 128) {
    if (few_rows)
      run(Count<1>{}, Count<8>{}, Count<2>{}, Count<4>{}, Count<2>{});
    else
      run(Count<1>{}, Count<8>{}, Count<1>{}, Count<4>{}, Count<2>{});
  } else if (few_rows) {
    if constexpr (kFull) run(Count<1>{}, Count<4>{}, Count<2>{}, Count<3>{}, Count<3>{});
  } else if (short_rows) {
    run(Count<1>{}, Count<4>{}, Count<1>{}, Count<3>{}, Count<3>{});
  } else {
    run(Count<2>{}, Count<4>{}, Count<1>{}, Count<4>{}, Count<2>{});
  }
  return check_launch("prompt_attention_kernel");
}

}  // namespace
}  // namespace klc

using namespace klc;

extern "C" int klc_attn_prompt(const klc_attn_prompt_args* args, void* stream) {
  KLC_REQUIRE(args != nullptr, KLC_ERR_ARGUMENT, "klc_attn_prompt: null pointer");
  const klc_attn_prompt_args& x = *args;
  KLC_REQUIRE(x.q && x.k && x.v && x.starts && x.out, KLC_ERR_ARGUMENT, "klc_attn_prompt: null pointer");
  KLC_REQUIRE(x.n_heads > 0 && x.n_kv > 0 && x.n_heads % x.n_kv == 0 && x.n_heads <= 4096 && x.head_dim >= 8 &&
                  x.head_dim % 8 == 0 && x.head_dim <= 128,
              KLC_ERR_SHAPE, "klc_attn_prompt: heads %lld / %lld, head_dim %lld (8..128, multiple of 8)",
              (long long)x.n_heads, (long long)x.n_kv, (long long)x.head_dim);
  const int64_t g = x.n_heads / x.n_kv;
  KLC_REQUIRE(x.tokens > 0 && x.n_seq > 0 && x.tokens < ((int64_t)1 << 30) && x.tokens * g < ((int64_t)1 << 30) &&
                  x.n_seq < ((int64_t)1 << 20) && (x.tokens * g / 64 + x.n_seq) * x.n_kv < ((int64_t)1 << 31),
              KLC_ERR_ARGUMENT, "klc_attn_prompt: %lld tokens in %lld sequences (tokens * group < 2^30)",
              (long long)x.tokens, (long long)x.n_seq);
  KLC_REQUIRE(x.q_stride >= x.n_heads * x.head_dim && x.k_stride >= x.n_kv * x.head_dim &&
                  x.v_stride >= x.n_kv * x.head_dim && (x.q_stride | x.k_stride | x.v_stride) % 8 == 0,
              KLC_ERR_SHAPE, "klc_attn_prompt: token strides %lld, %lld, %lld (multiples of 8, no overlap)",
              (long long)x.q_stride, (long long)x.k_stride, (long long)x.v_stride);
  KLC_REQUIRE(((uintptr_t)x.q | (uintptr_t)x.k | (uintptr_t)x.v | (uintptr_t)x.out) % 16 == 0, KLC_ERR_ARGUMENT,
              "klc_attn_prompt: q, k, v and out must be 16-byte aligned");
  KLC_REQUIRE(x.window >= 0 && x.window < ((int64_t)1 << 30) && x.scale > 0 && (float)x.scale > 0.f &&
                  (float)(x.scale * kLog2e) < INFINITY,
              KLC_ERR_ARGUMENT, "klc_attn_prompt: window %lld, scale %g", (long long)x.window, x.scale);
  KLC_REQUIRE(x.dtype == KLC_DTYPE_BF16 || x.dtype == KLC_DTYPE_F16, KLC_ERR_UNSUPPORTED,
              "klc_attn_prompt: dtype %lld (bfloat16 or float16)", (long long)x.dtype);
  auto in = [](const void* p) { return static_cast<const uint16_t*>(p); };
  const PromptArgs a{in(x.q), in(x.k), in(x.v), in(x.sinks), static_cast<const int32_t*>(x.starts),
                     static_cast<uint16_t*>(x.out), x.q_stride, x.k_stride, x.v_stride, (int)x.tokens, (int)x.n_seq,
                     (int)x.n_heads, (int)x.n_kv, (int)x.head_dim, (int)x.window, (float)(x.scale * kLog2e)};
  const hipStream_t st = as_stream(stream);
  const bool f16 = x.dtype == KLC_DTYPE_F16;
  if (x.head_dim == 64) return f16 ? launch_prompt<64, true, true>(a, st) : launch_prompt<64, false, true>(a, st);
  if (x.head_dim == 128) return f16 ? launch_prompt<128, true, true>(a, st) : launch_prompt<128, false, true>(a, st);
  if (x.head_dim < 64) return f16 ? launch_prompt<64, true, false>(a, st) : launch_prompt<64, false, false>(a, st);
  return f16 ? launch_prompt<128, true, false>(a, st) : launch_prompt<128, false, false>(a, st);
}
