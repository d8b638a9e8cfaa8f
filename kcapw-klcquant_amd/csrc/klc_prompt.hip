// Attention of whole prompts (gfx950): causal, grouped heads, sequences of
// different lengths packed one behind the other.
#include <math.h>

#include "klc_flash.h"

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

// One step of the ring: tile j has landed for every wave of the workgroup and
// every wave is done with tile j - 1.
template <int kOutstanding>
__device__ __forceinline__ void tile_barrier() {
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(kOutstanding));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

constexpr int kPromptRing = 3;

// What a workgroup works on, the same for all its threads.
struct PromptTile {
  int begin, len;   // the sequence
  int row0, last;   // its rows (token, query head of the group) here, first and last
  int kvh, g;
};

// The rows of one wave from w_row on, 32 RB of them, over every tile of keys
// that a row of the workgroup sees.  Without kCareful it stores nothing and
// returns true if a result has a NaN or infinity that may come from a value
// the row must not see (0 * inf in the matrix instruction); kCareful keeps
// those out.
template <int DP, bool kF16, bool kFull, int RB, int W, int KT, bool kCareful>
__device__ __forceinline__ bool prompt_rows(const PromptArgs& a, const PromptTile& t, int w_row, lds_u8 ring) {
  using F = Flash<DP, kF16, kFull, RB, KT>;
  constexpr int kLoads = 2 * F::kDmas / W;  // load instructions of a wave and tile
  static_assert(F::kDmas % W == 0, "the tile's loads split evenly over the waves");
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int tok_lo = t.row0 / t.g, tok_hi = t.last / t.g;  // tokens of the workgroup's rows, and of the wave's
  const int w_lo = min(w_row, t.last) / t.g, w_hi = min(w_row + 32 * RB - 1, t.last) / t.g;
  const bool w_live = w_row <= t.last;

  F f;
  f.init(ring, a.d);
  int tok[RB], head[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = min(w_row + 32 * rb + lane % 32, t.last);
    tok[rb] = row / t.g;
    head[rb] = t.kvh * t.g + row - tok[rb] * t.g;
    const uint16_t* src = a.q + (t.begin + tok[rb]) * a.q_stride + (int64_t)head[rb] * a.d;
#pragma unroll
    for (int st = 0; st < F::kSteps; ++st) {
      const int c = 2 * st + lane / 32;
      f.q[rb][st] = u32x4_t{0, 0, 0, 0};
      if (kFull || 8 * c < a.d) f.q[rb][st] = *reinterpret_cast<const u32x4_t*>(src + 8 * c);
    }
    if (a.sinks != nullptr) {
      const float sink = sink_log2(a.sinks[head[rb]]);
      f.m[rb] = sink;
      f.l[rb] = sink == -INFINITY || lane >= 32 ? 0.f : 1.f + (sink - sink);
    }
  }

  const int first = a.window > 0 ? max(0, tok_lo - a.window + 1) / KT * KT : 0;
  const int n_tiles = (tok_hi - first) / KT + 1;
  const uint16_t* kb = a.k + t.begin * a.k_stride + (int64_t)t.kvh * a.d;
  const uint16_t* vb = a.v + t.begin * a.v_stride + (int64_t)t.kvh * a.d;
  auto load = [&](int j) {
    const int base = first + j * KT, stage = (j % kPromptRing) * F::kStage;
#pragma unroll
    for (int i = 0; i < F::kDmas / W; ++i) {
      const int n = wave + i * W, r = F::dma_row(n);
      const int64_t key = min(base + r, t.len - 1);
      const int c = 8 * F::dma_chunk(r, a.d);
      const lds_u8 dst = ring + stage + n * 1024;
      load_to_lds(kb + key * a.k_stride + c, dst);
      load_to_lds(vb + key * a.v_stride + c, dst + F::kMatBytes);
    }
  };
#pragma unroll
  for (int j = 0; j < kPromptRing - 1; ++j)
    if (j < n_tiles) load(j);
  for (int j = 0; j < n_tiles; ++j) {
    if (j + 1 < n_tiles)
      tile_barrier<kLoads*(kPromptRing - 2)>();
    else
      tile_barrier<0>();
    if (j + kPromptRing - 1 < n_tiles) load(j + kPromptRing - 1);
    const int k0 = first + j * KT, stage = (j % kPromptRing) * F::kStage;
    if (!w_live || k0 > w_hi || (a.window > 0 && k0 + KT - 1 <= w_lo - a.window)) continue;
    const bool masked = k0 + KT - 1 > w_lo || (a.window > 0 && k0 <= w_hi - a.window);
    f32x16_t sc[RB][KT / 32];
    f.scores(stage, sc);
    u32x4_t p[RB][KT / 16];
    // key k0 + 4 (lane / 32) + off is visible for low < off <= rel
    auto rel = [&](int rb) { return tok[rb] - k0 - 4 * (lane / 32); };
    auto low = [&](int rb) { return a.window > 0 ? rel(rb) - a.window : -0x40000000; };
    if (masked) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int b = 0; b < KT / 32; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int off = 32 * b + 8 * (e / 4) + e % 4;
            sc[rb][b][e] = off <= rel(rb) && off > low(rb) ? sc[rb][b][e] : -INFINITY;
          }
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) f.softmax(rb, sc[rb], a.c2, p[rb]);
    if (!kCareful || !masked) {
      f.values(stage, p);
    } else {
      u32x4_t seen[RB][KT / 16];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int x = 0; x < KT / 16; ++x)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const int off = 16 * x + 8 * (e / 4) + e % 4;
            auto one = [&](int o) { return o <= rel(rb) && o > low(rb) ? 1.f : 0.f; };
            seen[rb][x][e / 2] = pack2<kF16>(one(off), one(off + 1));
          }
      f.values_careful(stage, p, seen);
    }
  }
  if constexpr (!kCareful) {
    bool odd = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int db = 0; db < F::kDimBlocks; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) odd |= !(fabsf(f.o[rb][db][e]) < INFINITY);
    if (__syncthreads_or(odd)) return true;
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const float sum = add_halves(f.l[rb]);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no key and no sink: zeros
    if (w_row + 32 * rb + lane % 32 > t.last) continue;
    uint16_t* dst = a.out + ((int64_t)(t.begin + tok[rb]) * a.n_heads + head[rb]) * a.d + 4 * (lane / 32);
#pragma unroll
    for (int db = 0; db < F::kDimBlocks; ++db)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int at = 32 * db + 2 * e;
        if (!kFull && at + 4 * (lane / 32) >= a.d) continue;
        const u32x2_t w = {pack2<kF16>(f.o[rb][db][e] * inv, f.o[rb][db][e + 1] * inv),
                           pack2<kF16>(f.o[rb][db][e + 2] * inv, f.o[rb][db][e + 3] * inv)};
        *reinterpret_cast<u32x2_t*>(dst + at) = w;
      }
  }
  return false;
}

// Workgroup: W waves x 32 RB rows of one KV head, a row being (token, query
// head of the group), so that a group's heads share every K and V tile and a
// tile of rows covers few tokens (little of the diagonal is wasted).
template <int DP, bool kF16, bool kFull, int RB, int W, int KT>
__global__ __launch_bounds__(64 * W, DP == 64 ? 2 : 1) void prompt_attention_kernel(PromptArgs a) {
  constexpr int kRows = 32 * RB * W;
  __shared__ __align__(1024) uint8_t ring[kPromptRing * Flash<DP, kF16, kFull, RB, KT>::kStage];
  PromptTile t;
  t.g = a.n_heads / a.n_kv;
  t.kvh = blockIdx.x % a.n_kv;
  // Tile i belongs to the last sequence s with start_s * g / kRows + s <= i: each sequence owns at least as many
  // tiles as its rows need, and the list needs no pass over the lengths.  Late tiles, the longest of a
  // sequence, go first.
  const int i = (int)(gridDim.x / a.n_kv) - 1 - (int)(blockIdx.x / a.n_kv);
  auto start_of = [&](int s) { return min(max(a.starts[s], 0), a.tokens); };
  auto tile_of = [&](int s) { return (int)((int64_t)start_of(s) * t.g / kRows) + s; };
  int s = 0, step = 1;
  while (step < a.n_seq) step <<= 1;
  for (; step > 0; step >>= 1)
    if (s + step < a.n_seq && tile_of(s + step) <= i) s += step;
  s = __builtin_amdgcn_readfirstlane(s);
  t.begin = __builtin_amdgcn_readfirstlane(start_of(s));
  t.len = __builtin_amdgcn_readfirstlane(start_of(s + 1)) - t.begin;
  const int64_t row0 = (int64_t)(i - tile_of(s)) * kRows, seq_rows = (int64_t)t.len * t.g;
  if (row0 < 0 || row0 >= seq_rows) return;  // no tile of an (empty) sequence
  t.row0 = (int)row0;
  t.last = (int)(min(row0 + kRows, seq_rows) - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), w_row = t.row0 + wave * 32 * RB;
  if (prompt_rows<DP, kF16, kFull, RB, W, KT, false>(a, t, w_row, (lds_u8)ring))
#pragma unroll 1
    for (int rb = 0; rb < RB; ++rb) {
      prompt_rows<DP, kF16, kFull, 1, W, KT, true>(a, t, w_row + 32 * rb, (lds_u8)ring);
      __syncthreads();
    }
}

template <int DP, bool kF16, bool kFull>
int launch_prompt(const PromptArgs& a, hipStream_t st) {
  const int64_t g = a.n_heads / a.n_kv;
  constexpr int RB = DP == 64 ? 2 : 1, W = 4, KT = 64;
  const int64_t tiles = a.tokens * g / (32 * RB * W) + a.n_seq;
  prompt_attention_kernel<DP, kF16, kFull, RB, W, KT><<<(unsigned)(tiles * a.n_kv), 64 * W, 0, st>>>(a);
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
                  (float)x.scale < INFINITY,
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
