// The weights that new tokens' queries give the cached keys, summed key by key
// (gfx950):
//
//   w_j (+)= sum_i 2^(c2 q_i . k_j - l_i),  l_i = log2(e) lse_i
//
// over the rows i, (new token, head of the group), that see key j.  The new
// tokens' own keys start at the sum, the others have it added.
//
// A wave keeps 64 keys in registers as the matrix instruction's columns, and
// rows come past in tiles of 32 through LDS: a lane has 16 rows of its one
// key, so that the sums over rows never leave it but at the end.  KW waves
// take other keys of the same rows, 4 / KW others rows of the same keys.
#include <math.h>

#include "klc_paged_tiles.h"

namespace klc {
namespace {

constexpr int kWaveKeys = 64;
constexpr int kTileRows32 = 32;

struct KeyWeightArgs {
  const uint16_t* q;                // bfloat16 [tokens] rows
  const float* lse;                 // [tokens][n_heads]
  const uint16_t* k_pages;          // [n_pages][page][n_kv][d]
  const int32_t *tables, *lengths;  // [n_seq][width], [n_seq]
  const int32_t *starts, *rows;     // [n_seq + 1], [n_seq]
  float* weights;                   // [n_rows][n_kv][capacity]
  int64_t q_stride, capacity;
  int n_seq, n_rows, n_heads, n_kv, d, n_pages, page_log2, width, window, first, blocks;
  float c2;
};

template <int DP, bool kF16, bool kFull, int KW>
__global__ __launch_bounds__(kWave * kWaves, 2) void key_weights_kernel(KeyWeightArgs a) {
  using F = AttnWave<DP, kF16, kFull, 1, kTileRows32>;
  constexpr int RW = kWaves / KW, kStepRows = RW * kTileRows32, kBlock = KW * kWaveKeys;
  constexpr int kThreads = kWave * kWaves, kPasses = kStepRows * F::kChunks / kThreads, kPassRows = kThreads / F::kChunks;
  static_assert(kPasses * kPassRows == kStepRows, "");
  __shared__ __align__(1024) uint8_t tile[2][kStepRows * F::kRowBytes];
  __shared__ __align__(16) float factor[2][kStepRows], log_norm[2][kStepRows];
  __shared__ __align__(16) int place[2][kStepRows];
  __shared__ double joined[kWaves][kWave];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane / 32;
  const int kw = wave % KW, rw = wave / KW;
  const int kvh = blockIdx.x % a.n_kv, block = blockIdx.x / a.n_kv % a.blocks, seq = blockIdx.x / (a.n_kv * a.blocks);
  const int g = a.n_heads / a.n_kv;
  const int begin = table_at(a.starts, seq), count = table_at(a.starts, seq + 1) - begin;
  const int64_t room = (int64_t)a.width << a.page_log2;
  const int asked = table_at(a.lengths, seq), n = (int)min((int64_t)max(asked, 0), room), out_row = table_at(a.rows, seq);
  const int base = n - count;
  const int b0 = block * kBlock, b1 = min(b0 + kBlock, n) - 1;  // the block's keys
  if (b0 >= n) return;
  // the tokens that see one of them
  const int t_lo = max(0, b0 - base), t_hi = a.window > 0 && b0 >= a.first ? min(count - 1, b1 + a.window - 1 - base) : count - 1;
  if (t_lo > t_hi || (unsigned)out_row >= (unsigned)a.n_rows) return;
  const int r_lo = t_lo * g, r_end = (t_hi + 1) * g;

  // rows of a step to LDS, by all threads: chunk threadIdx % kChunks of every kPassRows-th row
  const int chunk = threadIdx.x % F::kChunks;
  u32x4_t held[kPasses];
  float held_lse[kPasses];
  int held_place[kPasses];
  auto fetch = [&](int row0) {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = row0 + i * kPassRows + (int)threadIdx.x / F::kChunks;
      const bool live = row < r_end;
      const int tok = min(row, r_end - 1) / g, head = kvh * g + min(row, r_end - 1) - tok * g;
      held[i] = u32x4_t{0, 0, 0, 0};
      if (kFull || 8 * chunk < a.d)
        held[i] = *reinterpret_cast<const u32x4_t*>(a.q + (begin + tok) * a.q_stride + (int64_t)head * a.d + 8 * chunk);
      held_lse[i] = a.lse[(int64_t)(begin + tok) * a.n_heads + head];
      held_place[i] = live ? base + tok : -1;
    }
  };
  auto put = [&](int slot) {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = i * kPassRows + (int)threadIdx.x / F::kChunks;
      float c2 = a.c2;
      if constexpr (kF16) {
        // times a power of two that brings the row's largest value to [1, 2), as the attention kernels' queries
        typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
        u16x2_t pair = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pair = __builtin_elementwise_max(pair, __builtin_bit_cast(u16x2_t, held[i][e] & 0x7fff7fffu));
        uint32_t most = (uint32_t)max(pair.x, pair.y) << 16;
#pragma unroll
        for (int off = 1; off < F::kChunks; off <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, off));
        int ex = (int)(most >> 23) - 127;
        if (most >= 0x7f800000u || most == 0) ex = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          held[i][e] = pack2<true>(__builtin_amdgcn_ldexpf(__uint_as_float(held[i][e] << 16), -ex),
                                   __builtin_amdgcn_ldexpf(__uint_as_float(held[i][e] & 0xffff0000u), -ex));
        c2 *= __builtin_amdgcn_ldexpf(1.f, ex);
      }
      *reinterpret_cast<u32x4_t*>(tile[slot] + row * F::kRowBytes + ((chunk ^ F::swizzle(row % 32)) << 4)) = held[i];
      if (chunk == 0) {
        factor[slot][row] = c2;
        log_norm[slot][row] = held_lse[i] * kLog2e;
        place[slot][row] = held_place[i];
      }
    }
  };
  fetch(r_lo);

  // the wave's keys
  u32x4_t k[2][F::kSteps];
  int key[2];
  bool bad[2];
  const int32_t* table = a.tables + (int64_t)seq * a.width;
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    key[kb] = b0 + kw * kWaveKeys + 32 * kb + lane % 32;
    const int at = min(key[kb], b1), page = table[at >> a.page_log2];
    bad[kb] = (unsigned)page >= (unsigned)a.n_pages || asked > room;
    const uint16_t* src = a.k_pages + ((((int64_t)(bad[kb] ? 0 : page) << a.page_log2) + (at & ((1 << a.page_log2) - 1))) * a.n_kv + kvh) * a.d;
    load_query<F>(k[kb], src, a.d);
  }
  put(0);
  __syncthreads();
  double total[2] = {0., 0.};
  int slot = 0;
  for (int row0 = r_lo; row0 < r_end; row0 += kStepRows, slot ^= 1) {
    const bool more = row0 + kStepRows < r_end;
    if (more) fetch(row0 + kStepRows);
    const int mine = row0 + rw * kTileRows32;
    if (mine < r_end) {
      f32x16_t s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
#pragma unroll
      for (int st = 0; st < F::kSteps; ++st) {
        if (!kFull && 16 * st >= a.d) break;
        const u32x4_t q = *reinterpret_cast<const u32x4_t*>(tile[slot] + (rw * 32 + lane % 32) * F::kRowBytes +
                                                            (((2 * st + half) ^ F::swizzle(lane % 32)) << 4));
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) s[kb] = mfma32<kF16>(q, k[kb][st], s[kb]);
      }
      // all of its rows see all keys of the wave
      const int first_pos = base + mine / g, last_pos = base + (mine + 31) / g;
      const int k_lo = b0 + kw * kWaveKeys, k_hi = k_lo + kWaveKeys - 1;
      const bool whole = mine + 32 <= r_end && k_hi <= first_pos && (a.window == 0 || k_lo > last_pos - a.window);
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int at = rw * 32 + 8 * q4 + 4 * half;
        if (mine + 8 * q4 >= r_end) break;
        const f32x4_t norm = *reinterpret_cast<const f32x4_t*>(&log_norm[slot][at]);
        f32x4_t c2 = {a.c2, a.c2, a.c2, a.c2};
        if constexpr (kF16) c2 = *reinterpret_cast<const f32x4_t*>(&factor[slot][at]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) s[kb][4 * q4 + e] = __builtin_amdgcn_exp2f(fmaf(s[kb][4 * q4 + e], c2[e], -norm[e]));
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int pos = place[slot][at + e];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
              if (key[kb] > pos || (a.window > 0 && key[kb] <= pos - a.window && key[kb] >= a.first)) s[kb][4 * q4 + e] = 0.f;
          }
        }
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        float sum = 0.f;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          if (mine + 8 * q4 < r_end) sum += (s[kb][4 * q4] + s[kb][4 * q4 + 1]) + (s[kb][4 * q4 + 2] + s[kb][4 * q4 + 3]);
        total[kb] += (double)sum;  // as many sums as the chunk has tiles of rows
      }
    }
    if (more) put(slot ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) total[kb] += __shfl_xor(total[kb], 32);
  // lane l has key l of the wave's 64
  double sum = half == 0 ? total[0] : total[1];
  const int own = b0 + kw * kWaveKeys + lane;
  const bool wrong = half == 0 ? bad[0] : bad[1];
  if constexpr (RW > 1) {
    joined[wave][lane] = sum;
    __syncthreads();
    if (rw != 0) return;
#pragma unroll
    for (int i = 1; i < RW; ++i) sum += joined[i * KW + kw][lane];
  }
  if (own > b1 || own >= a.capacity) return;
  float* dst = a.weights + ((int64_t)out_row * a.n_kv + kvh) * a.capacity + own;
  if (wrong) sum = (double)__uint_as_float(0x7fc00000u);
  *dst = (float)(own >= base ? sum : (double)*dst + sum);
}

template <int DP, bool kF16, bool kFull, int KW>
void run_key_weights(KeyWeightArgs a, hipStream_t st) {
  a.blocks = (int)((((int64_t)a.width << a.page_log2) + KW * kWaveKeys - 1) / (KW * kWaveKeys));
  key_weights_kernel<DP, kF16, kFull, KW><<<(unsigned)((int64_t)a.n_seq * a.blocks * a.n_kv), kWave * kWaves, 0, st>>>(a);
}

template <int DP, bool kF16, bool kFull>
int launch_key_weights(const KeyWeightArgs& a, int64_t tokens, hipStream_t st) {
  const int64_t keys = (int64_t)a.width << a.page_log2, rows = tokens / a.n_seq * (a.n_heads / a.n_kv);
  const int64_t wgs = a.n_seq * a.n_kv * ((keys + 4 * kWaveKeys - 1) / (4 * kWaveKeys));
  if (rows <= 32 || wgs >= 768)
    run_key_weights<DP, kF16, kFull, 4>(a, st);
  else
    run_key_weights<DP, kF16, kFull, 1>(a, st);
  return check_launch("key_weights_kernel");
}

}  // namespace
}  // namespace klc

using namespace klc;

extern "C" int klc_attn_key_weights(const klc_attn_key_weights_args* args, void* stream) {
  KLC_REQUIRE(args != nullptr, KLC_ERR_ARGUMENT, "klc_attn_key_weights: null pointer");
  const klc_attn_key_weights_args& x = *args;
  KLC_REQUIRE(x.q && x.lse && x.k_pages && x.lengths && x.plan && x.rows && x.weights && (x.tables || x.table_width == 0),
              KLC_ERR_ARGUMENT, "klc_attn_key_weights: null pointer");
  const int64_t d = x.head_dim;
  KLC_REQUIRE(x.n_heads > 0 && x.n_kv > 0 && x.n_heads % x.n_kv == 0 && x.n_heads <= 4096 && d >= 8 && d % 8 == 0 && d <= 128,
              KLC_ERR_SHAPE, "klc_attn_key_weights: heads %lld / %lld, head_dim %lld (8..128, multiple of 8)",
              (long long)x.n_heads, (long long)x.n_kv, (long long)d);
  KLC_REQUIRE(x.page_size >= 16 && x.page_size <= 4096 && (x.page_size & (x.page_size - 1)) == 0 && x.n_pages > 0 &&
                  x.n_pages < ((int64_t)1 << 31) && x.n_pages * x.page_size < ((int64_t)1 << 31) && x.table_width >= 0 &&
                  x.table_width < ((int64_t)1 << 25) && x.table_width * x.page_size < ((int64_t)1 << 29),
              KLC_ERR_SHAPE, "klc_attn_key_weights: %lld pages of %lld tokens (a power of two, 16..4096), tables of %lld",
              (long long)x.n_pages, (long long)x.page_size, (long long)x.table_width);
  KLC_REQUIRE(x.n_seq > 0 && x.n_seq < ((int64_t)1 << 20) && x.tokens >= x.n_seq && x.tokens * (x.n_heads / x.n_kv) < ((int64_t)1 << 30) &&
                  x.n_rows > 0 && x.n_rows < ((int64_t)1 << 31) && x.capacity > 0 && x.capacity < ((int64_t)1 << 31) &&
                  x.n_seq * x.n_kv * (x.table_width * x.page_size / kWaveKeys + 1) < ((int64_t)1 << 31),
              KLC_ERR_ARGUMENT, "klc_attn_key_weights: %lld tokens of %lld sequences, %lld rows of %lld weights", (long long)x.tokens,
              (long long)x.n_seq, (long long)x.n_rows, (long long)x.capacity);
  KLC_REQUIRE(x.q_stride >= x.n_heads * d && x.q_stride % 8 == 0, KLC_ERR_SHAPE,
              "klc_attn_key_weights: q stride %lld (a multiple of 8, no overlap)", (long long)x.q_stride);
  KLC_REQUIRE(((uintptr_t)x.q | (uintptr_t)x.k_pages) % 16 == 0 && ((uintptr_t)x.lse | (uintptr_t)x.weights) % 4 == 0, KLC_ERR_ARGUMENT,
              "klc_attn_key_weights: q and pages must be 16-byte aligned");
  KLC_REQUIRE(x.window >= 0 && x.window < ((int64_t)1 << 30) && x.first >= 0 && x.first < ((int64_t)1 << 29) &&
                  (x.first == 0 || x.window > 0) && x.scale > 0 && (float)x.scale > 0.f && (float)(x.scale * kLog2e) < INFINITY,
              KLC_ERR_ARGUMENT, "klc_attn_key_weights: window %lld, %lld first tokens, scale %g", (long long)x.window,
              (long long)x.first, x.scale);
  KLC_REQUIRE(x.kv_dtype == KLC_DTYPE_BF16 || x.kv_dtype == KLC_DTYPE_F16, KLC_ERR_UNSUPPORTED,
              "klc_attn_key_weights: kv_dtype %lld (bfloat16 or float16)", (long long)x.kv_dtype);
  if (x.table_width == 0) return KLC_OK;  // no key
  auto in = [](const void* v) { return static_cast<const uint16_t*>(v); };
  auto index = [](const void* v) { return static_cast<const int32_t*>(v); };
  int page_log2 = 0;
  while ((1 << page_log2) < x.page_size) ++page_log2;
  const KeyWeightArgs a{in(x.q), static_cast<const float*>(x.lse), in(x.k_pages), index(x.tables), index(x.lengths),
                        index(x.plan), index(x.rows), static_cast<float*>(x.weights), x.q_stride, x.capacity, (int)x.n_seq,
                        (int)x.n_rows, (int)x.n_heads, (int)x.n_kv, (int)d, (int)x.n_pages, page_log2, (int)x.table_width,
                        (int)x.window, (int)x.first, 0, (float)(x.scale * kLog2e)};
  const hipStream_t st = as_stream(stream);
  const bool f16 = x.kv_dtype == KLC_DTYPE_F16;
  const int64_t t = x.tokens;
  if (d == 64) return f16 ? launch_key_weights<64, true, true>(a, t, st) : launch_key_weights<64, false, true>(a, t, st);
  if (d == 128) return f16 ? launch_key_weights<128, true, true>(a, t, st) : launch_key_weights<128, false, true>(a, t, st);
  if (d < 64) return f16 ? launch_key_weights<64, true, false>(a, t, st) : launch_key_weights<64, false, false>(a, t, st);
  return f16 ? launch_key_weights<128, true, false>(a, t, st) : launch_key_weights<128, false, false>(a, t, st);
}
