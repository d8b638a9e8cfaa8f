// The weights that new tokens' queries give the cached keys, summed key by key
// (gfx950):
//
//   w_j (+)= sum_i 2^(c2 q_i . k_j - l_i),  l_i = log2(e) lse_i
//
// over the rows i, (new token, head of the group), that see key j.  The new
// tokens' own keys start at the sum, the others have it added.
//
// A wave keeps 64 keys in registers as the matrix instruction's columns, and
// rows come past in tiles of 32 through LDS, for the four waves of a
// workgroup: a lane has 16 rows of its one key, so that the sums over rows
// never leave it but at the end.  Long chunks' rows go to several workgroups,
// as many as the plan says, whose float64 sums a second launch adds in their
// order.
//
// What bounds it (64 heads over 8 of size 64): the exponentials and the two
// instructions beside each, 46 us of the 66 that 1,000 tokens over 4,000 take,
// 164 for a prompt of 4,096; steps by memory, 64 of 1,000 to 2,000 keys in 26
// us (4.0 TB/s), and the start and end of a workgroup for 256 keys.
#include <math.h>

#include <algorithm>

#include "klc_paged_tiles.h"

namespace klc {
namespace {

constexpr int kWaveKeys = 64;
constexpr int kBlockKeys = kWaves * kWaveKeys;
constexpr int kRows = 32;  // of a tile
constexpr int kPartTiles = 8;

struct KeyWeightArgs {
  const uint16_t* q;                // bfloat16 [tokens] rows
  const float* lse;                 // [tokens][n_heads]
  const uint16_t *k_pages, *v_pages;  // [n_pages][page][n_kv][d]; values are not read
  const int32_t *tables, *lengths;  // [n_seq][width], [n_seq]
  const int32_t *starts, *rows;     // [n_seq + 1], [n_seq]
  const int32_t* items;             // of the plan: sequence, part of its rows, parts, its first part among the joined
  float* weights;                   // [n_rows][n_kv][capacity]
  double* part;                     // [parts][n_kv][width * page]
  int64_t q_stride, capacity;
  int n_rows, n_heads, n_kv, d, n_pages, page_log2, width, window, first, blocks;
  float c2;
};

// The keys of a block that some new token sees, and the rows that see one of them.
struct BlockRows {
  int base, last;     // the first new token's key, the block's last key
  int row0, row_end;  // none: row0 >= row_end
  __device__ __forceinline__ BlockRows(const KeyWeightArgs& a, int count, int n, int b0) {
    const int g = a.n_heads / a.n_kv;
    base = n - count;
    last = min(b0 + kBlockKeys, n) - 1;
    const int t_lo = max(0, b0 - base);
    const int t_hi = a.window > 0 && b0 >= a.first ? (int)min((int64_t)count - 1, (int64_t)last + a.window - 1 - base) : count - 1;
    row0 = t_lo * g;
    row_end = b0 < n ? (t_hi + 1) * g : 0;
  }
  // rows of a part, in whole tiles: one part is not cut, others have at least kPartTiles
  __device__ __forceinline__ int per(int parts) const {
    const int tiles = (row_end - row0 + kRows - 1) / kRows;
    return (parts == 1 ? tiles : max((tiles + parts - 1) / parts, kPartTiles)) * kRows;
  }
};

__device__ __forceinline__ void write_weight(const KeyWeightArgs& a, int out_row, int kvh, int key, int base, double sum) {
  if (key >= a.capacity) return;
  float* dst = a.weights + ((int64_t)out_row * a.n_kv + kvh) * a.capacity + key;
  *dst = (float)(key >= base ? sum : (double)*dst + sum);
}

template <int DP, bool kF16, bool kFull>
__global__ __launch_bounds__(kWave * kWaves, DP == 64 ? 4 : 2) void key_weights_kernel(KeyWeightArgs a) {
  using F = AttnWave<DP, kF16, kFull, 1, kRows>;
  constexpr int kThreads = kWave * kWaves, kPassRows = kThreads / F::kChunks, kPasses = kRows / kPassRows;
  static_assert(kPasses * kPassRows == kRows, "");
  // the block's keys on their way into registers, then two tiles of rows
  constexpr int kTileBytes = kRows * F::kRowBytes, kWaveBytes = 8192, kStageKeys = kWaveBytes / F::kRowBytes;
  __shared__ __align__(1024) uint8_t lds[kWaves * kWaveBytes];
  __shared__ __align__(16) float factor[2][kRows], log_norm[2][kRows];
  __shared__ __align__(16) int place[2][kRows];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane / 32;
  // Each record's blocks begin one further on, or where blocks and CUs agree in number, one CU would have all parts of
  // the block that has most rows (6,000 tokens over 2,000, a window of 128 and 4 first tokens, 176 us instead of 273).
  const int list = blockIdx.x / a.n_kv, item = list / a.blocks;
  const int kvh = blockIdx.x % a.n_kv, block = (list + item) % a.blocks;
  const int32_t* rec = a.items + (int64_t)item * 4;
  const int seq = table_at(rec, 0), part = table_at(rec, 1), parts = table_at(rec, 2), offset = table_at(rec, 3);
  const int begin = table_at(a.starts, seq), count = table_at(a.starts, seq + 1) - begin;
  const int64_t room = (int64_t)a.width << a.page_log2;
  const int asked = table_at(a.lengths, seq), n = (int)min((int64_t)max(asked, 0), room), out_row = table_at(a.rows, seq);
  const int b0 = block * kBlockKeys;
  const BlockRows rows(a, count, n, b0);
  if (rows.row0 >= rows.row_end || (unsigned)out_row >= (unsigned)a.n_rows) return;
  const int g = a.n_heads / a.n_kv, base = rows.base, b1 = rows.last;
  const int per = rows.per(parts);
  if (part * (int64_t)per >= rows.row_end - rows.row0) return;  // the others have all its rows
  const int r_lo = rows.row0 + part * per, r_end = min(r_lo + per, rows.row_end);

  // rows of a tile to LDS, by all threads: chunk threadIdx % kChunks of every kPassRows-th row
  const int chunk = threadIdx.x % F::kChunks, tile_row = threadIdx.x / F::kChunks;
  const int step_tok = kRows / g, step_head = kRows - step_tok * g;
  u32x4_t held[kPasses];
  float held_lse[kPasses];
  int tok[kPasses], head[kPasses];  // of the rows that are fetched next
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    tok[p] = (r_lo + p * kPassRows + tile_row) / g;
    head[p] = r_lo + p * kPassRows + tile_row - tok[p] * g;
  }
  auto fetch = [&]() {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int t = min(tok[p], count - 1);  // past the last row: something, masked
      const int64_t at = begin + t;
      held[p] = u32x4_t{0, 0, 0, 0};
      if (kFull || 8 * chunk < a.d)
        held[p] = *reinterpret_cast<const u32x4_t*>(a.q + at * a.q_stride + (kvh * g + head[p]) * a.d + 8 * chunk);
      held_lse[p] = a.lse[at * a.n_heads + kvh * g + head[p]];
    }
  };
  auto put = [&](int slot, int row0) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = p * kPassRows + tile_row;
      float c2 = a.c2;
      if constexpr (kF16) {
        // times a power of two that brings the row's largest value to [1, 2), as the attention kernels' queries
        typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
        u16x2_t pair = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pair = __builtin_elementwise_max(pair, __builtin_bit_cast(u16x2_t, held[p][e] & 0x7fff7fffu));
        uint32_t most = (uint32_t)max(pair.x, pair.y) << 16;
#pragma unroll
        for (int off = 1; off < F::kChunks; off <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, off));
        int ex = (int)(most >> 23) - 127;
        if (most >= 0x7f800000u || most == 0) ex = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          held[p][e] = pack2<true>(__builtin_amdgcn_ldexpf(__uint_as_float(held[p][e] << 16), -ex),
                                   __builtin_amdgcn_ldexpf(__uint_as_float(held[p][e] & 0xffff0000u), -ex));
        c2 *= __builtin_amdgcn_ldexpf(1.f, ex);
      }
      *reinterpret_cast<u32x4_t*>(lds + slot * kTileBytes + row * F::kRowBytes + ((chunk ^ F::swizzle(row)) << 4)) = held[p];
      if (chunk == 0) {
        factor[slot][row] = c2;
        log_norm[slot][row] = held_lse[p] * kLog2e;
        place[slot][row] = row0 + row < r_end ? base + tok[p] : -1;
      }
      tok[p] += step_tok;
      head[p] += step_head;
      if (head[p] >= g) head[p] -= g, ++tok[p];
    }
  };

  u32x4_t k[2][F::kSteps];
  bool bad[2];
  double total[2] = {0., 0.};
  const int k_lo = b0 + wave * kWaveKeys, key0 = k_lo + lane % 32;
  fetch();
  // the wave's keys, whole rows at a time: read by the lanes that need them, 32 bytes of a row an instruction, 200
  // steps of 1,500 keys take 70 us instead of 64
  const int32_t* table = a.tables + (int64_t)seq * a.width;
  PageLoads<KeyWeightArgs, F, kStageKeys, kStageKeys / F::kRowsPerDma, 1> pages(a, 0, kvh);
  pages.hold(table, min(k_lo, b1) >> a.page_log2, a.width);
  const lds_u8 mine = (lds_u8)lds + wave * kWaveBytes;
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    if (kb * 32 % kStageKeys == 0) {
      tile_wait<63, false>();  // the keys before them have been read
      pages.template load<true, false>(k_lo + 32 * kb, within(0, b1), mine, mine);
      tile_wait<0, false>();
    }
#pragma unroll
    for (int st = 0; st < F::kSteps; ++st) {
      k[kb][st] = u32x4_t{0, 0, 0, 0};
      if (kFull || 16 * st + 8 * half < a.d)
        k[kb][st] = *reinterpret_cast<const u32x4_t*>(lds + wave * kWaveBytes + (32 * kb % kStageKeys + lane % 32) * F::kRowBytes +
                                                      (((2 * st + half) ^ F::swizzle(lane % 32)) << 4));
    }
    bad[kb] = (unsigned)table[min(key0 + 32 * kb, b1) >> a.page_log2] >= (unsigned)a.n_pages || asked > room;
  }
  __syncthreads();  // the keys have been read
  put(0, r_lo);
  __syncthreads();
  int slot = 0;
  const uint32_t reach = a.window > 0 ? a.window : 0x7fffffffu;
  // tokens of the tile's first and last row, and their heads
  int first_tok = r_lo / g, first_head = r_lo - first_tok * g, last_tok = (r_lo + kRows - 1) / g, last_head = r_lo + kRows - 1 - last_tok * g;
  auto move_on = [&](int& t, int& h) {
    t += step_tok, h += step_head;
    if (h >= g) h -= g, ++t;
  };
  for (int row0 = r_lo; row0 < r_end; row0 += kRows, slot ^= 1, move_on(first_tok, first_head), move_on(last_tok, last_head)) {
    const bool more = row0 + kRows < r_end;
    if (more) fetch();
    f32x16_t s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
#pragma unroll
    for (int st = 0; st < F::kSteps; ++st) {
      if (!kFull && 16 * st >= a.d) break;
      const u32x4_t q = *reinterpret_cast<const u32x4_t*>(lds + slot * kTileBytes + lane % 32 * F::kRowBytes +
                                                          (((2 * st + half) ^ F::swizzle(lane % 32)) << 4));
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) s[kb] = mfma32<kF16>(q, k[kb][st], s[kb]);
    }
    // whole: its rows see all keys of the wave
    const bool whole = row0 + kRows <= r_end && k_lo + kWaveKeys - 1 <= base + first_tok &&
                       (a.window == 0 || k_lo > base + last_tok - a.window);
    // none: no row of it sees one
    const bool none = k_lo > base + last_tok || (a.window > 0 && k_lo + kWaveKeys - 1 <= base + first_tok - a.window && k_lo >= a.first);
    float sum[2] = {0.f, 0.f};
    // the weights of the lane's rows 8 q4 on, four of each key
    auto weigh = [&](int q4, f32x4_t (&p)[2]) {
      const int at = 8 * q4 + 4 * half;
      const f32x4_t norm = *reinterpret_cast<const f32x4_t*>(&log_norm[slot][at]);
      f32x4_t c2 = {a.c2, a.c2, a.c2, a.c2};
      if constexpr (kF16) c2 = *reinterpret_cast<const f32x4_t*>(&factor[slot][at]);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) p[kb][e] = __builtin_amdgcn_exp2f(fmaf(s[kb][4 * q4 + e], c2[e], -norm[e]));
    };
    if (whole) {  // by itself, so that nothing divides its instructions
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        f32x4_t p[2];
        weigh(q4, p);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) sum[kb] += (p[kb][0] + p[kb][1]) + (p[kb][2] + p[kb][3]);
      }
    } else if (!none) {
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        if (row0 + 8 * q4 >= r_end) break;
        f32x4_t p[2];
        weigh(q4, p);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int pos = place[slot][8 * q4 + 4 * half + e];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            const int key = key0 + 32 * kb;
            bool seen = (uint32_t)(pos - key) < reach;
            if (k_lo < a.first) seen = seen || (key < a.first && key <= pos);
            if (!seen) p[kb][e] = 0.f;
          }
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) sum[kb] += (p[kb][0] + p[kb][1]) + (p[kb][2] + p[kb][3]);
      }
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) total[kb] += (double)sum[kb];  // as many sums as the chunk has tiles of rows
    if (more) put(slot ^ 1, row0 + kRows);
    __syncthreads();
  }
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) total[kb] += __shfl_xor(total[kb], 32);
  // lane l has key l of the wave's 64
  double sum = half == 0 ? total[0] : total[1];
  const int own = k_lo + lane;
  if (own > b1) return;
  if (half == 0 ? bad[0] : bad[1]) sum = (double)__uint_as_float(0x7fc00000u);
  if (parts > 1)
    a.part[((int64_t)(offset + part) * a.n_kv + kvh) * room + own] = sum;
  else
    write_weight(a, out_row, kvh, own, base, sum);
}

// The parts' sums of one key a thread, in their order.
__global__ __launch_bounds__(kBlockKeys) void key_weights_join_kernel(KeyWeightArgs a) {
  const int i = blockIdx.x, kvh = i % a.n_kv, block = i / a.n_kv % a.blocks;
  const int32_t* rec = a.items + (int64_t)(i / (a.n_kv * a.blocks)) * 4;
  const int seq = table_at(rec, 0), parts = table_at(rec, 2), offset = table_at(rec, 3);
  const int count = table_at(a.starts, seq + 1) - table_at(a.starts, seq), out_row = table_at(a.rows, seq);
  const int64_t room = (int64_t)a.width << a.page_log2;
  const int n = (int)min((int64_t)max(table_at(a.lengths, seq), 0), room), key = block * kBlockKeys + (int)threadIdx.x;
  const BlockRows rows(a, count, n, block * kBlockKeys);
  if (rows.row0 >= rows.row_end || (unsigned)out_row >= (unsigned)a.n_rows || key > rows.last) return;
  const int per = rows.per(parts), held = min(parts, (rows.row_end - rows.row0 + per - 1) / per);
  const double* part = a.part + ((int64_t)offset * a.n_kv + kvh) * room + key;
  double sum = 0.;
  constexpr int kAhead = 8;
  for (int p = 0; p < held; p += kAhead) {
    double x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) x[i] = part[(int64_t)min(p + i, held - 1) * a.n_kv * room];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (p + i < held) sum += x[i];
  }
  write_weight(a, out_row, kvh, key, rows.base, sum);
}

template <int DP, bool kF16, bool kFull>
int launch_key_weights(const KeyWeightArgs& a, int64_t items, int64_t joins, hipStream_t st) {
  const int64_t lists = (int64_t)a.blocks * a.n_kv;
  key_weights_kernel<DP, kF16, kFull><<<(unsigned)(items * lists), kWave * kWaves, 0, st>>>(a);
  const int rc = check_launch("key_weights_kernel");
  if (rc || joins == 0) return rc;
  key_weights_join_kernel<<<(unsigned)(joins * lists), kBlockKeys, 0, st>>>(a);
  return check_launch("key_weights_join_kernel");
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
  KLC_REQUIRE(x.page_size * x.n_kv * d < ((int64_t)1 << 30), KLC_ERR_SHAPE,
              "klc_attn_key_weights: pages of %lld tokens of %lld x %lld (below 2 GiB)", (long long)x.page_size, (long long)x.n_kv,
              (long long)d);
  KLC_REQUIRE(x.n_rows > 0 && x.n_rows < ((int64_t)1 << 31) && x.capacity > 0 && x.capacity < ((int64_t)1 << 31) && x.items > 0 &&
                  x.joins >= 0 && x.joins <= x.items && x.parts >= 0 && x.parts <= x.items &&
                  x.items < kMostBlocks && x.items * x.n_kv * (x.table_width * x.page_size / kBlockKeys + 1) < kMostBlocks,
              KLC_ERR_ARGUMENT, "klc_attn_key_weights: a plan of %lld items, %lld joins, %lld parts; %lld rows of %lld weights",
              (long long)x.items, (long long)x.joins, (long long)x.parts, (long long)x.n_rows, (long long)x.capacity);
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
  const int64_t keys = x.table_width * x.page_size, need = 8 * x.parts * x.n_kv * keys;
  KLC_REQUIRE(need == 0 || (x.workspace && (uintptr_t)x.workspace % 8 == 0 && x.workspace_bytes >= need), KLC_ERR_ARGUMENT,
              "klc_attn_key_weights: workspace of %lld bytes, need %lld, 8-byte aligned", (long long)x.workspace_bytes, (long long)need);
  auto in = [](const void* v) { return static_cast<const uint16_t*>(v); };
  auto index = [](const void* v) { return static_cast<const int32_t*>(v); };
  int page_log2 = 0;
  while ((1 << page_log2) < x.page_size) ++page_log2;
  const KeyWeightArgs a{in(x.q), static_cast<const float*>(x.lse), in(x.k_pages), in(x.k_pages), index(x.tables), index(x.lengths),
                        index(x.plan), index(x.rows), index(x.plan) + x.at_items, static_cast<float*>(x.weights),
                        static_cast<double*>(x.workspace), x.q_stride, x.capacity, (int)x.n_rows, (int)x.n_heads, (int)x.n_kv, (int)d, (int)x.n_pages, page_log2, (int)x.table_width,
                        (int)x.window, (int)x.first, (int)((keys + kBlockKeys - 1) / kBlockKeys), (float)(x.scale * kLog2e)};
  const hipStream_t st = as_stream(stream);
  const bool f16 = x.kv_dtype == KLC_DTYPE_F16;
  if (d == 64) return f16 ? launch_key_weights<64, true, true>(a, x.items, x.joins, st) : launch_key_weights<64, false, true>(a, x.items, x.joins, st);
  if (d == 128) return f16 ? launch_key_weights<128, true, true>(a, x.items, x.joins, st) : launch_key_weights<128, false, true>(a, x.items, x.joins, st);
  if (d < 64) return f16 ? launch_key_weights<64, true, false>(a, x.items, x.joins, st) : launch_key_weights<64, false, false>(a, x.items, x.joins, st);
  return f16 ? launch_key_weights<128, true, false>(a, x.items, x.joins, st) : launch_key_weights<128, false, false>(a, x.items, x.joins, st);
}
