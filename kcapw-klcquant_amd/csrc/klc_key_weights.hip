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
// never leave it but at the end, 16 at a time in float32 and those sums in
// float64.  A list made on the host has the workgroups:
// a block of keys that new tokens see, and a part of the rows that see it.
// Parts' float64 sums are added by a second launch, in their order.
//
// The list goes by what each sequence's rows see: a grid over the longest
// sequence of a batch took 133 us for 127 steps of 200 to 1,000 keys and one of
// 32,000, the list 34, and a row of sums over all keys for every part 1 GB for
// 64 suffixes of 100 tokens beside a step of 131,072, the list's blocks 6 MB.
//
// What bounds it (64 heads over 8 of size 64): the exponentials and the two
// instructions beside each, 46 us of the 67 that 1,000 tokens over 4,000 take,
// 143 for a prompt of 4,096; steps by memory, 64 of 1,000 to 2,000 keys in 26
// us (4.0 TB/s), and the start and end of a workgroup for 256 keys.
#include <math.h>

#include <algorithm>
#include <type_traits>
#include <utility>
#include <vector>

#include "klc_key_blocks.h"
#include "klc_paged_tiles.h"

namespace klc {
namespace {

constexpr int kWaveKeys = kBlockKeys / kWaves;
constexpr int kRows = kRowTile;

struct KeyWeightArgs {
  const uint16_t* q;                // bfloat16 [tokens] rows
  const float* lse;                 // [tokens][n_heads]
  const uint16_t *k_pages, *v_pages;  // [n_pages][page][n_kv][d]; values are not read
  const int32_t *tables, *lengths;  // [n_seq][width], [n_seq]
  const int32_t *rows, *items;      // [n_seq], the list
  float* weights;                   // [n_rows][n_kv][capacity]
  double* part;                     // [parts of all joined blocks][n_kv][kBlockKeys]
  int64_t q_stride, capacity;
  int n_rows, n_heads, n_kv, group, d, n_pages, page_log2, width, window, first;
  float c2;

  // from a kernel's arguments at `place`
  static __device__ __forceinline__ KeyWeightArgs at(uintptr_t place) {
    struct {
      int32_t word[sizeof(KeyWeightArgs) / 4];
    } words;
#pragma unroll
    for (size_t i = 0; i < sizeof(KeyWeightArgs) / 4; ++i) words.word[i] = table_at((const int32_t*)place, i);
    KeyWeightArgs a = __builtin_bit_cast(KeyWeightArgs, words);
    // of global memory, which the compiler knows of arguments alone: loads that may be from LDS wait for it too
    auto known = [](auto*& p) { p = (std::remove_reference_t<decltype(p)>)(__attribute__((address_space(1))) void*)(uintptr_t)p; };
    known(a.q), known(a.lse), known(a.k_pages), known(a.v_pages), known(a.tables), known(a.lengths), known(a.rows), known(a.items),
        known(a.weights), known(a.part);
    return a;
  }
};

// What a listed workgroup has to do, the same for all its threads.
struct WeightItem {
  int kvh, part, parts, least, seq, begin, out_row, listed;
  int64_t scratch;  // of the part, in `part`
  ListPlace place;
  bool wrong;       // the sequence is longer than its table
  KeyBlocks keys;
  __device__ __forceinline__ WeightItem(const KeyWeightArgs& a, int workgroup)
      : kvh(workgroup % a.n_kv), place(0), keys(0, 0, 1, 0, 0) {
    const int32_t* item = a.items + (int64_t)(workgroup / a.n_kv) * kListRecord;
    seq = table_at(item, 0);
    part = table_at(item, 1);
    parts = table_at(item, 2);
    place = ListPlace(table_at(item, 3));
    scratch = ((int64_t)table_at(item, 4) * a.n_kv + kvh) * kBlockKeys;
    begin = table_at(item, 5);
    least = table_at(item, 7);
    out_row = table_at(a.rows, seq);
    const int64_t room = (int64_t)a.width << a.page_log2;
    const int count = table_at(item, 6), asked = table_at(a.lengths, seq);
    wrong = asked > room;
    keys = KeyBlocks((int)min((int64_t)max(asked, 0), room), count, a.group, a.window, a.first);
    listed = keys.begin(place.head) + place.index;
  }
  __device__ __forceinline__ bool known(const KeyWeightArgs& a) const { return (unsigned)out_row < (unsigned)a.n_rows; }
};

__device__ __forceinline__ void write_weight(const KeyWeightArgs& a, int out_row, int kvh, int key, int base, double sum) {
  if (key >= a.capacity) return;
  float* dst = a.weights + ((int64_t)out_row * a.n_kv + kvh) * a.capacity + key;
  *dst = (float)(key >= base ? sum : (double)*dst + sum);
}

constexpr int kWeightLds = kWaves * 8192;
struct RowTiles {
  float factor[2][kRows], log_norm[2][kRows];
  int place[2][kRows];
};

// The sums of rows r_lo up to r_end of the sequence over a block of its keys: to `part`, or, if there is none, to the weights.
template <int DP, bool kF16, bool kFull>
__device__ __forceinline__ void block_weights(const KeyWeightArgs& a, const WeightItem& it, int block, int r_lo, int r_end,
                                              double* part, uint8_t (&lds)[kWeightLds], RowTiles& tiles) {
  using F = AttnWave<DP, kF16, kFull, 1, kRows>;
  constexpr int kThreads = kWave * kWaves, kPassRows = kThreads / F::kChunks, kPasses = kRows / kPassRows;
  static_assert(kPasses * kPassRows == kRows, "");
  // the block's keys on their way into registers, then two tiles of rows
  constexpr int kTileBytes = kRows * F::kRowBytes, kWaveBytes = kWeightLds / kWaves, kStageKeys = kWaveBytes / F::kRowBytes;
  auto &factor = tiles.factor, &log_norm = tiles.log_norm;
  auto& place = tiles.place;
  int thread = threadIdx.x;
  asm volatile("" : "+v"(thread));  // what is worked out of it is not held over blocks
  const int lane = thread % kWave, wave = __builtin_amdgcn_readfirstlane(thread / kWave), half = lane / 32;
  const int kvh = it.kvh, begin = it.begin, count = it.keys.count, g = it.keys.g, base = it.keys.base;
  const int b0 = block * kBlockKeys, b1 = min(b0 + kBlockKeys, it.keys.n) - 1;

  // rows of a tile to LDS, by all threads: chunk threadIdx % kChunks of every kPassRows-th row
  const int chunk = thread % F::kChunks, tile_row = thread / F::kChunks;
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
  double total[2] = {0., 0.};
  const int k_lo = b0 + wave * kWaveKeys, key0 = k_lo + lane % 32;
  fetch();
  // the wave's keys, whole rows at a time: read by the lanes that need them, 32 bytes of a row an instruction, 200
  // steps of 1,500 keys take 70 us instead of 64
  const int32_t* table = a.tables + (int64_t)it.seq * a.width;
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
  }
  __syncthreads();  // the keys have been read
  // the rows, asked for before the keys, from here on: worked on sooner they would hold up the last keys' loads
#pragma unroll
  for (int p = 0; p < kPasses; ++p) asm volatile("" : "+v"(held[p]), "+v"(held_lse[p]));
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
  // what no row sees keeps its weight, whichever keys share its block
  if (it.keys.sees(own) && (it.wrong || (unsigned)table[own >> a.page_log2] >= (unsigned)a.n_pages)) sum = (double)__uint_as_float(0x7fc00000u);
  if (part != nullptr)
    part[own - b0] = sum;
  else
    write_weight(a, it.out_row, kvh, own, base, sum);
}

template <int DP, bool kF16, bool kFull>
__global__ __launch_bounds__(kWave * kWaves, DP == 64 ? 4 : 3) void key_weights_kernel(KeyWeightArgs) {
  __shared__ __align__(1024) uint8_t lds[kWeightLds];
  __shared__ __align__(16) RowTiles tiles;
  // The listed block, and behind a sequence's last one those that it has grown into, whose rows are in one part.
  bool more = true;
#pragma unroll 1
  for (int grown = 0; more; ++grown) {
    // the arguments and the item are read again for every block: held over the work on one, 28 to 62 scalars spill
    int workgroup = blockIdx.x;
    uintptr_t args = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(workgroup), "+s"(args));
    const KeyWeightArgs a = KeyWeightArgs::at(args);
    const WeightItem it(a, workgroup);
    const int block = it.listed + grown, end = it.keys.end(it.place.head);
    if (!it.known(a) || block >= end) return;
    more = it.place.last && it.part == 0 && block + 1 < end;
    const int r0 = it.keys.row_begin(block), r1 = it.keys.row_end(block);
    const int per = KeyBlocks::per(r1 - r0, grown ? 1 : it.parts, it.least);
    const int64_t from = r0 + (int64_t)it.part * per;
    if (r0 >= r1 || from >= r1) continue;  // no row, or the others have them all
    block_weights<DP, kF16, kFull>(a, it, block, (int)from, min((int)from + per, r1),
                                   grown || it.parts == 1 ? nullptr : a.part + it.scratch, lds, tiles);
  }
}

// The parts' sums of one key a thread, in their order.
__global__ __launch_bounds__(kBlockKeys) void key_weights_join_kernel(KeyWeightArgs a) {
  const WeightItem it(a, blockIdx.x);
  const int key = it.listed * kBlockKeys + (int)threadIdx.x;
  if (!it.known(a) || it.listed >= it.keys.end(it.place.head) || key >= it.keys.n) return;
  const int rows = it.keys.row_end(it.listed) - it.keys.row_begin(it.listed);
  if (rows <= 0) return;
  const int per = KeyBlocks::per(rows, it.parts, it.least), held = (rows + per - 1) / per;
  const double* part = a.part + it.scratch + threadIdx.x;
  double sum = 0.;
  constexpr int kAhead = 8;
  for (int p = 0; p < held; p += kAhead) {
    double x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) x[i] = part[(int64_t)min(p + i, held - 1) * a.n_kv * kBlockKeys];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (p + i < held) sum += x[i];
  }
  write_weight(a, it.out_row, it.kvh, key, it.keys.base, sum);
}

template <int DP, bool kF16, bool kFull>
int launch_key_weights(const KeyWeightArgs& a, int64_t items, int64_t joins, hipStream_t st) {
  key_weights_kernel<DP, kF16, kFull><<<(unsigned)(items * a.n_kv), kWave * kWaves, 0, st>>>(a);
  const int rc = check_launch("key_weights_kernel");
  if (rc || joins == 0) return rc;
  key_weights_join_kernel<<<(unsigned)(joins * a.n_kv), kBlockKeys, 0, st>>>(a);
  return check_launch("key_weights_join_kernel");
}

}  // namespace
}  // namespace klc

using namespace klc;

extern "C" int klc_attn_weight_list(const int32_t* plan, const int64_t* sizes, const int32_t* lengths, int64_t n_seq,
                                    int64_t n_heads, int64_t n_kv, int64_t window, int64_t first, int32_t* list,
                                    int64_t capacity, int64_t* list_sizes) {
  KLC_REQUIRE(plan && sizes && lengths && list_sizes && (list || capacity == 0), KLC_ERR_ARGUMENT,
              "klc_attn_weight_list: null pointer");
  KLC_REQUIRE(n_seq > 0 && n_seq < ((int64_t)1 << 20) && n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && n_heads <= 4096 &&
                  window >= 0 && window < ((int64_t)1 << 30) && first >= 0 && first < ((int64_t)1 << 29) &&
                  (first == 0 || window > 0),
              KLC_ERR_ARGUMENT, "klc_attn_weight_list: %lld sequences, heads %lld / %lld, window %lld, %lld first tokens",
              (long long)n_seq, (long long)n_heads, (long long)n_kv, (long long)window, (long long)first);
  const int64_t at = sizes[8], records = sizes[9], g = n_heads / n_kv;
  KLC_REQUIRE(plan[0] == 0 && plan[n_seq] == sizes[1] && sizes[1] * g < ((int64_t)1 << 30) && records >= n_seq && at > n_seq &&
                  at + records * kPartRecord == sizes[0],
              KLC_ERR_ARGUMENT, "klc_attn_weight_list: not a plan of %lld sequences", (long long)n_seq);
  for (int64_t s = 0; s < n_seq; ++s)
    KLC_REQUIRE(plan[s + 1] > plan[s] && lengths[s] >= plan[s + 1] - plan[s] && lengths[s] < (1 << 29), KLC_ERR_ARGUMENT,
                "klc_attn_weight_list: sequence %lld of %d new tokens among %d (at least one, below 2^29)", (long long)s,
                plan[s + 1] - plan[s], lengths[s]);
  try {
    const int least = least_tiles(plan, lengths, n_seq, g, n_kv, window, first);
    std::vector<int64_t> scratch(n_seq);  // of a sequence's first joined block
    int64_t joins = 0, others = 0, singles = 0, parts_held = 0;
    // each(record, whether of first tokens, blocks, parts of their rows, place of the first block's sums)
    auto walk = [&](auto each) {
      for (int64_t i = 0; i < records; ++i) {
        const int32_t* rec = plan + at + i * kPartRecord;
        const int s = rec[0];
        const KeyBlocks keys(lengths[s], plan[s + 1] - plan[s], (int)g, (int)window, (int)first);
        int64_t place = scratch[s];
        for (const bool head : {true, false}) {
          const int parts = keys.parts(head, rec[2], least);
          // behind the first tokens' blocks there may be one that no key is in yet
          const int64_t blocks = head ? keys.heads : std::max(1, keys.end(false) - keys.low);
          if (rec[1] < parts) each(rec, head, blocks, parts, place);
          if (parts > 1) place += blocks * parts;
        }
      }
    };
    for (int64_t i = 0; i < records; ++i) {
      const int32_t* rec = plan + at + i * kPartRecord;
      KLC_REQUIRE(rec[0] >= 0 && rec[0] < n_seq && rec[1] >= 0 && rec[1] < rec[2], KLC_ERR_ARGUMENT,
                  "klc_attn_weight_list: not a plan of %lld sequences", (long long)n_seq);
    }
    walk([&](const int32_t* rec, bool, int64_t blocks, int parts, int64_t) {
      if (rec[1] == 0 && parts > 1) {
        joins += blocks;
        scratch[rec[0]] += blocks * parts;
        parts_held += blocks * parts;
      }
      if (rec[1] > 0) others += blocks;
      if (parts == 1) singles += blocks;
    });
    const int64_t items = joins + others + singles;
    KLC_REQUIRE(items * n_kv < kMostBlocks, KLC_ERR_ARGUMENT, "klc_attn_weight_list: %lld blocks of keys of %lld heads are too many",
                (long long)items, (long long)n_kv);
    list_sizes[0] = items * kListRecord;
    list_sizes[1] = items, list_sizes[2] = joins, list_sizes[3] = parts_held;
    if (list_sizes[0] > capacity) return KLC_OK;
    for (int64_t s = 0, sum = 0; s < n_seq; ++s) sum += std::exchange(scratch[s], sum);
    // Each sequence's blocks begin one further on, or where blocks and CUs agree in number one CU would have the same block
    // of all of them (64 steps of 1,000 to 2,000 keys listed for 2,048: 26.4 us instead of 29.2).  In order: the first
    // parts of joined blocks, which the second launch takes too, their other parts, and what is not joined.
    int32_t *first_parts = list, *other_parts = first_parts + joins * kListRecord, *whole = other_parts + others * kListRecord;
    walk([&](const int32_t* rec, bool head, int64_t blocks, int parts, int64_t place) {
      int32_t*& to = parts == 1 ? whole : rec[1] == 0 ? first_parts : other_parts;
      for (int64_t i = 0; i < blocks; ++i) {
        const int64_t b = (i + rec[0]) % blocks;
        const int32_t item[kListRecord] = {rec[0], rec[1], parts, ListPlace::of(head, b == blocks - 1, b),
                                           parts == 1 ? 0 : (int32_t)(place + b * parts + rec[1]), plan[rec[0]],
                                           plan[rec[0] + 1] - plan[rec[0]], least};
        to = std::copy(item, item + kListRecord, to);
      }
    });
  } catch (const std::exception& e) {
    return set_error(KLC_ERR_ARGUMENT, "klc_attn_weight_list: %s", e.what());
  }
  return KLC_OK;
}

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
                  x.items < kMostBlocks && x.items * x.n_kv < kMostBlocks,
              KLC_ERR_ARGUMENT, "klc_attn_key_weights: a list of %lld items, %lld joins, %lld parts; %lld rows of %lld weights",
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
  const int64_t need = 8 * x.parts * x.n_kv * kBlockKeys;
  KLC_REQUIRE(need == 0 || (x.workspace && (uintptr_t)x.workspace % 8 == 0 && x.workspace_bytes >= need), KLC_ERR_ARGUMENT,
              "klc_attn_key_weights: workspace of %lld bytes, need %lld, 8-byte aligned", (long long)x.workspace_bytes, (long long)need);
  // lists are copied to four values behind a multiple of 8; the plan's own records, which list no workgroups, are at one
  KLC_REQUIRE(x.at_items > 0 && x.at_items % 8 == 4, KLC_ERR_ARGUMENT,
              "klc_attn_key_weights: at_items %lld is not a list's (klc_attn_weight_list)", (long long)x.at_items);
  auto in = [](const void* v) { return static_cast<const uint16_t*>(v); };
  auto index = [](const void* v) { return static_cast<const int32_t*>(v); };
  int page_log2 = 0;
  while ((1 << page_log2) < x.page_size) ++page_log2;
  const KeyWeightArgs a{in(x.q), static_cast<const float*>(x.lse), in(x.k_pages), in(x.k_pages), index(x.tables), index(x.lengths),
                        index(x.rows), index(x.plan) + x.at_items, static_cast<float*>(x.weights),
                        static_cast<double*>(x.workspace), x.q_stride, x.capacity, (int)x.n_rows, (int)x.n_heads, (int)x.n_kv, (int)(x.n_heads / x.n_kv), (int)d, (int)x.n_pages, page_log2, (int)x.table_width,
                        (int)x.window, (int)x.first, (float)(x.scale * kLog2e)};
  const hipStream_t st = as_stream(stream);
  const bool f16 = x.kv_dtype == KLC_DTYPE_F16;
  if (d == 64) return f16 ? launch_key_weights<64, true, true>(a, x.items, x.joins, st) : launch_key_weights<64, false, true>(a, x.items, x.joins, st);
  if (d == 128) return f16 ? launch_key_weights<128, true, true>(a, x.items, x.joins, st) : launch_key_weights<128, false, true>(a, x.items, x.joins, st);
  if (d < 64) return f16 ? launch_key_weights<64, true, false>(a, x.items, x.joins, st) : launch_key_weights<64, false, false>(a, x.items, x.joins, st);
  return f16 ? launch_key_weights<128, true, false>(a, x.items, x.joins, st) : launch_key_weights<128, false, false>(a, x.items, x.joins, st);
}
