// Attention of a decode batch over a paged KV cache (gfx950): one token of
// each sequence, whose first tokens may be a prefix that all sequences share.
//
// The prefix's keys are read once for the whole batch: its query rows are
// (sequence, head of the group) pairs, many rows to a tile of keys, split
// over the keys.  Each sequence's own keys are read by the workgroups of that
// sequence.  Every part leaves its sum, maximum and normaliser in float32 and
// a last kernel joins them.
#include <math.h>

#include "klc_flash.h"

namespace klc {
namespace {

constexpr int kOwnTile = 32;      // keys of a tile of the sequences' own parts
constexpr int kOwnRing = 3;
constexpr int kSharedTile = 64;
constexpr int kSharedRing = 3;
constexpr int kSharedWaves = 4;
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
  int n_seq, n_heads, n_kv, d, n_pages, page_log2, width, prefix, window, shared_splits, own_splits, shared_tiles;
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

template <int DP, int RB, class F>
__device__ __forceinline__ void store_part(const BatchArgs& a, const F& f, int rb, int64_t row, int split, bool bad) {
  const int lane = threadIdx.x % kWave, splits = a.shared_splits + a.own_splits;
  const float sum = add_halves(f.l[rb]);
  const int64_t at = row * splits + split;
  if (lane < 32) a.part_ml[at] = make_float2(f.m[rb], bad ? __uint_as_float(0x7fc00000u) : sum);
  float* dst = a.part_o + at * a.d + 4 * (lane / 32);
#pragma unroll
  for (int db = 0; db < F::kDimBlocks; ++db)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int dim = 32 * db + 2 * e;
      if (dim + 4 * (lane / 32) >= a.d) continue;
      *reinterpret_cast<float4*>(dst + dim) = make_float4(f.o[rb][db][e], f.o[rb][db][e + 1], f.o[rb][db][e + 2], f.o[rb][db][e + 3]);
    }
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

// The prefix's part: workgroup (KV head, tile of rows, split of the keys).
template <int DP, bool kF16, bool kFull>
__global__ __launch_bounds__(64 * kSharedWaves) void batch_shared_kernel(BatchArgs a) {
  using F = Flash<DP, kF16, kFull, 1, kSharedTile>;
  constexpr int KT = kSharedTile, W = kSharedWaves, kLoads = 2 * F::kDmas / W;
  __shared__ __align__(1024) uint8_t ring_mem[kSharedRing * F::kStage];
  const lds_u8 ring = (lds_u8)ring_mem;
  const int g = a.n_heads / a.n_kv, rows = a.n_seq * g;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int kvh = blockIdx.x % a.n_kv, row_tile = blockIdx.x / a.n_kv, split = blockIdx.y;
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
    const lds_u8 stage = ring + ((j - first) % kSharedRing) * F::kStage;
#pragma unroll
    for (int i = 0; i < F::kDmas / W; ++i) {
      const int n = wave + i * W, r = F::dma_row(n);
      const PageRow p = page_row(a.prefix_table, j * KT + n * F::kRowsPerDma, j * KT + r, 0, a.prefix - 1, a.page_log2, a.n_pages);
      bad |= p.bad;
      const int64_t at = p.row * kv_stride + (int64_t)kvh * a.d + 8 * F::dma_chunk(r, a.d);
      typedef __attribute__((address_space(3))) void* lds_void;
      __builtin_amdgcn_global_load_lds(a.k_pages + at, (lds_void)(stage + n * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds(a.v_pages + at, (lds_void)(stage + F::kMatBytes + n * 1024), 16, 0, 0);
    }
  };
#pragma unroll
  for (int i = 0; i < kSharedRing - 1; ++i)
    if (first + i < end_tile) load(first + i);
  for (int j = first; j < end_tile; ++j) {
    if (j + 1 < end_tile)
      tile_wait<kLoads*(kSharedRing - 2), true>();
    else
      tile_wait<0, true>();
    if (j + kSharedRing - 1 < end_tile) load(j + kSharedRing - 1);
    const int stage = ((j - first) % kSharedRing) * F::kStage;
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
  const bool any_bad = __syncthreads_or(bad);
  if (w_row + lane % 32 < rows) store_part<DP, 1>(a, f, 0, (int64_t)b * a.n_heads + head, split, any_bad);
}

// A sequence's own part, and with a window or no shared pass its part of the
// prefix: a wave takes (sequence, KV head, split of the keys).  The keys are
// listed as [prefix, padded to kPrefixAlign][own].
template <int DP, bool kF16, bool kFull>
__global__ __launch_bounds__(64) void batch_own_kernel(BatchArgs a) {
  using F = Flash<DP, kF16, kFull, 1, kOwnTile>;
  constexpr int KT = kOwnTile, kLoads = 2 * F::kDmas;
  __shared__ __align__(1024) uint8_t ring_mem[kOwnRing * F::kStage];
  const lds_u8 ring = (lds_u8)ring_mem;
  const int g = a.n_heads / a.n_kv, lane = threadIdx.x;
  const int kvh = blockIdx.x % a.n_kv, split = blockIdx.x / a.n_kv, b = blockIdx.y;
  int n = a.lengths[b];
  n = __builtin_amdgcn_readfirstlane(n);
  if (n < 0) return;  // no sequence: the join writes its zeros
  const int64_t room = (int64_t)a.width << a.page_log2;
  bool bad = n > room;
  n = (int)min((int64_t)n, room);
  const int pad = (a.prefix + kPrefixAlign - 1) / kPrefixAlign * kPrefixAlign;
  const bool shared = a.shared_splits > 0;
  // first visible key, and the lists' visible range
  const int seen = a.window > 0 ? min(a.window, a.prefix + n) : a.prefix + n, low = a.prefix + n - seen;
  const int begin = shared || low >= a.prefix ? pad + max(0, low - a.prefix) : low;
  const int end = n > 0 ? pad + n : a.prefix;
  const int first_tile = begin / KT, n_tiles = begin < end ? (end - 1) / KT + 1 - first_tile : 0;
  const int per = max((n_tiles + a.own_splits - 1) / a.own_splits, 1);
  const int first = first_tile + split * per, end_tile = min(first + per, first_tile + n_tiles);
  const int col = min(lane % 32, g - 1), head = kvh * g + col;
  F f;
  f.init(ring, a.d);
  const float c2 = a.c2 * load_query<F, kF16>(f.q[0], a.q + b * a.q_stride + (int64_t)head * a.d, a.d);
  const int64_t kv_stride = (int64_t)a.n_kv * a.d;
  const int32_t* own_table = a.tables + (int64_t)b * a.width;
  auto load = [&](int j) {
    const lds_u8 stage = ring + ((j - first) % kOwnRing) * F::kStage;
    const bool own = j * KT >= pad;
    const int base = own ? j * KT - pad : j * KT, last = own ? n - 1 : a.prefix - 1;
    const int visible = own ? max(begin - pad, 0) : begin;
#pragma unroll
    for (int i = 0; i < F::kDmas; ++i) {
      const int r = F::dma_row(i);
      const PageRow p = page_row(own ? own_table : a.prefix_table, base + i * F::kRowsPerDma, base + r, visible, last, a.page_log2, a.n_pages);
      bad |= p.bad;
      const int64_t at = p.row * kv_stride + (int64_t)kvh * a.d + 8 * F::dma_chunk(r, a.d);
      typedef __attribute__((address_space(3))) void* lds_void;
      __builtin_amdgcn_global_load_lds(a.k_pages + at, (lds_void)(stage + i * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds(a.v_pages + at, (lds_void)(stage + F::kMatBytes + i * 1024), 16, 0, 0);
    }
  };
#pragma unroll
  for (int i = 0; i < kOwnRing - 1; ++i)
    if (first + i < end_tile) load(first + i);
  for (int j = first; j < end_tile; ++j) {
    if (j + 1 < end_tile)
      tile_wait<kLoads*(kOwnRing - 2), false>();
    else
      tile_wait<0, false>();
    if (j + kOwnRing - 1 < end_tile) load(j + kOwnRing - 1);
    const int stage = ((j - first) % kOwnRing) * F::kStage;
    const int from = max(0, begin - j * KT), to = min(KT, (j * KT >= pad ? end : a.prefix) - j * KT);
    const bool part = from > 0 || to < KT;
    if (part) {
      clear_values<F, KT>(ring + stage, from, to, lane, 64);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    f32x16_t sc[1][KT / 32];
    f.scores(stage, sc);
    if (part) {
#pragma unroll
      for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = 32 * kb + 8 * (e / 4) + e % 4 + 4 * (lane / 32);
          if (key < from || key >= to) sc[0][kb][e] = -INFINITY;
        }
    }
    u32x4_t p[1][KT / 16];
    f.softmax(0, sc[0], c2, p[0]);
    f.values(stage, p);
  }
  if (lane % 32 < g) store_part<DP, 1>(a, f, 0, (int64_t)b * a.n_heads + head, a.shared_splits + split, __any(bad));
}

// out[row] = sum over the splits, a wave per row: lane l joins dims l and l + 64.
__global__ __launch_bounds__(256) void batch_join_kernel(BatchArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  if (row >= (int64_t)a.n_seq * a.n_heads) return;
  const int lane = threadIdx.x % kWave, splits = a.shared_splits + a.own_splits;
  const bool absent = a.lengths[row / a.n_heads] < 0;
  const float2* ml = a.part_ml + row * splits;
  const float sink = a.sinks != nullptr ? sink_log2(a.sinks[row % a.n_heads]) : -INFINITY;
  float o[2] = {0.f, 0.f}, sum = 0.f;
  if (!absent) {
    float top = sink;
    for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[s].x);
    const float base = top == -INFINITY ? 0.f : top;
    if (sink != -INFINITY) sum = exp2f(sink - base);
    for (int s = 0; s < splits; ++s) {
      const float2 x = ml[s];
      if (x.x == -INFINITY && x.y == 0.f) continue;  // a split without keys
      const float w = exp2f(x.x - base);
      sum += w * x.y;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < a.d) o[i] += w * a.part_o[(row * splits + s) * a.d + lane + 64 * i];
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + 64 * i < a.d) a.out[row * a.d + lane + 64 * i] = (uint16_t)f32_to_bf16_rne(o[i] * inv);
}

struct BatchPlan {
  int64_t shared_splits, shared_tiles, row_tiles, own_splits;
  int64_t splits() const { return shared_splits + own_splits; }
};
BatchPlan batch_plan(int64_t n_seq, int64_t n_heads, int64_t n_kv, int64_t prefix, int64_t max_own, int64_t window) {
  BatchPlan p{};
  const int64_t rows = n_seq * (n_heads / n_kv);
  p.row_tiles = (rows + 32 * kSharedWaves - 1) / (32 * kSharedWaves);
  const bool shared = prefix > 0 && window == 0 && n_seq > 1;
  int64_t keys = max_own + (shared ? 0 : prefix);
  if (window > 0 && window < keys) keys = window;
  if (shared) {
    const int64_t tiles = (prefix + kSharedTile - 1) / kSharedTile;
    const int64_t want = (256 + n_kv * p.row_tiles - 1) / (n_kv * p.row_tiles);
    p.shared_tiles = (tiles + want - 1) / want;
    p.shared_splits = (tiles + p.shared_tiles - 1) / p.shared_tiles;
  }
  const int64_t own_tiles = keys / kOwnTile + 2;
  const int64_t want = (1024 + n_seq * n_kv - 1) / (n_seq * n_kv), most = (own_tiles + 3) / 4;
  p.own_splits = want < most ? want : most;
  return p;
}

int64_t batch_bytes(const BatchPlan& p, int64_t n_seq, int64_t n_heads, int64_t d) {
  return n_seq * n_heads * p.splits() * (4 * d + 8);
}

template <int DP, bool kF16, bool kFull>
int launch_batch(const BatchArgs& a, const BatchPlan& p, hipStream_t st) {
  int rc;
  if (p.shared_splits > 0) {
    const dim3 grid((unsigned)(a.n_kv * p.row_tiles), (unsigned)p.shared_splits);
    batch_shared_kernel<DP, kF16, kFull><<<grid, 64 * kSharedWaves, 0, st>>>(a);
    if ((rc = check_launch("batch_shared_kernel"))) return rc;
  }
  const dim3 grid((unsigned)(a.n_kv * p.own_splits), (unsigned)a.n_seq);
  batch_own_kernel<DP, kF16, kFull><<<grid, 64, 0, st>>>(a);
  if ((rc = check_launch("batch_own_kernel"))) return rc;
  batch_join_kernel<<<(unsigned)(((int64_t)a.n_seq * a.n_heads + 3) / 4), 256, 0, st>>>(a);
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
  return batch_bytes(batch_plan(n_seq, n_heads, n_kv, prefix_len, max_own, window), n_seq, n_heads, head_dim);
}

extern "C" int klc_attn_batch(const void* q, const void* k_pages, const void* v_pages, const int32_t* tables,
                              const int32_t* lengths, const int32_t* prefix_table, const void* sinks, int64_t n_seq,
                              int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t q_stride, int64_t n_pages,
                              int64_t page_size, int64_t table_width, int64_t prefix_len, int64_t window, float scale,
                              int kv_dtype, void* workspace, int64_t workspace_bytes, void* out, void* stream) {
  KLC_REQUIRE(q && k_pages && v_pages && lengths && out && workspace, KLC_ERR_ARGUMENT, "klc_attn_batch: null pointer");
  KLC_REQUIRE((tables || table_width == 0) && (prefix_table || prefix_len == 0), KLC_ERR_ARGUMENT,
              "klc_attn_batch: null table");
  KLC_REQUIRE(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0 && n_pages > 0 &&
                  n_pages * page_size < ((int64_t)1 << 31) && table_width >= 0 && table_width < ((int64_t)1 << 25),
              KLC_ERR_SHAPE, "klc_attn_batch: %lld pages of %lld tokens (a power of two, 16..4096), tables of %lld",
              (long long)n_pages, (long long)page_size, (long long)table_width);
  const int64_t max_own = table_width * page_size;
  int rc = check_sizes("klc_attn_batch", n_seq, n_heads, n_kv, head_dim, prefix_len, max_own, window);
  if (rc) return rc;
  KLC_REQUIRE(q_stride >= n_heads * head_dim && q_stride % 8 == 0, KLC_ERR_SHAPE,
              "klc_attn_batch: q stride %lld (a multiple of 8, no overlap)", (long long)q_stride);
  KLC_REQUIRE(((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)workspace | (uintptr_t)out) % 16 == 0,
              KLC_ERR_ARGUMENT, "klc_attn_batch: q, pages, workspace and out must be 16-byte aligned");
  KLC_REQUIRE(scale > 0.f && scale < INFINITY, KLC_ERR_ARGUMENT, "klc_attn_batch: scale %g", (double)scale);
  KLC_REQUIRE(kv_dtype == KLC_DTYPE_BF16 || kv_dtype == KLC_DTYPE_F16, KLC_ERR_UNSUPPORTED,
              "klc_attn_batch: kv_dtype %d (bfloat16 or float16)", kv_dtype);
  const BatchPlan p = batch_plan(n_seq, n_heads, n_kv, prefix_len, max_own, window);
  const int64_t need = batch_bytes(p, n_seq, n_heads, head_dim);
  KLC_REQUIRE(workspace_bytes >= need, KLC_ERR_ARGUMENT, "klc_attn_batch: workspace of %lld bytes, need %lld",
              (long long)workspace_bytes, (long long)need);
  auto in = [](const void* x) { return static_cast<const uint16_t*>(x); };
  int page_log2 = 0;
  while ((1 << page_log2) < page_size) ++page_log2;
  float* part_o = static_cast<float*>(workspace);
  const BatchArgs a{in(q), in(k_pages), in(v_pages), tables, lengths, prefix_table, in(sinks),
                    static_cast<uint16_t*>(out), part_o,
                    reinterpret_cast<float2*>(part_o + n_seq * n_heads * p.splits() * head_dim), q_stride, (int)n_seq,
                    (int)n_heads, (int)n_kv, (int)head_dim, (int)n_pages, page_log2, (int)table_width, (int)prefix_len,
                    (int)window, (int)p.shared_splits, (int)p.own_splits, (int)p.shared_tiles, scale * kLog2e};
  const hipStream_t st = as_stream(stream);
  const bool f16 = kv_dtype == KLC_DTYPE_F16;
  if (head_dim == 64) return f16 ? launch_batch<64, true, true>(a, p, st) : launch_batch<64, false, true>(a, p, st);
  if (head_dim == 128) return f16 ? launch_batch<128, true, true>(a, p, st) : launch_batch<128, false, true>(a, p, st);
  if (head_dim < 64) return f16 ? launch_batch<64, true, false>(a, p, st) : launch_batch<64, false, false>(a, p, st);
  return f16 ? launch_batch<128, true, false>(a, p, st) : launch_batch<128, false, false>(a, p, st);
}
