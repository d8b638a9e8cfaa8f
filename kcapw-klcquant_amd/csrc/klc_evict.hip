// Eviction of the keys of least weight from a paged KV cache (gfx950), in
// place, for every layer and KV head by itself.
//
// A sequence of n keys keeps `keep`: the first `first`, the last `recent` and
// of those between them the ones of the largest weights, equal ones from the
// lowest place on.  Places below keep - recent hold their own key if it stays;
// the others, holes, take in order the kept keys from keep - recent on.  Those
// moves read and write different places, so they need no order, and few keys
// move when few leave.  Then the recent ones follow in order, read in pieces
// before the piece is written: a place may be both.
//
// One workgroup does all of a list's work, so that its steps wait for nothing
// but its own barriers: the least weight that stays by three passes over 11,
// 11 and 10 bits of the weights' order, then the holes, the keys behind them,
// the moves and the recent keys.
//
// What bounds it (8 KV heads of size 64): many lists by HBM, 36 layers of three
// sequences of up to 6,001 keys cut to 1,500 in 104 to 110 us by the card (545
// MB, 5.0 to 5.2 TB/s, a large copy's rate); few
// by that chain of steps, eight sequences of up to 2,064 keys cut to 2,000 in
// one layer in 13.  Weights held in registers between the steps, and the recent
// keys read ahead of the moves, changed neither.
#include <math.h>

#include "klc_common.h"

namespace klc {
namespace {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / kWave;
constexpr int kBins = 2048;

struct EvictArgs {
  uint8_t* pools;                           // [2 * layers][n_pages][page][n_kv][d], 16 bits each
  float* weights;                           // [layers][n_rows][n_kv][capacity]
  const int32_t *tables, *lengths, *rows;   // [n_seq][width], [n_seq], [n_seq]
  int32_t* kept;                            // [layers][n_seq][n_kv][keep]
  int32_t* holes;                           // as kept
  int64_t capacity;
  int n_seq, n_rows, n_kv, d, n_pages, page_log2, width, keep, recent, first;
};

// bits that ascend with the value, NaN above all, both zeros alike
__device__ __forceinline__ uint32_t order_bits(float w) {
  const uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if ((u & 0x7fffffffu) == 0) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// sum over the lanes before this one
__device__ __forceinline__ int rank_below(uint64_t ballot) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(ballot >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ballot, 0));
}

__global__ __launch_bounds__(kEvictThreads) void evict_kernel(EvictArgs a) {
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t wave_sum[kEvictWaves], wave_other[kEvictWaves];
  __shared__ uint32_t found[2];  // the digit, and how many of it and above it stay to be found
  const int t = threadIdx.x, lane = t % kWave, wave = t / kWave;
  const int kvh = blockIdx.x % a.n_kv, seq = blockIdx.x / a.n_kv % a.n_seq, layer = blockIdx.x / (a.n_kv * a.n_seq);
  const int n = a.lengths[seq], row = a.rows[seq];
  const int64_t list = ((int64_t)layer * a.n_seq + seq) * a.n_kv + kvh;
  int32_t *kept = a.kept + list * a.keep, *holes = a.holes + list * a.keep;
  const bool wrong = n > (int64_t)a.width << a.page_log2 || n > a.capacity || (unsigned)row >= (unsigned)a.n_rows;
  if (n <= a.keep || wrong) {
    for (int i = t; i < a.keep; i += kEvictThreads) kept[i] = i < n && !wrong ? i : -1;
    return;
  }
  float* weights = a.weights + (((int64_t)layer * a.n_rows + row) * a.n_kv + kvh) * a.capacity;
  const int ahead = a.keep - a.recent, middle_end = n - a.recent;
  const int wanted = ahead - a.first;  // of the middle

  // the digits of the wanted-th largest: `least` so far, of whose equals `need` stay
  uint32_t least = 0, mask = 0;
  int need = wanted;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = t; i < kBins; i += kEvictThreads) bins[i] = 0;
    __syncthreads();
    for (int i = a.first + t; i < middle_end; i += kEvictThreads) {
      const uint32_t u = order_bits(weights[i]), bin = (u >> shift) & ((1u << bits) - 1);
      bool open = (u & mask) == least;
      // lists have many equal weights, zeros above all: a wave's first two bins by one addition each
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint64_t all = __ballot(open);
        if (all == 0) break;
        const int leader = __ffsll((unsigned long long)all) - 1;
        const bool same = open && bin == (uint32_t)__builtin_amdgcn_readlane((int)bin, leader);
        const uint64_t alike = __ballot(same);
        if (lane == leader) atomicAdd(&bins[bin], (uint32_t)__popcll(alike));
        open = open && !same;
      }
      if (open) atomicAdd(&bins[bin], 1u);
    }
    __syncthreads();
    // the highest digit at which as many as needed are reached, from the top: thread t has digits 2047 - 2 t and the next
    const uint32_t hi = bins[kBins - 1 - 2 * t], lo = bins[kBins - 2 - 2 * t];
    uint32_t sum = hi + lo;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const uint32_t up = __shfl_up(sum, off);
      if (lane >= off) sum += up;
    }
    if (lane == kWave - 1) wave_sum[wave] = sum;
    __syncthreads();
    uint32_t before = sum - hi - lo;
    for (int w = 0; w < wave; ++w) before += wave_sum[w];
    if (before < (uint32_t)need && before + hi >= (uint32_t)need) found[0] = kBins - 1 - 2 * t, found[1] = need - before;
    if (before + hi < (uint32_t)need && before + hi + lo >= (uint32_t)need)
      found[0] = kBins - 2 - 2 * t, found[1] = need - before - hi;
    __syncthreads();
    if (wanted > 0) {
      least |= found[0] << shift;
      mask |= ((1u << bits) - 1) << shift;
      need = (int)found[1];
    }
    __syncthreads();
  }
  // 1 of a bool before this thread's place, over the workgroup, and in all
  auto scan = [&](bool x, uint32_t* sums, int& total) {
    const uint64_t ballot = __ballot(x);
    if (lane == 0) sums[wave] = __popcll(ballot);
    __syncthreads();
    int before = rank_below(ballot);
    total = 0;
    for (int w = 0; w < kEvictWaves; ++w) {
      const int c = (int)sums[w];
      if (w < wave) before += c;
      total += c;
    }
    return before;
  };
  // places in order: those below `ahead` stay or are holes, those from it on that stay go to the holes
  int equals = 0, hole_count = 0, moved = 0;
  for (int i0 = 0; i0 < middle_end; i0 += kEvictThreads) {
    const int i = i0 + t;
    const bool in = i < middle_end, middle = in && i >= a.first;
    const uint32_t u = middle ? order_bits(weights[i]) : 0;
    const bool equal = middle && wanted > 0 && u == least;
    int all;
    const int rank = equals + scan(equal, wave_sum, all);
    equals += all;
    const bool stays = in && (i < a.first || (wanted > 0 && u > least) || (equal && rank < need));
    const bool hole = in && i < ahead && !stays, goes = in && i >= ahead && stays;
    if (in && i < ahead && stays) kept[i] = i;
    // both lists in one scan: a count of at most 1024 in each half
    const uint64_t bh = __ballot(hole), bg = __ballot(goes);
    if (lane == 0) wave_other[wave] = (uint32_t)__popcll(bh) | (uint32_t)__popcll(bg) << 16;
    __syncthreads();
    uint32_t before = 0, sum = 0;
    for (int w = 0; w < kEvictWaves; ++w) {
      const uint32_t c = wave_other[w];
      if (w < wave) before += c;
      sum += c;
    }
    // a hole's rank never passes that of the key for it in what a thread reads below: all holes lie before all keys
    if (hole) holes[hole_count + (int)(before & 0xffff) + rank_below(bh)] = i;
    hole_count += (int)(sum & 0xffff);
    if (i0 + kEvictThreads > ahead) {  // the last holes are written, keys may go
      __threadfence_block();
      __syncthreads();
    }
    if (goes) {
      const int r = moved + (int)(before >> 16) + rank_below(bg);
      kept[holes[r]] = i;
    }
    moved += (int)(sum >> 16);
    __syncthreads();
  }
  for (int i = t; i < a.recent; i += kEvictThreads) kept[ahead + i] = middle_end + i;
  __threadfence_block();
  __syncthreads();

  // 16 bytes a thread of a key's row and, in the second half of its lanes, of its value's
  const int chunks = a.d / 8, lanes = 2 * chunks, per_step = kEvictThreads / lanes;
  const int mine = t / lanes, part = t % lanes;
  const bool worker = mine < per_step;
  const int64_t row_bytes = 2 * (int64_t)a.n_kv * a.d, page_bytes = row_bytes << a.page_log2;
  uint8_t* pool = a.pools + (int64_t)(2 * layer + (part >= chunks)) * a.n_pages * page_bytes + 2 * kvh * a.d + 16 * (part % chunks);
  const int32_t* table = a.tables + (int64_t)seq * a.width;
  auto at = [&](int place) -> u32x4_t* {
    const int page = table[place >> a.page_log2];
    if ((unsigned)page >= (unsigned)a.n_pages) return nullptr;
    return reinterpret_cast<u32x4_t*>(pool + page * page_bytes + (place & ((1 << a.page_log2) - 1)) * row_bytes);
  };
  constexpr int kDeep = 4;
  for (int r0 = 0; r0 < moved; r0 += kDeep * per_step) {
    u32x4_t x[kDeep];
    u32x4_t* dst[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int r = r0 + i * per_step + mine;
      dst[i] = nullptr;
      if (!worker || r >= moved) continue;
      const int to = holes[r], from = kept[to];
      const u32x4_t* src = at(from);
      dst[i] = at(to);
      if (src == nullptr) dst[i] = nullptr;
      if (dst[i] != nullptr) x[i] = *src;
    }
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (dst[i] != nullptr) *dst[i] = x[i];
  }
  for (int r = t; r < moved; r += kEvictThreads) {
    const int to = holes[r];
    weights[to] = weights[kept[to]];
  }
  __syncthreads();
  // the recent ones: a piece is read as a whole before it is written
  for (int r0 = 0; r0 < a.recent; r0 += kDeep * per_step) {
    u32x4_t x[kDeep];
    u32x4_t* dst[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int r = r0 + i * per_step + mine;
      dst[i] = nullptr;
      if (!worker || r >= a.recent) continue;
      const u32x4_t* src = at(middle_end + r);
      dst[i] = at(ahead + r);
      if (src == nullptr) dst[i] = nullptr;
      if (dst[i] != nullptr) x[i] = *src;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (dst[i] != nullptr) *dst[i] = x[i];
  }
  for (int r0 = 0; r0 < a.recent; r0 += kEvictThreads) {
    const float x = r0 + t < a.recent ? weights[middle_end + r0 + t] : 0.f;
    __syncthreads();
    if (r0 + t < a.recent) weights[ahead + r0 + t] = x;
  }
}

}  // namespace
}  // namespace klc

using namespace klc;

extern "C" int klc_kv_evict(const klc_kv_evict_args* args, void* stream) {
  KLC_REQUIRE(args != nullptr, KLC_ERR_ARGUMENT, "klc_kv_evict: null pointer");
  const klc_kv_evict_args& x = *args;
  KLC_REQUIRE(x.pools && x.weights && x.tables && x.lengths && x.rows && x.kept && x.workspace, KLC_ERR_ARGUMENT,
              "klc_kv_evict: null pointer");
  KLC_REQUIRE(x.n_layers > 0 && x.n_seq > 0 && x.n_kv > 0 && x.n_kv <= 4096 && x.head_dim >= 8 && x.head_dim % 8 == 0 &&
                  x.head_dim <= 128 && x.n_layers * x.n_seq * x.n_kv < ((int64_t)1 << 32) / kEvictThreads,
              KLC_ERR_SHAPE, "klc_kv_evict: %lld layers, %lld sequences, %lld KV heads, head_dim %lld (8..128, multiple of 8)",
              (long long)x.n_layers, (long long)x.n_seq, (long long)x.n_kv, (long long)x.head_dim);
  KLC_REQUIRE(x.page_size >= 16 && x.page_size <= 4096 && (x.page_size & (x.page_size - 1)) == 0 && x.n_pages > 0 &&
                  x.n_pages < ((int64_t)1 << 31) && x.n_pages * x.page_size < ((int64_t)1 << 31) && x.table_width > 0 &&
                  x.table_width < ((int64_t)1 << 25) && x.table_width * x.page_size < ((int64_t)1 << 29) &&
                  x.page_size * x.n_kv * x.head_dim < ((int64_t)1 << 30),
              KLC_ERR_SHAPE, "klc_kv_evict: %lld pages of %lld tokens (a power of two, 16..4096; below 2 GiB), tables of %lld",
              (long long)x.n_pages, (long long)x.page_size, (long long)x.table_width);
  KLC_REQUIRE(x.n_rows > 0 && x.n_rows < ((int64_t)1 << 31) && x.capacity > 0 && x.capacity < ((int64_t)1 << 31) && x.keep > 0 &&
                  x.keep < ((int64_t)1 << 29) && x.recent >= 0 && x.first >= 0 && x.recent + x.first <= x.keep,
              KLC_ERR_ARGUMENT, "klc_kv_evict: %lld keys kept, of them the first %lld and the last %lld; %lld rows of %lld weights",
              (long long)x.keep, (long long)x.first, (long long)x.recent, (long long)x.n_rows, (long long)x.capacity);
  KLC_REQUIRE((uintptr_t)x.pools % 16 == 0 && ((uintptr_t)x.weights | (uintptr_t)x.kept | (uintptr_t)x.workspace) % 4 == 0,
              KLC_ERR_ARGUMENT, "klc_kv_evict: pools must be 16-byte aligned");
  KLC_REQUIRE(x.workspace_bytes >= 4 * x.n_layers * x.n_seq * x.n_kv * x.keep, KLC_ERR_ARGUMENT,
              "klc_kv_evict: workspace of %lld bytes, need %lld", (long long)x.workspace_bytes,
              (long long)(4 * x.n_layers * x.n_seq * x.n_kv * x.keep));
  auto index = [](const void* v) { return static_cast<const int32_t*>(v); };
  int page_log2 = 0;
  while ((1 << page_log2) < x.page_size) ++page_log2;
  const EvictArgs a{static_cast<uint8_t*>(x.pools), static_cast<float*>(x.weights), index(x.tables), index(x.lengths),
                    index(x.rows), static_cast<int32_t*>(x.kept), static_cast<int32_t*>(x.workspace), x.capacity, (int)x.n_seq,
                    (int)x.n_rows, (int)x.n_kv, (int)x.head_dim, (int)x.n_pages, page_log2, (int)x.table_width, (int)x.keep,
                    (int)x.recent, (int)x.first};
  evict_kernel<<<(unsigned)(x.n_layers * x.n_seq * x.n_kv), kEvictThreads, 0, as_stream(stream)>>>(a);
  return check_launch("evict_kernel");
}
