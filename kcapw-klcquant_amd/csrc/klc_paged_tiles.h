// Tiles of keys from the pages of a KV cache (gfx950): what the attention
// kernels over a paged cache share.
#pragma once

#include "klc_attn_wave.h"

namespace klc {

constexpr int kWaves = 4;             // of a workgroup
constexpr int64_t kMostBlocks = 1 << 24;  // of a launch: its threads are counted in 32 bits
constexpr int kKeys = 32;             // that a wave takes at once
constexpr int kTileLds = 64 * 1024;   // for a workgroup's tiles: two workgroups fit a CU
// keys of the tiles that a workgroup's waves share: 16 KB of K and V
template <int DP>
constexpr int kSharedTile = DP == 64 ? 64 : 32;

typedef const __attribute__((address_space(4))) int32_t* const_i32;
// a uniform element of a table, by a scalar load: vector loads would wait behind the tiles in flight
__device__ __forceinline__ int32_t table_at(const int32_t* t, int64_t i) {
  return reinterpret_cast<const_i32>(reinterpret_cast<uintptr_t>(t))[i];
}

// A lane's chunks of its bfloat16 query row, as they are.
template <class F>
__device__ __forceinline__ void load_query(u32x4_t (&q)[F::kSteps], const uint16_t* src, int d) {
#pragma unroll
  for (int st = 0; st < F::kSteps; ++st) {
    const int c = 2 * st + (int)(threadIdx.x % kWave) / 32;
    q[st] = u32x4_t{0, 0, 0, 0};
    if (F::kWhole || 8 * c < d) q[st] = *reinterpret_cast<const u32x4_t*>(src + 8 * c);
  }
}

// Has the row waited for here: past the page numbers' wait it costs nothing,
// and later it would wait for the tiles in flight too.
template <class F>
__device__ __forceinline__ void settle_query(u32x4_t (&q)[F::kSteps]) {
#pragma unroll
  for (int st = 0; st < F::kSteps; ++st) asm volatile("" : "+v"(q[st]));
}

// The row in the cache's type.  A float16 cache takes it times a power of two
// that brings its largest value to [1, 2): float16 then holds every value down
// to 2^-17 as it is, and smaller ones to the nearest multiple of 2^-24, so
// that a score is off by at most 2^-25 of the largest |q| times sum |k|.  The
// returned factor puts the power back.
template <class F, bool kF16>
__device__ __forceinline__ float convert_query(u32x4_t (&q)[F::kSteps]) {
  if constexpr (!kF16) return 1.f;
  // bit patterns of positive values are in their order, NaN and infinity above the others
  typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
  u16x2_t pair = {0, 0};
#pragma unroll
  for (int st = 0; st < F::kSteps; ++st)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      pair = __builtin_elementwise_max(pair, __builtin_bit_cast(u16x2_t, q[st][e] & 0x7fff7fffu));
  uint32_t most = (uint32_t)max(pair.x, pair.y) << 16;
  const auto both = __builtin_amdgcn_permlane32_swap(most, most, false, false);
  most = max(both[0], both[1]);
  int ex = (int)(most >> 23) - 127;
  if (most >= 0x7f800000u || most == 0) ex = 0;
#pragma unroll
  for (int st = 0; st < F::kSteps; ++st)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      q[st][e] = pack2<true>(__builtin_amdgcn_ldexpf(__uint_as_float(q[st][e] << 16), -ex),
                             __builtin_amdgcn_ldexpf(__uint_as_float(q[st][e] & 0xffff0000u), -ex));
  return __builtin_amdgcn_ldexpf(1.f, ex);
}

// What a wave loads of a tile of KT keys: kCount instructions, the first of
// rows n0 and the others kStep instructions on, each of rows of one page.  The
// lanes hold 64 page numbers of the table, so that a tile costs no memory
// access but its loads (a scalar one would hold up the LDS reads, which wait
// by the same counter).
template <class Args, class F, int KT, int kCount, int kStep>
struct PageLoads {
  const Args& a;
  int n0;
  uint32_t row_bytes, page_bytes;  // of a token, of a page (below 2^31)
  const uint16_t *k0, *v0;         // the KV head's in the pools
  const int32_t* table;            // held: page numbers from + lane of its `size`
  int held, from, size;
  bool bad;
  uint32_t lane_off[kCount];       // bytes from an instruction's first key, for load_whole

  __device__ __forceinline__ PageLoads(const Args& args, int first, int kvh) : a(args), n0(first), table(nullptr), bad(false) {
    row_bytes = 2u * (uint32_t)(a.n_kv * a.d);
    page_bytes = row_bytes << a.page_log2;
    k0 = a.k_pages + (int64_t)kvh * a.d;
    v0 = a.v_pages + (int64_t)kvh * a.d;
  }
  __device__ __forceinline__ void hold(const int32_t* t, int at, int count) {
    table = t;
    from = at;
    size = count;
    held = t[min(from + (int)(threadIdx.x % kWave), size - 1)];
    asm volatile("" : "+v"(held));  // waited for here, not again (with the tiles in flight) at every use
  }
  // Loads the tile from key `base` of the held table on to K at `k` and V at `v` of LDS, or one of the two.  Key j's
  // row is that of key at(j), which ascends and stays in one page for the rows of one instruction: keys that are not
  // visible take a visible one's, so that only its pages are asked for.
  template <bool kKey = true, bool kValue = true, class At>
  __device__ __forceinline__ void load(int base, At at, lds_u8 k, lds_u8 v) {
    const int mask = (1 << a.page_log2) - 1;
    if ((at(base + KT - 1) >> a.page_log2) - from >= kWave) hold(table, at(base) >> a.page_log2, size);
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int n = n0 + i * kStep, r = F::dma_row(n);
      const int page = __builtin_amdgcn_readlane(held, (at(base + n * F::kRowsPerDma) >> a.page_log2) - from);
      const bool wrong = (unsigned)page >= (unsigned)a.n_pages;
      bad |= wrong;
      const uint64_t start = (uint64_t)(wrong ? 0u : (uint32_t)page) * page_bytes;
      const uint32_t off = (uint32_t)(at(base + r) & mask) * row_bytes + 16u * (uint32_t)F::dma_chunk(r, a.d);
      if constexpr (kKey) load_to_lds(reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(k0) + start), off, k + n * 1024);
      if constexpr (kValue) load_to_lds(reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(v0) + start), off, v + n * 1024);
    }
  }
  // The same for a tile whose keys are all visible: what differs among lanes is worked out once.
  __device__ __forceinline__ void prepare_whole() {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int n = n0 + i * kStep, r = F::dma_row(n);
      lane_off[i] = (uint32_t)(r - n * F::kRowsPerDma) * row_bytes + 16u * (uint32_t)F::dma_chunk(r, a.d);
    }
  }
  template <bool kKey = true, bool kValue = true>
  __device__ __forceinline__ void load_whole(int base, lds_u8 k, lds_u8 v) {
    const int mask = (1 << a.page_log2) - 1;
    if (((base + KT - 1) >> a.page_log2) - from >= kWave) hold(table, base >> a.page_log2, size);
    auto start = [&](int key) {
      const int page = __builtin_amdgcn_readlane(held, (key >> a.page_log2) - from);
      const bool wrong = (unsigned)page >= (unsigned)a.n_pages;
      bad |= wrong;
      return (uint64_t)(wrong ? 0u : (uint32_t)page) * page_bytes + (uint32_t)(key & mask) * row_bytes;
    };
    auto bring = [&](int i, uint64_t at) {
      const int n = n0 + i * kStep;
      if constexpr (kKey) load_to_lds(reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(k0) + at), lane_off[i], k + n * 1024);
      if constexpr (kValue) load_to_lds(reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(v0) + at), lane_off[i], v + n * 1024);
    };
    if (mask + 1 >= KT) {  // one page
      const uint64_t at = start(base);
#pragma unroll
      for (int i = 0; i < kCount; ++i) bring(i, at + (uint32_t)((n0 + i * kStep) * F::kRowsPerDma) * row_bytes);
    } else {
#pragma unroll
      for (int i = 0; i < kCount; ++i) bring(i, start(base + (n0 + i * kStep) * F::kRowsPerDma));
    }
  }
};

// Keys outside first..last take the nearest visible one's row.
__device__ __forceinline__ auto within(int first, int last) {
  return [=](int key) { return min(max(key, first), last); };
}

// The tile's loads have landed: of the wave's own, or with kBarrier of every
// wave of the workgroup, each of which is then done with the tile before.
template <int kOutstanding, bool kBarrier>
__device__ __forceinline__ void tile_wait() {
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(kOutstanding));
  if constexpr (kBarrier) __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

template <int kValue>
struct Count {
  static constexpr int value = kValue;
};

// Four dims of a wave's sums, as its lane holds them: block e of 32 dims / 8.
template <class F>
__device__ __forceinline__ f32x4_t quad(const F& f, int i) {
  const f32x16_t& o = f.o[0][i / 4];
  const int e = i % 4 * 4;
  return f32x4_t{o[e], o[e + 1], o[e + 2], o[e + 3]};
}
// the first of them
__device__ __forceinline__ int quad_dim(int i) { return 8 * i + 4 * ((int)(threadIdx.x % kWave) / 32); }

}  // namespace klc
