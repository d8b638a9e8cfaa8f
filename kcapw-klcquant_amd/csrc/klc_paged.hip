// A paged KV cache of many sequences (gfx950): rotation and append of new
// tokens, and copies of pages between slots of the pools.
#include <stdlib.h>

#include "klc_common.h"

namespace klc {
namespace {

constexpr int kPagedThreads = 256;

__device__ __forceinline__ uint16_t store_bits(float f, bool f16) {
  return f16 ? __half_as_ushort(__float2half_rn(f)) : (uint16_t)f32_to_bf16_rne(f);
}

struct AppendArgs {
  const uint16_t *q, *k, *v, *cos, *sin;  // [tokens] rows, [n_positions][d / 2]
  const int32_t *positions, *slots;
  uint16_t *q_out, *k_out, *k_pages, *v_pages;
  int64_t q_stride, k_stride, v_stride;
  int tokens, n_slots, n_positions, n_heads, n_kv, d;
  bool f16;
};

// q' = (q_lo c - q_hi s, q_hi c + q_lo s), k' the same, and k', v to their
// page.  A thread takes V elements of a row and the V it is rotated with (half
// a head further on): a head of q or k, or the two halves of a value head.
// Bound by HBM: every element once in and once out in 16-byte accesses (8 of
// head sizes that are no multiple of 16): 6,001 tokens of 64 and 8 heads of
// size 64, 130 MB, in 26 to 29 us; 64 tokens in 3.6 us, the launch.
template <int V>
__global__ __launch_bounds__(kPagedThreads) void paged_append_kernel(AppendArgs a) {
  typedef uint16_t vec_t __attribute__((ext_vector_type(V)));
  const int half = a.d / 2, per_row = half / V, rows = a.n_heads + 2 * a.n_kv, per_token = rows * per_row;
  const int64_t i = (int64_t)blockIdx.x * kPagedThreads + threadIdx.x;
  if (i >= (int64_t)a.tokens * per_token) return;
  const int t = (int)(i / per_token), u = (int)(i - (int64_t)t * per_token);
  const int row = u / per_row, j = (u - row * per_row) * V;
  const bool is_q = row < a.n_heads, is_v = row >= a.n_heads + a.n_kv;
  const int head = is_q ? row : is_v ? row - a.n_heads - a.n_kv : row - a.n_heads;
  const uint16_t* src = (is_q ? a.q + t * a.q_stride : is_v ? a.v + t * a.v_stride : a.k + t * a.k_stride) + (int64_t)head * a.d + j;
  const vec_t x = *reinterpret_cast<const vec_t*>(src), y = *reinterpret_cast<const vec_t*>(src + half);
  const int slot = is_q ? -1 : a.slots[t];
  const bool kept = slot >= 0 && slot < a.n_slots;
  const int64_t at = ((int64_t)slot * a.n_kv + head) * a.d + j;
  vec_t lo, hi;
  if (is_v) {
    if (!kept) return;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      lo[e] = a.f16 ? store_bits(bf16_to_f32(x[e]), true) : x[e];
      hi[e] = a.f16 ? store_bits(bf16_to_f32(y[e]), true) : y[e];
    }
    *reinterpret_cast<vec_t*>(a.v_pages + at) = lo;
    *reinterpret_cast<vec_t*>(a.v_pages + at + half) = hi;
    return;
  }
  const int pos = a.positions[t];
  const bool known = pos >= 0 && pos < a.n_positions;
  const int64_t angle = (int64_t)(known ? pos : 0) * half + j;
  const vec_t c = *reinterpret_cast<const vec_t*>(a.cos + angle), s = *reinterpret_cast<const vec_t*>(a.sin + angle);
  float first[V], second[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    // products of bfloat16 values are exact in float32: one rounding of the sum there, one to the result's type
    const float xf = bf16_to_f32(x[e]), yf = bf16_to_f32(y[e]), cf = bf16_to_f32(c[e]), sf = bf16_to_f32(s[e]);
    first[e] = known ? fmaf(xf, cf, -(yf * sf)) : __uint_as_float(0x7fc00000u);
    second[e] = known ? fmaf(yf, cf, xf * sf) : __uint_as_float(0x7fc00000u);
    lo[e] = (uint16_t)f32_to_bf16_rne(first[e]);
    hi[e] = (uint16_t)f32_to_bf16_rne(second[e]);
  }
  uint16_t* dst = is_q ? a.q_out : a.k_out;
  if (dst != nullptr) {
    dst += ((int64_t)t * (is_q ? a.n_heads : a.n_kv) + head) * a.d + j;
    *reinterpret_cast<vec_t*>(dst) = lo;
    *reinterpret_cast<vec_t*>(dst + half) = hi;
  }
  if (!kept) return;
  if (a.f16) {
#pragma unroll
    for (int e = 0; e < V; ++e) lo[e] = store_bits(first[e], true), hi[e] = store_bits(second[e], true);
  }
  *reinterpret_cast<vec_t*>(a.k_pages + at) = lo;
  *reinterpret_cast<vec_t*>(a.k_pages + at + half) = hi;
}

// Page moves of one launch, in its arguments: no copy to the device, and a
// graph keeps them.
constexpr int kMovesPerLaunch = 384;
struct Moves {
  int32_t src[kMovesPerLaunch], dst[kMovesPerLaunch];
};
// Bound by HBM.  16 bytes a thread, past the caches on both ways, as neither
// page is soon read: 400 pages of 64 KB in 8 pools (419 MB moved) take 73 us
// (5.7 TB/s), 16 in 72 pools (151 MB) 27; cached 78 and 30, with 32 bytes a
// thread 81 and 28, with 64 82 and 32, with 64 cached 88 and 37.
constexpr int kCopyBytes = kPagedThreads * 16;  // of a workgroup

__global__ __launch_bounds__(kPagedThreads) void copy_pages_kernel(uint8_t* __restrict__ pool, int64_t pool_bytes,
                                                                   int64_t page_bytes, Moves moves) {
  uint8_t* base = pool + blockIdx.z * pool_bytes;
  const int64_t at = (int64_t)blockIdx.x * kCopyBytes + threadIdx.x * 16;
  if (at >= page_bytes) return;
  const u32x4_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(base + moves.src[blockIdx.y] * page_bytes + at));
  __builtin_nontemporal_store(x, reinterpret_cast<u32x4_t*>(base + moves.dst[blockIdx.y] * page_bytes + at));
}

}  // namespace
}  // namespace klc

using namespace klc;

extern "C" int klc_kv_append(const klc_kv_append_args* args, void* stream) {
  KLC_REQUIRE(args != nullptr, KLC_ERR_ARGUMENT, "klc_kv_append: null pointer");
  const klc_kv_append_args& x = *args;
  KLC_REQUIRE(x.q && x.k && x.v && x.cos_half && x.sin_half && x.positions && x.slots && x.q_out && x.k_pages && x.v_pages,
              KLC_ERR_ARGUMENT, "klc_kv_append: null pointer");
  KLC_REQUIRE(x.n_heads > 0 && x.n_kv > 0 && x.n_heads <= 4096 && x.n_kv <= 4096 && x.head_dim >= 8 &&
                  x.head_dim % 8 == 0 && x.head_dim <= 128,
              KLC_ERR_SHAPE, "klc_kv_append: heads %lld / %lld, head_dim %lld (8..128, multiple of 8)",
              (long long)x.n_heads, (long long)x.n_kv, (long long)x.head_dim);
  KLC_REQUIRE(x.tokens > 0 && x.tokens < ((int64_t)1 << 30) && x.n_positions > 0 &&
                  x.n_positions < ((int64_t)1 << 31) && x.n_slots > 0 && x.n_slots < ((int64_t)1 << 31),
              KLC_ERR_ARGUMENT, "klc_kv_append: %lld tokens, %lld positions, %lld slots", (long long)x.tokens,
              (long long)x.n_positions, (long long)x.n_slots);
  KLC_REQUIRE(x.q_stride >= x.n_heads * x.head_dim && x.k_stride >= x.n_kv * x.head_dim &&
                  x.v_stride >= x.n_kv * x.head_dim && (x.q_stride | x.k_stride | x.v_stride) % 8 == 0,
              KLC_ERR_SHAPE, "klc_kv_append: token strides %lld, %lld, %lld (multiples of 8, no overlap)",
              (long long)x.q_stride, (long long)x.k_stride, (long long)x.v_stride);
  KLC_REQUIRE(((uintptr_t)x.q | (uintptr_t)x.k | (uintptr_t)x.v | (uintptr_t)x.cos_half | (uintptr_t)x.sin_half |
               (uintptr_t)x.q_out | (uintptr_t)x.k_out | (uintptr_t)x.k_pages | (uintptr_t)x.v_pages) % 16 == 0,
              KLC_ERR_ARGUMENT, "klc_kv_append: tensors must be 16-byte aligned");
  KLC_REQUIRE(x.kv_dtype == KLC_DTYPE_BF16 || x.kv_dtype == KLC_DTYPE_F16, KLC_ERR_UNSUPPORTED,
              "klc_kv_append: kv_dtype %lld (bfloat16 or float16)", (long long)x.kv_dtype);
  auto in = [](const void* p) { return static_cast<const uint16_t*>(p); };
  auto index = [](const void* p) { return static_cast<const int32_t*>(p); };
  auto out = [](void* p) { return static_cast<uint16_t*>(p); };
  const AppendArgs a{in(x.q), in(x.k), in(x.v), in(x.cos_half), in(x.sin_half), index(x.positions), index(x.slots),
                     out(x.q_out), out(x.k_out), out(x.k_pages), out(x.v_pages), x.q_stride, x.k_stride, x.v_stride,
                     (int)x.tokens, (int)x.n_slots, (int)x.n_positions, (int)x.n_heads, (int)x.n_kv, (int)x.head_dim,
                     x.kv_dtype == KLC_DTYPE_F16};
  const bool wide = x.head_dim % 16 == 0;
  const int64_t items = x.tokens * (x.n_heads + 2 * x.n_kv) * (x.head_dim / 2 / (wide ? 8 : 4));
  const int64_t blocks = (items + kPagedThreads - 1) / kPagedThreads;
  KLC_REQUIRE(blocks < ((int64_t)1 << 31), KLC_ERR_SHAPE, "klc_kv_append: %lld tokens of %lld heads",
              (long long)x.tokens, (long long)x.n_heads);
  if (wide)
    paged_append_kernel<8><<<(unsigned)blocks, kPagedThreads, 0, as_stream(stream)>>>(a);
  else
    paged_append_kernel<4><<<(unsigned)blocks, kPagedThreads, 0, as_stream(stream)>>>(a);
  return check_launch("paged_append_kernel");
}

extern "C" int klc_kv_copy_pages(void* pools, int64_t n_pools, int64_t n_pages, int64_t page_bytes, const int32_t* src,
                                 const int32_t* dst, int64_t n, void* stream) {
  KLC_REQUIRE(pools && src && dst, KLC_ERR_ARGUMENT, "klc_kv_copy_pages: null pointer");
  KLC_REQUIRE(n_pools > 0 && n_pools <= 65535 && n_pages > 0 && n_pages < ((int64_t)1 << 31) && page_bytes > 0 &&
                  page_bytes % 16 == 0 && page_bytes <= ((int64_t)1 << 30) && n >= 0 && (uintptr_t)pools % 16 == 0,
              KLC_ERR_ARGUMENT,
              "klc_kv_copy_pages: %lld moves in %lld pools of %lld pages of %lld bytes (a multiple of 16, 16-byte aligned)",
              (long long)n, (long long)n_pools, (long long)n_pages, (long long)page_bytes);
  if (n == 0) return KLC_OK;
  // destinations, a bit a page
  uint8_t* taken = static_cast<uint8_t*>(calloc((size_t)(n_pages + 7) / 8, 1));
  KLC_REQUIRE(taken != nullptr, KLC_ERR_ARGUMENT, "klc_kv_copy_pages: no memory to check %lld pages", (long long)n_pages);
  int64_t bad = -1;
  bool range = false;
  for (int64_t i = 0; i < n && bad < 0; ++i) {
    range = src[i] < 0 || src[i] >= n_pages || dst[i] < 0 || dst[i] >= n_pages;
    if (range || (taken[dst[i] / 8] >> dst[i] % 8 & 1)) bad = i;
    else taken[dst[i] / 8] |= (uint8_t)(1 << dst[i] % 8);
  }
  for (int64_t i = 0; i < n && bad < 0; ++i)
    if (taken[src[i] / 8] >> src[i] % 8 & 1) bad = i;
  free(taken);
  KLC_REQUIRE(bad < 0 || !range, KLC_ERR_ARGUMENT, "klc_kv_copy_pages: move %lld from page %d to page %d of %lld",
              (long long)bad, src[bad], dst[bad], (long long)n_pages);
  KLC_REQUIRE(bad < 0, KLC_ERR_ARGUMENT,
              "klc_kv_copy_pages: move %lld from page %d to page %d: a destination is another move's source or destination",
              (long long)bad, src[bad], dst[bad]);
  for (int64_t at = 0; at < n; at += kMovesPerLaunch) {
    const int count = (int)(n - at < kMovesPerLaunch ? n - at : kMovesPerLaunch);
    Moves m;
    for (int i = 0; i < kMovesPerLaunch; ++i) {
      m.src[i] = src[at + (i < count ? i : 0)];
      m.dst[i] = dst[at + (i < count ? i : 0)];
    }
    const dim3 grid((unsigned)((page_bytes + kCopyBytes - 1) / kCopyBytes), (unsigned)count, (unsigned)n_pools);
    copy_pages_kernel<<<grid, kPagedThreads, 0, as_stream(stream)>>>(static_cast<uint8_t*>(pools), n_pages * page_bytes,
                                                                     page_bytes, m);
    const int rc = check_launch("copy_pages_kernel");
    if (rc) return rc;
  }
  return KLC_OK;
}
