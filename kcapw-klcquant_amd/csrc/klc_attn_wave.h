// Attention over tiles of keys with matrix instructions (gfx950): what the
// prompt and the batch attention kernels share.
//
// A wave owns RB blocks of 32 query rows and takes the keys in tiles of KT.
// It computes the transposed product S^T = K Q^T with v_mfma_f32_32x32x16, so
// a lane holds scores of ONE query row (column lane % 32): 16 of every 32
// keys, the other 16 in lane ^ 32.  The running maximum and sum of the
// softmax then need one exchange between the two halves a tile, and the
// probabilities are, in the registers where they are, the B operand of
// O^T = V^T P^T: the accumulator's row order (8 (i / 4) + 4 (lane / 32) +
// i % 4) only permutes the keys of the contraction, and the V operand is read
// with the same permutation by LDS transpose reads.
//
// K and V tiles come into LDS by global-to-LDS loads (no register round
// trip), 16-byte chunks of a row in XOR order so that neither the K reads
// (32 rows x 16 bytes) nor the V transpose reads (4 rows x 64 bytes) meet in
// a bank.
#pragma once

#include "klc_common.h"

namespace klc {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t* lds_u8;
typedef __attribute__((address_space(3))) const uint8_t* lds_cu8;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLazyMax = 8.f;  // powers of two that a score may pass the running maximum by before it moves

template <bool kF16>
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// two floats rounded to nearest even in the matrix operand's type
template <bool kF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const f32x2_t v = {a, b};
  if constexpr (kF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

// acc + both halves of a packed pair, in float32
template <bool kF16>
__device__ __forceinline__ float add2(uint32_t p, float acc) {
  if constexpr (kF16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, p), f16x2_t{(_Float16)1.f, (_Float16)1.f}, acc, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, p), bf16x2_t{(__bf16)1.f, (__bf16)1.f}, acc, false);
}

// 16 bytes a lane from memory to dst + 16 lane of LDS (dst uniform), counted
// by vmcnt.  In assembly because the compiler, told of the load, waits for
// every load in flight before any LDS read that might meet it; the kernels'
// own waits order them by tile.  It has no output register, and nothing reads
// its LDS before those waits.  m0 is reserved, so that the compiler keeps
// nothing in it and naming it as clobbered has no defined meaning; no other
// instruction of these kernels uses it, which a test of the compiled code checks.
__device__ __forceinline__ void load_to_lds(const uint16_t* src, lds_u8 dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"((uint32_t)(uintptr_t)dst), "v"(src)
               : "memory");
}

// the same from base + offset bytes, base uniform and offset below 2^31
__device__ __forceinline__ void load_to_lds(const uint16_t* base, uint32_t offset, lds_u8 dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"((uint32_t)(uintptr_t)dst), "v"(offset), "s"(base)
               : "memory");
}

// the other half's value beside the lane's own: both halves get the same pair
__device__ __forceinline__ float max_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// a sink logit in powers of two; a finite one stays finite
__device__ __forceinline__ float sink_log2(uint16_t bits) {
  const float sink = bf16_to_f32(bits);
  return fabsf(sink) < INFINITY ? fminf(fmaxf(sink * kLog2e, -3e38f), 3e38f) : sink;
}

// One wave's state and one tile's work.
//   DP     head size the tiles are laid out for (64 or 128)
//   kFull  the head size is DP; else it is d < DP, a multiple of 8
//   RB     blocks of 32 query rows
//   KT     keys of a tile (32 or 64)
template <int DP, bool kF16, bool kFull, int RB, int KT>
struct AttnWave {
  static constexpr bool kWhole = kFull;
  static constexpr int kRowBytes = 2 * DP;
  static constexpr int kChunks = DP / 8;                // 16-byte chunks of a row
  static constexpr int kSteps = DP / 16;                // MFMAs of a score block
  static constexpr int kDimBlocks = DP / 32;
  static constexpr int kMatBytes = KT * kRowBytes;      // one tile of K or of V
  static constexpr int kStage = 2 * kMatBytes;
  static constexpr int kRowsPerDma = kWave / kChunks;   // rows that one load instruction of a wave brings
  static constexpr int kDmas = KT / kRowsPerDma;        // load instructions of a tile of K or of V

  u32x4_t q[RB][kSteps];
  f32x16_t o[RB][kDimBlocks];
  float m[RB], l[RB];  // maximum (in powers of two, scaled) and this half's part of the sum

  lds_cu8 k_at[kSteps];          // this lane's K chunk of step s, key lane % 32
  lds_cu8 v_at[2][kDimBlocks];   // its V piece of (8-key half u, dim block)
  int d;

  // position of chunk c of row r
  static __device__ __forceinline__ int swizzle(int r) {
    if constexpr (DP == 64) {
      const int x = (r >> 1) & 7;
      return ((x & 1) << 2) | (x & 2) | (x >> 2);
    } else {
      return ((r & 3) << 2) | ((r >> 2) & 3);
    }
  }

  __device__ __forceinline__ void init(lds_u8 ring, int head_dim) {
    d = kFull ? DP : head_dim;
    const int lane = threadIdx.x % kWave, h = lane / 32, key = lane % 32, i = lane % 16, grp = (lane / 16) % 2;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      k_at[s] = ring + key * kRowBytes + (((2 * s + h) ^ swizzle(key)) << 4);
      asm volatile("" : "+v"(k_at[s]));  // the LDS reads are ordered by the ring's own waits
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int db = 0; db < kDimBlocks; ++db) {
        const int row = 8 * u + 4 * h + i / 4, chunk = 4 * db + 2 * grp + (i % 4) / 2;
        v_at[u][db] = ring + row * kRowBytes + ((chunk ^ swizzle(row)) << 4) + (i & 1) * 8;
        asm volatile("" : "+v"(v_at[u][db]));
      }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m[rb] = -INFINITY;
      l[rb] = 0.f;
#pragma unroll
      for (int db = 0; db < kDimBlocks; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[rb][db][e] = 0.f;
    }
  }

  // Load instruction n of a K or V tile: the row it brings to this lane, and the chunk of that row.
  static __device__ __forceinline__ int dma_row(int n) { return n * kRowsPerDma + (int)(threadIdx.x % kWave) / kChunks; }
  static __device__ __forceinline__ int dma_chunk(int row, int head_dim) {
    const int c = (int)(threadIdx.x % kChunks) ^ swizzle(row);
    return kFull ? c : min(c, head_dim / 8 - 1);  // chunks past the head repeat its last: their K is cleared, their V unused
  }

  // Scores of the K tile at `stage`: s[rb][kb][i] is q . k of key 32 kb + 8 (i / 4) + 4 (lane / 32) + i % 4.
  __device__ __forceinline__ void scores(int stage, f32x16_t (&s)[RB][KT / 32]) const {
    const bool upper = threadIdx.x % kWave >= 32;
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[rb][kb][e] = 0.f;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      if (!kFull && 16 * st >= d) break;
#pragma unroll
      for (int kb = 0; kb < KT / 32; ++kb) {
        u32x4_t k = *reinterpret_cast<__attribute__((address_space(3))) const u32x4_t*>(k_at[st] + stage + kb * 32 * kRowBytes);
        if (!kFull && 16 * st + 8 >= d && upper) k = u32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) s[rb][kb] = mfma32<kF16>(k, q[rb][st], s[rb][kb]);
      }
    }
  }

  // Brings row block rb's maximum up to the scores s, and what was summed below the old one to the new.
  __device__ __forceinline__ void raise(int rb, const f32x16_t (&s)[KT / 32], float c2) {
    float t = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) t = fmaxf(t, s[kb][e]);
    t = max_halves(t) * c2;
    // the maximum moves only when a row's scores pass it by 2^8: below that the sums cannot overflow, and the
    // rescaling of o (all of it, 32 to 128 registers) is skipped for most tiles
    if (__any(t > m[rb] + kLazyMax)) {
      const float next = fmaxf(m[rb], t), base = next == -INFINITY ? 0.f : next;
      const float alpha = __builtin_amdgcn_exp2f(m[rb] - base);
      m[rb] = next;
      l[rb] *= alpha;
#pragma unroll
      for (int db = 0; db < kDimBlocks; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[rb][db][e] *= alpha;
    }
  }

  // p = exp2(c2 s - m) of row block rb, packed, and its part of the sum; with kPlain also of the sum of p before packing
  template <bool kPlain = false>
  __device__ __forceinline__ void weigh(int rb, const f32x16_t (&s)[KT / 32], float c2, u32x4_t (&p)[KT / 16],
                                        float* plain = nullptr) {
    const float base = m[rb] == -INFINITY ? 0.f : m[rb];
    float sum = l[rb];
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[kb][e], c2, -base)), y = __builtin_amdgcn_exp2f(fmaf(s[kb][e + 1], c2, -base));
        if constexpr (kPlain) *plain += x + y;
        const uint32_t w = pack2<kF16>(x, y);
        p[2 * kb + e / 8][(e % 8) / 2] = w;
        sum = add2<kF16>(w, sum);  // the sum of what the values are multiplied by
      }
    l[rb] = sum;
  }

  __device__ __forceinline__ void softmax(int rb, const f32x16_t (&s)[KT / 32], float c2, u32x4_t (&p)[KT / 16]) {
    raise(rb, s, c2);
    weigh(rb, s, c2, p);
  }

  __device__ __forceinline__ u32x4_t v_operand(int stage, int t, int db) const {
    typedef __attribute__((address_space(3))) s16x4_t* tr_ptr;
    const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(v_at[0][db] + stage + 16 * t * kRowBytes));
    const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(v_at[1][db] + stage + 16 * t * kRowBytes));
    const u32x2_t x = __builtin_bit_cast(u32x2_t, a), y = __builtin_bit_cast(u32x2_t, b);
    return u32x4_t{x.x, x.y, y.x, y.y};
  }

  __device__ __forceinline__ void values(int stage, const u32x4_t (&p)[RB][KT / 16]) {
#pragma unroll
    for (int t = 0; t < KT / 16; ++t)
#pragma unroll
      for (int db = 0; db < kDimBlocks; ++db) {
        if (!kFull && 32 * db >= d) break;
        const u32x4_t v = v_operand(stage, t, db);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) o[rb][db] = mfma32<kF16>(v, p[rb][t], o[rb][db]);
      }
  }
};

// Clears the V rows of a tile outside [from, to), whose values no query sees
// (0 * inf would make NaN of them); the caller orders it.
template <class F, int KT>
__device__ __forceinline__ void clear_values(lds_u8 values, int from, int to, int thread, int threads) {
  for (int i = thread; i < KT * F::kChunks; i += threads) {
    const int r = i / F::kChunks;
    if (r < from || r >= to)
      *reinterpret_cast<__attribute__((address_space(3))) u32x4_t*>(values + i * 16) = u32x4_t{0, 0, 0, 0};
  }
}

}  // namespace klc
