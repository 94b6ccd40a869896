// The 8-bit KV cache's records and its number format, shared by the kernels that write and read them.
//
// Page records (include/jit_moe.h): per (page, kv head) 4,224 bytes = 33 lines of 128 --
//   [0, 2048)     K codes [2][4][16 slots][16 dims]: dim 64 i + 16 g + x.  The 16 bytes a lane (g = lane / 16,
//                 slot = lane % 16) loads are its operand rows of two 16x16x32 matrix instructions, and a wave's
//                 load is 1 KB contiguous.
//   [2048, 4096)  V codes [2][4][16][4][4]: dim 16 (4 q + c) + r, slot 4 g + j.  Lane (g, r)'s 16 bytes are 4 of its
//                 keys in each of 4 output tiles.
//   [4096, 4224)  fp32 scales, K of the 16 slots, then V: one line, read as the float4 of a lane's 4 keys.
// A block is one token of one kv head (K and V apart).  Tokens arrive one at a time: a longer block would be rounded
// again whenever a louder token joins it, and what the cache holds of given k and v would depend on how they arrived.
// (Attention's own bits are another matter: a prompt chunk's key parts are chosen by the chunk.)  Its scale is a power
// of two: e4m3 keeps its relative precision at any scale, code x scale is exact in bf16, and the conversions that take a
// power of two apply it for nothing.
#pragma once

#include "common.hpp"

namespace kv8 {

constexpr int kD = JIT_HEAD_DIM;
constexpr int kPage = JIT_PAGE_TOKENS;
constexpr int kRec = JIT_KV8_RECORD_BYTES;
constexpr int kVOff = kPage * kD, kScaleOff = 2 * kPage * kD;
static_assert(kRec == kScaleOff + 2 * kPage * 4, "K codes, V codes, scales");
constexpr int kMinExp = -100, kMaxExp = 118;  // a scale's exponent: 2^-e and 448 2^e stay normal fp32 numbers

// (a pool has fewer than 2^32 records: one 32 x 32 -> 64 bit product)
__device__ __forceinline__ const uint8_t *record(const uint8_t *pool, int page, int Hkv, int h) {
  return pool + (uint64_t)((uint32_t)page * (uint32_t)Hkv + (uint32_t)h) * kRec;
}
__device__ __forceinline__ uint8_t *record(uint8_t *pool, int page, int Hkv, int h) {
  return pool + (uint64_t)((uint32_t)page * (uint32_t)Hkv + (uint32_t)h) * kRec;
}

// The scale's exponent of a block whose largest finite magnitude is amax: amax 2^-e lies in (224, 448] (1.75 2^8 is
// the largest e4m3), clamped; 0 for a block of zeros.
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u == 0) return 0;
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kMinExp ? kMinExp : (e > kMaxExp ? kMaxExp : e);
}
__device__ __forceinline__ float exp_bits(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
// |x| of a finite x, else 0: a block's scale comes from its finite values
__device__ __forceinline__ float mag(float x) { return finite(x) ? fabsf(x) : 0.0f; }
// x 2^-e ready for the conversion: within +-448 (past it only where e was clamped), NaN where x is not finite
__device__ __forceinline__ float to_code_range(float x, float inv) {
  const float y = x * inv;
  return finite(x) ? fminf(fmaxf(y, -448.0f), 448.0f) : __uint_as_float(0x7fc00000u);
}
// two e4m3 codes (round to nearest even) in the low 16 bits
__device__ __forceinline__ uint32_t codes2(float a, float b) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}

// ------------------------------------------------------------------ reading
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2v_t __attribute__((ext_vector_type(2)));

union FragH {  // 8 fp16 = one 32x32x16 operand fragment of one lane
  f16x8_t v;
  uint32_t u[4];
  uint4 q;
};

// four codes -> two words of bf16 (times the power of two s) or fp16: exact, 4 significant bits
__device__ __forceinline__ void to_bf16(uint32_t w, float s, uint32_t &lo, uint32_t &hi) {
  lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false));
  hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true));
}
__device__ __forceinline__ void to_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
  lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
  hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
}
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  const f16x2_t v = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(uint32_t, v);
}
// the bytes of a word of 4 consecutive keys of which the first n count
__device__ __forceinline__ uint32_t keep_bytes(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u; }

}  // namespace kv8
