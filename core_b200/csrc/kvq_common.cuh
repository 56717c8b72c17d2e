// The quantised KV cache's layout, shared by its writer, its reader and the
// attention over it.
//
// A row is one token of one KV head: 128 channels in 4 or 8 bits, with an f16
// scale s and an f16 zero z for each group of 32, 64 or 128 neighbouring
// channels; a code n stands for n s + z.  codes (B, Hkv, capacity, 16 bits)
// bytes, meta (B, Hkv, capacity, 128 / group) words (s in the low half).
//
// Inside a 32-bit word, even channels lie in the low half and odd ones in the
// high half (4 bits: e0 e2 e4 e6 e1 e3 e5 e7 from the lowest nibble up; 8 bits:
// e0 e2 e1 e3), so that one mask takes a pair of neighbouring channels out as
// the two halves of a register.
//
// Keys: the 16-byte chunk t (8 bits: chunks t and 4 + t) of a row holds what
// lane t of a quad feeds to the matrix instruction, channels 32 b + 8 t .. + 7
// for b = 0..3 (8 bits: b = 0, 1 and b = 2, 3).  Values: words in channel order.
// The exclusive-ors with the token's low bits keep the attention kernel's shared
// memory reads free of bank conflicts: a tile's bytes arrive as they lie here.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace core {
namespace kvq {

constexpr int kD = 128;
constexpr float kLimit = 61440.0f;  // inputs saturate here: n s + z then stays within f16

// Byte exclusive-or of a row's offsets for token `tok`.
template <int kBits>
__device__ __forceinline__ uint32_t key_swizzle(uint32_t tok) {
  return kBits == 4 ? 0u : (tok & 1u) << 6;
}
template <int kBits>
__device__ __forceinline__ uint32_t value_swizzle(uint32_t tok) {
  return kBits == 4 ? (tok & 2u) << 4 : (tok & 3u) << 5;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  return __byte_perm(a, b, sel);
}

__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// (a & mask) | bits in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(bits));
  return d;
}

// Pair i of a word (4 bits: i = 0..3, 8 bits: i = 0, 1) as two f16 integers
// n, through 1024 + n (exponent bits or-ed above the code), from which the
// offset is taken off exactly.  The upper nibble of a byte is read in place
// as 16 n: (1024 + 16 n) / 16 - 64.
template <int kBits>
__device__ __forceinline__ __half2 code_pair(uint32_t w, int i) {
  const __half2 off = __floats2half2_rn(-1024.f, -1024.f);
  if (kBits == 8)
    return __hadd2(as_half2(and_or(i ? w >> 8 : w, 0x00ff00ffu, 0x64006400u)), off);
  const uint32_t x = i & 2 ? w >> 8 : w;
  if (i & 1)
    return __hfma2(as_half2(and_or(x, 0x00f000f0u, 0x64006400u)), __floats2half2_rn(0.0625f, 0.0625f),
                   __floats2half2_rn(-64.f, -64.f));
  return __hadd2(as_half2(and_or(x, 0x000f000fu, 0x64006400u)), off);
}

}  // namespace kvq
}  // namespace core
