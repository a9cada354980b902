// The 4-bit cache format: MX fp4.  32 neighbouring dims of a token's head share a
// power of two 2^e, held as the byte e + 127 (255: the group holds a NaN or an
// infinity and is NaN as a whole), and each dim is an e2m1 code: sign, then 0, 1/2, 1,
// 3/2, 2, 3, 4 or 6 times 2^e.
//
// e is the least with max |x| <= 7 * 2^e, so that every dim is within half of its
// step (the top step, 4 to 6 and on to 8, is 2), held within [-125, 125]: the least
// level is then a normal number in 32 bits and in bf16, and the largest finite.
//
// A block of one KV head: block_size * D / 2 bytes of codes, an even dim in the low
// nibble, then block_size * D / 32 scale bytes.  A row of 64 query dims against a
// token's keys is one matrix instruction's operand as it lies in memory, so keys are
// token by token.  Values enter their product transposed, a lane holding four tokens
// of D / 16 dims, so they lie four tokens at a time, sixteenth after sixteenth of the
// dims, and the scale bytes of four tokens are one word.
#pragma once

#include <stdint.h>

namespace fd {

// Byte of a token's dims [d, d + 1] within its block, and of dims [d, d + 31]' scale.
template <int D>
__host__ __device__ __forceinline__ int fp4_key_at(int tok, int d) {
  return tok * (D / 2) + d / 2;
}
template <int D>
__host__ __device__ __forceinline__ int fp4_value_at(int tok, int d) {
  constexpr int P = D / 16;  // dims of a piece
  return (tok >> 2) * (2 * D) + (d / P) * (2 * P) + (tok & 3) * (P / 2) + (d % P) / 2;
}
template <int D>
__host__ __device__ __forceinline__ int fp4_key_scale_at(int block_size, int tok, int d) {
  return block_size * (D / 2) + tok * (D / 32) + d / 32;
}
template <int D>
__host__ __device__ __forceinline__ int fp4_value_scale_at(int block_size, int tok, int d) {
  return block_size * (D / 2) + (tok >> 2) * (D / 8) + (d / 32) * 4 + (tok & 3);
}

constexpr uint32_t kFp4NaN = 255;

// Scale byte of a group whose largest magnitude has these bits in 32-bit floating
// point: the exponent rounded up past 1.75 (7 = 1.75 * 2^2).
__host__ __device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return kFp4NaN;
  const uint32_t b = (amax_bits + 0x1fffffu) >> 23;
  return b < 4 ? 2 : (b > 254 ? 252 : b - 2);
}

// What every entry point asks of the caches (defined beside the append); fn names it
// in error messages.
int check_fp4_caches(const char* fn, int64_t head_dim, int64_t block_size, int64_t num_blocks, int64_t num_kv_heads,
                     const void* k_cache, const int64_t* k_stride, const void* v_cache, const int64_t* v_stride);

}  // namespace fd
