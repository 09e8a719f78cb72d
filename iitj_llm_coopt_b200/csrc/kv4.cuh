// The packed key/value cache: keys and values of a token in 4-bit codes.
//
// A head of a token holds D = 32 G numbers.  Each group of 32 neighbouring numbers x (as the engine's type holds them) has a zero
// point z and a step s, both bfloat16, and a code n in 0 .. 15 for every number; the cache's number is z + s n:
//
//   z = the largest bfloat16 <= min x      (exact for a bfloat16 engine: z then is the minimum itself)
//   s = bfloat16((max x - z) * (1 / 15))   (0 below the smallest normal float32: the group is its zero point)
//   n = clamp(rint((x - z) * (1 / s)), 0, 15)
//
// all in float32, rounded operation by operation, so the codes are defined to the bit.  A number is off by at most s / 2 (rounding s to
// bfloat16 moves the top code's number by up to 15 s 2^-8, which is less) and float32's roundings.  z + 15 s is not finite if a number of
// the group is not, if the group spans more than float32 does, or if it lies so near float32's largest number that a step rounded up
// passes it; a token with such a group in its key or its value keeps, in that head, a key whose z and s are NaN and a value of zeros:
// whoever sees the token gets NaN, and whoever does not see it cannot get one from a probability of 0 times it.  Every value that the
// cache holds is finite.
//
// A page is kv_heads blocks, one per key/value head; a block is
//   [page_size][16 G] key codes, [page_size][4 G] key (s, z), [page_size][16 G] value codes, [page_size][4 G] value (s, z)
// 40 G bytes a token (160 at D = 128, where bfloat16 takes 512), and one block is one contiguous run of bytes.  page_size is a multiple
// of 4, so every region starts on a 16-byte boundary and is read and copied in pieces of 16 bytes.
// Which nibble is which number follows from the matrix instructions that read them without a shuffle (attention_kv4_single.cu):
//   key row    word j G + g (32 bits, j < 4):       numbers 32 g + 8 j + {0, 2, 4, 6, 1, 3, 5, 7}, low nibble first
//   value row  half-word c G + g (16 bits, c < 8):  numbers 32 g + 8 (c / 2) + (c % 2) + {0, 2, 4, 6}, low nibble first
#pragma once

#include "common.cuh"

namespace {

constexpr int kKv4TokenBytes = 40;      // per group: 16 + 4 of the key, 16 + 4 of the value
constexpr int kKv4MaxDim = 256;

__host__ __device__ __forceinline__ bool kv4_geometry(int head_dim, int page_size) {
    return head_dim >= 32 && head_dim <= kKv4MaxDim && head_dim % 32 == 0 && page_size >= 4 && page_size % 4 == 0;
}
// Byte offsets inside the block of one key/value head.
__host__ __device__ __forceinline__ size_t kv4_block_bytes(int page_size, int groups) { return (size_t)page_size * kKv4TokenBytes * groups; }
__host__ __device__ __forceinline__ int kv4_key_par(int page_size, int groups) { return page_size * 16 * groups; }
__host__ __device__ __forceinline__ int kv4_value_codes(int page_size, int groups) { return page_size * 20 * groups; }
__host__ __device__ __forceinline__ int kv4_value_par(int page_size, int groups) { return page_size * 36 * groups; }

// (s, z) of a stored pair: s in the low half, z in the high half.
__device__ __forceinline__ float kv4_step(uint32_t par) { return __uint_as_float(par << 16); }
__device__ __forceinline__ float kv4_zero(uint32_t par) { return __uint_as_float(par & 0xffff0000u); }

// Number i (0 .. 7) of a key word is the nibble at this bit.
__host__ __device__ __forceinline__ constexpr int kv4_bit(int i) { return 4 * (i >> 1) + 16 * (i & 1); }

}  // namespace
