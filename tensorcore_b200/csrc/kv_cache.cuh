// Layout of the paged 4-bit key/value cache, shared by the kernels that write it (kv_cache.cu) and read it
// (attention_paged.cu, attention_paged_tc.cu).
//
// A page holds `page_tokens` tokens (a multiple of 16) of every K/V head: per head page_tokens / 16 tiles, a tile 16
// tokens of one head, 576 bytes for each of the NB = head_dim / 32 blocks of a row:
//
//   keys' codes     [token 16][t 4][block NB] words: nibble j is element 32 block + 8 t + j
//   keys' scales    [token 16][block NB] fp16
//   values' codes   [h 2][g 8][t 4][block NB] words: half e, nibble i is element 32 block + 4 g + i of token 8 h + 2 t + e
//   values' scales  [h 2][t 4][block NB][e 2] fp16
//
// The orders are those of the m16n8k16 fragments of the decode kernel (keys as rows of K Q^T, elements as rows of
// V^T P^T): lane 4 g + t finds its part of 16 keys in two pieces of 4 NB bytes, of 16 values too, neighbouring lanes
// in neighbouring pieces, and one mask turns a word into two binary16 operands.  A tile is one run of bytes, a multiple of 64, and so is
// a head's part of a page: a bulk copy each.
#pragma once

#include <stdint.h>

namespace tcb {
namespace kv {

constexpr int kTile = 16;                                             // tokens of a tile
__host__ __device__ constexpr int tile_bytes(int nb) { return 576 * nb; }
__host__ __device__ constexpr int key_scales_at(int nb) { return 256 * nb; }
__host__ __device__ constexpr int values_at(int nb) { return 288 * nb; }
__host__ __device__ constexpr int value_scales_at(int nb) { return 544 * nb; }
// Byte offsets inside a tile, of token r's part.
__host__ __device__ constexpr int key_word(int nb, int r, int t, int block) { return ((r * 4 + t) * nb + block) * 4; }
__host__ __device__ constexpr int key_scale(int nb, int r, int block) { return key_scales_at(nb) + (r * nb + block) * 2; }
__host__ __device__ constexpr int value_half(int nb, int r, int g, int block) {
    return values_at(nb) + ((((r >> 3) * 8 + g) * 4 + ((r & 7) >> 1)) * nb + block) * 4 + (r & 1) * 2;
}
__host__ __device__ constexpr int value_scale(int nb, int r, int block) {
    return value_scales_at(nb) + (((r >> 3) * 4 + ((r & 7) >> 1)) * nb + block) * 4 + (r & 1) * 2;
}

// A word's eight codes minus 8 as fp16 pairs: nibbles 0 and 4, 1 and 5, 2 and 6, 3 and 7.  Put under 1024 or 64, whose last places are 1
// and 1 / 16, less 1032 or 72: exact (a known way to make small integers floating-point numbers).
__device__ __forceinline__ uint32_t less8_low(uint32_t x) {
    uint32_t r;
    asm("{\n\t.reg .b32 t;\n\tlop3.b32 t, %1, %2, %3, 0xEA;\n\tadd.rn.f16x2 %0, t, %4;\n\t}" : "=r"(r) : "r"(x), "r"(0x000F000Fu), "r"(0x64006400u), "r"(0xE408E408u));
    return r;
}
__device__ __forceinline__ uint32_t less8_high(uint32_t x) {
    uint32_t r;
    asm("{\n\t.reg .b32 t;\n\tlop3.b32 t, %1, %2, %3, 0xEA;\n\tadd.rn.f16x2 %0, t, %4;\n\t}" : "=r"(r) : "r"(x), "r"(0x00F000F0u), "r"(0x54005400u), "r"(0xD480D480u));
    return r;
}
__device__ __forceinline__ void less8(uint32_t w, uint32_t (&r)[4]) {
    r[0] = less8_low(w);
    r[1] = less8_high(w);
    r[2] = less8_low(w >> 8);
    r[3] = less8_high(w >> 8);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
}  // namespace kv
}  // namespace tcb
