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

}  // namespace kv
}  // namespace tcb
