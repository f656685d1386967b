// kv4.cuh -- layout of the 4-bit key / value cache, shared by the kernels that
// write it (kv4_cache.cu) and the attention that reads it (kv4_decode.cu).
//
// A pool is [num_blocks][num_kv_heads][block_size / 16] tiles; a tile holds 16
// consecutive tokens of one kv head:
//   key codes    16 * D / 2 bytes
//   value codes  16 * D / 2 bytes
//   scales       16 tokens x [keys: D / G x (lo, scale) | values: the same],
//                two 16-bit numbers (bf16 or f16, the type of the rows) each
// so any run of tokens is a run of whole tiles, each contiguous in memory.
// A code c of a group of G dims stands for lo + scale * c.
//
// Codes are packed eight to a 32-bit word, and words are ordered so that a lane
// of a warp reads what it feeds to mma.m16n8k16 from global memory with wide loads (16
// bytes; 8 for keys of 64 dims), a warp's adjacent.  Lane l = 4 r + q (r = l / 4, q = l % 4):
//   keys (A operand, rows = tokens r and r + 8): lane q of row t owns the
//     words j = 4 i + q (dims 8 j .. 8 j + 7, in order, nibble n = dim 8 j +
//     n), adjacent in memory; rows of more than 128 dims are cut into planes
//     of 128;
//   values (A operand of V^T P, columns = tokens 2q, 2q + 1, 2q + 8, 2q + 9):
//     a 16-bit unit is four codes of one token, and a word is the same unit of
//     two adjacent tokens, so a code and its neighbour token's code lie 16 bits
//     apart.  Lane (r, q) owns words (pair, u, half): nibble n is dim 64 u + 32
//     (n >> 1) + 4 r + 2 half + (n & 1), which keeps every m16 tile of dims
//     inside one group of 32.  16-byte planes of [r][q][4 words].
#pragma once

#include "common.cuh"

namespace fa {
namespace kv4 {

constexpr int kTileTokens = 16;

__host__ __device__ constexpr int code_bytes(int d) { return kTileTokens * d / 2; }  // keys or values
__host__ __device__ constexpr int scale_bytes(int groups) { return kTileTokens * groups * 8; }
__host__ __device__ constexpr int tile_bytes(int d, int groups) {
  return 2 * code_bytes(d) + scale_bytes(groups);
}

// Byte offset of key word j of token t (inside the tile's key codes).
template <int kD>
__host__ __device__ constexpr int key_word(int t, int j) {
  constexpr int kPlaneDims = kD < 128 ? kD : 128;
  constexpr int kW = kPlaneDims / 32;  // words of a lane in a plane's row
  const int plane = j / (kPlaneDims / 8), jj = j % (kPlaneDims / 8);
  return plane * (kTileTokens * kPlaneDims / 2) + t * (kPlaneDims / 2) + ((jj % 4) * kW + jj / 4) * 4;
}
// Byte offset of the 16-bit value unit (u, r, half) of token t (inside the
// tile's value codes).
template <int kD>
__host__ __device__ constexpr int value_unit(int t, int u, int r, int half) {
  constexpr int kU = kD / 64;
  const int q = (t % 8) / 2, idx = ((t / 8) * kU + u) * 2 + half;
  return (idx / 4) * 512 + (r * 4 + q) * 16 + (idx % 4) * 4 + (t % 2) * 2;
}

// A pool of `slots` = num_blocks * block_size token slots, below 2^32, and
// fewer than 2^31 tiles (either would be larger than the GPU's memory).
struct Pool {
  uint8_t *data;
  uint32_t slots;
  int block_size, tiles_per_block, heads, tile_bytes;
  // x / tiles_per_block for x < 2^28, as (x * div_mul) >> div_shift
  uint32_t div_mul, div_shift;
  __device__ __forceinline__ uint8_t *tile(uint32_t block, int head, uint32_t tile_in_block) const {
    const uint32_t at = (block * heads + head) * tiles_per_block + tile_in_block;
    return data + static_cast<uint64_t>(at) * static_cast<uint32_t>(tile_bytes);
  }
};

}  // namespace kv4
}  // namespace fa
