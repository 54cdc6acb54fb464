// The 4-bit KV cache: tile layout and the arithmetic of its codes.
//
// [block][kv_head][2 (K, V)] tiles of Q4_TILE_BYTES: HY_BLOCK rows (tokens) of 64
// code bytes, then HY_BLOCK rows of 8 parameter bytes, four fp16: (scale, minimum)
// of dimensions 0-63, (scale, minimum) of dimensions 64-127.  K and V of one block
// and head are adjacent, so a decode work item fetches both with one bulk copy.
// Word i (32 bits, little endian) of a row holds dimensions 8i..8i+7: nibble j is
// dimension 8i + 2j and nibble 4 + j dimension 8i + 2j + 1, so that masking a
// shifted word with 0x000f000f leaves two neighbouring dimensions in the halves of
// a register.  A code c stands for scale * c + minimum.
//
// 64 dimensions share a scale: with 32 the parameters would be 16 bytes a row (80
// bytes instead of 72, and the cache is read at HBM speed), with 128 the step
// would follow the whole row's range.  The parameters are fp16 (11 significant
// bits: the minimum's rounding stays below a fiftieth of a step), so rows are
// clamped to +-Q4_LIMIT as they are written; codes are taken against the rounded
// parameters, which keeps the reconstruction within half a step of the input (plus
// the parameters' own rounding at the ends of the range).
#pragma once

#include "common.cuh"
#include <cuda_fp16.h>

#define Q4_ROW_BYTES   (HY_HEAD_DIM / 2)                 // codes of one row: 64
#define Q4_PARAM_BYTES 8                                  // parameters of one row
#define Q4_PARAM_OFF   (HY_BLOCK * Q4_ROW_BYTES)         // 1024
#define Q4_TILE_BYTES  (HY_BLOCK * (Q4_ROW_BYTES + Q4_PARAM_BYTES))   // 1152
#define Q4_LIMIT       32768.0f

// First byte of the tile of (block, kv head, K or V) in one layer.
HY_DEVICE size_t q4_tile(int blk, int head, int kv, int kv_heads) {
  return (((size_t)blk * kv_heads + head) * 2 + kv) * Q4_TILE_BYTES;
}

// (scale, minimum) as a half2: .x scale, .y minimum.
HY_DEVICE __half2 q4_as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
HY_DEVICE uint32_t q4_as_u32(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }

// The 8 values (dimensions 8i..8i+7, in order) of word i in fp32.  scale * code is
// exact (11 + 4 bits), so the sum is the only rounding.
HY_DEVICE void q4_values(uint32_t w, float scale, float low, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = fmaf((float)((w >> (4 * j)) & 15u), scale, low);
    x[2 * j + 1] = fmaf((float)((w >> (16 + 4 * j)) & 15u), scale, low);
  }
}
