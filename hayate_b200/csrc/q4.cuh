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
// bits), so rows are clamped to +-Q4_LIMIT as they are written; codes are taken against
// the rounded parameters, which keeps the reconstruction within half a step of the input
// but for what their rounding cuts off at the ends of the range: up to 15 steps times
// 2^-11 at the top, and |minimum| 2^-11 at either end.  Where the range holds 0 the minimum
// is at most 15 steps, and that is a hundredth of a step; a half row that lies far from 0
// against its range loses accuracy to it (1000 to 1002: a step of 0.133 and an error of
// up to 0.25, half of fp16's spacing there).
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

// The nibbles at bits `at` (0, 4, 8 or 12) and 16 + at of w, two neighbouring dimensions,
// as floats: under the exponent of 2^23 a nibble n is 2^23 + n, exactly (a conversion
// instruction runs at a quarter of the rate).
HY_DEVICE float2 q4_nibbles(uint32_t w, int at) {
  return __fadd2_rn(make_float2(__uint_as_float(((w >> at) & 15u) | 0x4b000000u),
                                __uint_as_float(((w >> (16 + at)) & 15u) | 0x4b000000u)),
                    make_float2(-8388608.0f, -8388608.0f));
}

// The 8 values (dimensions 8i..8i+7, in order) of word i in fp32.  scale * code is
// exact (11 + 4 bits), so the sum is the only rounding.
HY_DEVICE void q4_values(uint32_t w, float scale, float low, float2 (&x)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    x[j] = __ffma2_rn(q4_nibbles(w, 4 * j), make_float2(scale, scale), make_float2(low, low));
}

// The values of a word's nibbles as fp16 pairs: x[j] = (nibble j, nibble 4 + j),
// scaled.  s2 and m2 hold the scale and minimum of the low halves' and the high
// halves' nibbles.  A nibble under the exponent of 1024 is the number 1024 + n (in
// bits 0-3) or 1024 + 16 n (in bits 4-7), from which n follows exactly; the only
// rounding is the last multiply-add's, to fp16 (2^-11 relative, an eighth of bf16's).
// The exponent trick for 4-bit codes is a published one: Kim, Henry, Fahim, Awadalla, "Who
// Says Elephants Can't Run: Bringing Large Scale MoE Models into Cloud Scale Production",
// 2022.
HY_DEVICE uint32_t q4_lop_or(uint32_t w, uint32_t mask) {
  uint32_t r;                                   // (w & mask) | 0x64006400
  asm("lop3.b32 %0, %1, %2, 0x64006400, 0xea;" : "=r"(r) : "r"(w), "r"(mask));
  return r;
}
HY_DEVICE void q4_expand(uint32_t w, __half2 s2, __half2 m2, uint32_t (&x)[4]) {
  const __half2 k1024 = q4_as_half2(0xe400e400u);      // -1024
  const __half2 k16th = q4_as_half2(0x2c002c00u);      // 1/16
  const __half2 k64 = q4_as_half2(0xd400d400u);        // -64
  const uint32_t w8 = w >> 8;
  const __half2 n0 = __hadd2(q4_as_half2(q4_lop_or(w, 0x000f000fu)), k1024);
  const __half2 n1 = __hfma2(q4_as_half2(q4_lop_or(w, 0x00f000f0u)), k16th, k64);
  const __half2 n2 = __hadd2(q4_as_half2(q4_lop_or(w8, 0x000f000fu)), k1024);
  const __half2 n3 = __hfma2(q4_as_half2(q4_lop_or(w8, 0x00f000f0u)), k16th, k64);
  x[0] = q4_as_u32(__hfma2(n0, s2, m2));
  x[1] = q4_as_u32(__hfma2(n1, s2, m2));
  x[2] = q4_as_u32(__hfma2(n2, s2, m2));
  x[3] = q4_as_u32(__hfma2(n3, s2, m2));
}

// A query row in fp16 is taken times 2^-e, e the exponent of its largest |element|
// (any bf16 row then fits fp16, and what falls below fp16's normal range is 2^-14 of
// the row's largest element); the score is multiplied by 2^e in fp32.
HY_DEVICE void q4_query_scale(float amax, float& down, float& up) {
  const int e = min(max((__float_as_int(amax) >> 23) & 255, 1), 253);
  const bool finite = amax < INFINITY;            // NaN and infinities pass unscaled
  down = finite ? __int_as_float((254 - e) << 23) : 1.0f;
  up = finite ? __int_as_float(e << 23) : 1.0f;
}
