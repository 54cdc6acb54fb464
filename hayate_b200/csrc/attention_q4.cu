// Varlen paged GQA attention over the 4-bit KV cache (layout: q4.cuh).
//
// Semantics as attention.cu: the j-th query token of sequence i sits at position
// prefix_i + j (prefix_i = seq_len_k_i - q_len_i) and attends to keys
// [0, prefix_i + j] of its own sequence (hayate/model/attention.py:52-64 with the
// masks of hayate/model/qwen.py:66-106); here a key or value is what its codes
// stand for, scale * code + minimum.
#include "attention.cuh"
#include "q4.cuh"

#include <math.h>

namespace {

// ------------------------------------------------------------------ scalar path
// One warp per (query token, query head), every key visited in order with a
// running maximum and sum: fp32 throughout, whatever T is.
template <typename T> HY_DEVICE void load4(const T* p, float (&f)[4]);
template <> HY_DEVICE void load4<float>(const float* p, float (&f)[4]) {
  const float4 u = *reinterpret_cast<const float4*>(p);
  f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
}
template <> HY_DEVICE void load4<__nv_bfloat16>(const __nv_bfloat16* p, float (&f)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u);
  f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
}
HY_DEVICE void store4(float* p, const float (&f)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
}
HY_DEVICE void store4(__nv_bfloat16* p, const float (&f)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
}

// This lane's 4 dimensions (4 lane .. 4 lane + 3) of row `off` of a tile.
HY_DEVICE void row4(const uint8_t* tile, int off, int lane, float (&f)[4]) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + off * Q4_ROW_BYTES + 4 * (lane >> 1));
  const uint32_t p = *reinterpret_cast<const uint32_t*>(tile + Q4_PARAM_OFF + off * Q4_PARAM_BYTES +
                                                        4 * (lane >> 4));
  const float2 sm = __half22float2(q4_as_half2(p));
  const uint32_t n = w >> (8 * (lane & 1));      // nibbles j, j + 1 and, 16 bits up, their partners
  f[0] = fmaf((float)(n & 15u), sm.x, sm.y);
  f[1] = fmaf((float)((n >> 16) & 15u), sm.x, sm.y);
  f[2] = fmaf((float)((n >> 4) & 15u), sm.x, sm.y);
  f[3] = fmaf((float)((n >> 20) & 15u), sm.x, sm.y);
}

template <typename T>
__global__ void __launch_bounds__(256) attn_q4_scalar_kernel(
    const T* __restrict__ q, T* __restrict__ out, int tokens, int q_heads, int kv_heads,
    const uint8_t* __restrict__ cache_layer, int num_blocks,
    const int32_t* __restrict__ block_tables, int bt_pitch,
    const int32_t* __restrict__ seq_bt_row, const int32_t* __restrict__ cu_q,
    const int32_t* __restrict__ seq_lens_k, int S, float scale, int32_t* err) {
  hy_grid_wait();
  hy_grid_trigger();
  const int lane = threadIdx.x & 31;
  const long total = (long)min(tokens, cu_q[S]) * q_heads;   // rows past the last sequence stay
  const long nwarps = (long)gridDim.x * (blockDim.x >> 5);
  for (long w = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < total; w += nwarps) {
    const int row = (int)(w / q_heads), hq = (int)(w % q_heads);
    const int g = hq / HY_GROUP;
    int lo = 0, hi = S;                     // seq = last i with cu_q[i] <= row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu_q[mid] <= row) lo = mid; else hi = mid;
    }
    const int seq = lo;
    const int prefix = seq_lens_k[seq] - (cu_q[seq + 1] - cu_q[seq]);
    const int key_end = prefix + (row - cu_q[seq]) + 1;
    if (prefix < 0 || (long)key_end > (long)bt_pitch * HY_BLOCK) {
      hy_flag(err, HY_ERR_BOUNDS);
      continue;
    }
    const int32_t* bt = block_tables + (size_t)(seq_bt_row ? seq_bt_row[seq] : seq) * bt_pitch;
    float qv[4];
    load4(q + ((size_t)row * q_heads + hq) * HY_HEAD_DIM + 4 * lane, qv);
    float m = -INFINITY, l = 0.f;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int key = 0; key < key_end; ++key) {
      const int blk = bt[key / HY_BLOCK];
      if (blk < 0 || blk >= num_blocks) { hy_flag(err, HY_ERR_BOUNDS); break; }
      const uint8_t* tile = cache_layer + q4_tile(blk, g, 0, kv_heads);
      float kv[4];
      row4(tile, key % HY_BLOCK, lane, kv);
      float s = qv[0] * kv[0] + qv[1] * kv[1] + qv[2] * kv[2] + qv[3] * kv[3];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      s *= scale;
      const float m_new = fmaxf(m, s);
      const float alpha = expf(m - m_new);
      const float p = expf(s - m_new);
      l = l * alpha + p;
      row4(tile + Q4_TILE_BYTES, key % HY_BLOCK, lane, kv);
#pragma unroll
      for (int d = 0; d < 4; ++d) acc[d] = acc[d] * alpha + p * kv[d];
      m = m_new;
    }
    const float inv = 1.f / l;
#pragma unroll
    for (int d = 0; d < 4; ++d) acc[d] *= inv;
    store4(out + ((size_t)row * q_heads + hq) * HY_HEAD_DIM + 4 * lane, acc);
  }
}

template <typename T>
cudaError_t launch_scalar(const void* q, void* out, int tokens, int q_heads, int kv_heads,
                          const uint8_t* cache_layer, int num_blocks,
                          const int32_t* block_tables, int bt_pitch, const int32_t* seq_bt_row,
                          const int32_t* cu_q, const int32_t* seq_lens_k, int S, float scale,
                          int32_t* err, cudaStream_t st) {
  const long blocks = ((long)tokens * q_heads + 7) / 8;
  return hy_launch(attn_q4_scalar_kernel<T>, dim3((int)(blocks < 148L * 32 ? blocks : 148L * 32)),
                   dim3(256), 0, st, static_cast<const T*>(q), static_cast<T*>(out), tokens,
                   q_heads, kv_heads, cache_layer, num_blocks, block_tables, bt_pitch, seq_bt_row,
                   cu_q, seq_lens_k, S, scale, err);
}

}  // namespace

cudaError_t hy_launch_attn_q4_scalar(int dtype, const void* q, void* out, int tokens, int q_heads,
                                     int kv_heads, const void* cache_layer, int num_blocks,
                                     const int32_t* block_tables, int bt_pitch,
                                     const int32_t* seq_bt_row, const int32_t* cu_q,
                                     const int32_t* seq_lens_k, int S, float scale, int32_t* err,
                                     cudaStream_t st) {
  const uint8_t* c = static_cast<const uint8_t*>(cache_layer);
  if (dtype == 0)
    return launch_scalar<__nv_bfloat16>(q, out, tokens, q_heads, kv_heads, c, num_blocks,
                                        block_tables, bt_pitch, seq_bt_row, cu_q, seq_lens_k, S,
                                        scale, err, st);
  return launch_scalar<float>(q, out, tokens, q_heads, kv_heads, c, num_blocks, block_tables,
                              bt_pitch, seq_bt_row, cu_q, seq_lens_k, S, scale, err, st);
}
