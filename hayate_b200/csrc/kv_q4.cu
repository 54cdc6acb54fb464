// Writing the 4-bit KV cache and reading it back.
//
// Both are one pass over rows of 128 (token, K or V, head): 16 lanes per row, one
// 32-bit code word (8 dimensions) per lane, the 8 lanes of a half row agreeing on
// its scale and minimum by three shuffles.  They do what hy_kv_append and a gather
// of its cache do (hayate/model/attention.py:52-54 keeps the cache in the model
// dtype; the reference has no quantised one).
//
// Bound by memory: a bf16 row moves 256 + 72 bytes.
#include "q4.cuh"

namespace {

constexpr int Q4_THREADS = 256;
constexpr int Q4_LANES = HY_HEAD_DIM / 8;             // lanes per row
constexpr int Q4_ROWS = Q4_THREADS / Q4_LANES;        // rows per CTA pass
#ifndef HY_Q4_UNROLL
#define HY_Q4_UNROLL 4
#endif
constexpr int Q4_UNROLL = HY_Q4_UNROLL;               // rows in flight per lane

// 8 consecutive elements as loaded, and their values.
template <typename T> struct Raw8;
template <> struct Raw8<__nv_bfloat16> {
  uint4 a;
  HY_DEVICE void load(const __nv_bfloat16* p) { a = __ldg(reinterpret_cast<const uint4*>(p)); }
  HY_DEVICE void get(float (&f)[8]) const {
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
};
template <> struct Raw8<float> {
  float4 a, b;
  HY_DEVICE void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  HY_DEVICE void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};

HY_DEVICE void store8(__nv_bfloat16* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]),
                                            pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
HY_DEVICE void store8(float* p, const float (&f)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}

// Code word of this lane's 8 values and its half row's (scale, minimum); the 8
// lanes of a half row call it together (xor 1, 2, 4 stay inside it).  Every step is
// an IEEE fp32 operation, so the codes are the same whatever computes them.
HY_DEVICE uint32_t quantise8(float (&x)[8], __half2& par) {
  bool nan = false;
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    nan |= x[i] != x[i];
    x[i] = fminf(fmaxf(x[i], -Q4_LIMIT), Q4_LIMIT);
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  // a NaN anywhere in the half row: it reads back as NaN
  const unsigned votes = __ballot_sync(0xffffffffu, nan);
  if ((votes >> (threadIdx.x & 24)) & 0xffu) {
    par = __half2half2(__ushort_as_half(0x7fff));
    return 0u;
  }
  const __half scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  const __half low = __float2half_rn(lo);
  par = __halves2half2(scale, low);
  const float s = __half2float(scale), m = __half2float(low);
  const float inv = s > 0.f ? __fdiv_rn(1.0f, s) : 0.f;   // a constant half row: codes 0
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = rintf(__fmul_rn(__fsub_rn(x[i], m), inv));
    const uint32_t code = (uint32_t)fminf(fmaxf(c, 0.f), 15.f);
    w |= code << (4 * (i >> 1) + 16 * (i & 1));
  }
  return w;
}

template <typename T>
__global__ void __launch_bounds__(Q4_THREADS) kv_append_q4_kernel(
    const T* __restrict__ k, long ldk, const T* __restrict__ v, long ldv, int tokens,
    int kv_heads, const int32_t* __restrict__ slots, uint8_t* __restrict__ cache, int num_blocks,
    int32_t* err) {
  hy_grid_wait();
  hy_grid_trigger();
  const int grp = threadIdx.x / Q4_LANES, l = threadIdx.x % Q4_LANES;
  const int R = 2 * kv_heads;
  const int total = tokens * R, stride = (int)gridDim.x * Q4_ROWS;
  // every lane of a warp makes the same trips: the shuffles below need them all
  const int first = (int)blockIdx.x * Q4_ROWS;
  for (int base = first; base < total; base += stride * Q4_UNROLL) {
    Raw8<T> raw[Q4_UNROLL];
    uint8_t* dst[Q4_UNROLL];                        // the row's codes
    int par_at[Q4_UNROLL];                          // its parameters, from there
#pragma unroll
    for (int u = 0; u < Q4_UNROLL; ++u) {
      const int i = base + u * stride + grp;
      dst[u] = nullptr;
      if (i < total) {
        const int t = i / R, r = i - t * R;
        const int kv = r >= kv_heads, h = kv ? r - kv_heads : r;
        raw[u].load((kv ? v + (size_t)t * ldv : k + (size_t)t * ldk) + h * HY_HEAD_DIM + 8 * l);
        const int slot = slots[t];
        const int blk = slot / HY_BLOCK, off = slot % HY_BLOCK;
        if (slot >= 0 && blk >= num_blocks) hy_flag(err, HY_ERR_BOUNDS);
        else if (slot >= 0) {
          dst[u] = cache + q4_tile(blk, h, kv, kv_heads) + off * Q4_ROW_BYTES;
          par_at[u] = Q4_PARAM_OFF - off * (Q4_ROW_BYTES - Q4_PARAM_BYTES);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < Q4_UNROLL; ++u) {
      if (__any_sync(0xffffffffu, dst[u] != nullptr)) {
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (dst[u]) raw[u].get(x);
        __half2 par;
        const uint32_t w = quantise8(x, par);
        if (dst[u]) {
          reinterpret_cast<uint32_t*>(dst[u])[l] = w;
          if ((l & 7) == 0)
            *reinterpret_cast<uint32_t*>(dst[u] + par_at[u] + 4 * (l >> 3)) = q4_as_u32(par);
        }
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(Q4_THREADS) kv_read_q4_kernel(
    const uint8_t* __restrict__ cache, int num_blocks, int kv_heads,
    const int32_t* __restrict__ slots, int tokens, T* __restrict__ k_out, T* __restrict__ v_out,
    int32_t* err) {
  hy_grid_wait();
  hy_grid_trigger();
  const int grp = threadIdx.x / Q4_LANES, l = threadIdx.x % Q4_LANES;
  const int R = 2 * kv_heads;
  const int total = tokens * R, stride = (int)gridDim.x * Q4_ROWS;
  for (int base = (int)blockIdx.x * Q4_ROWS + grp; base < total; base += stride * Q4_UNROLL) {
    uint32_t w[Q4_UNROLL], par[Q4_UNROLL];
    T* dst[Q4_UNROLL];
#pragma unroll
    for (int u = 0; u < Q4_UNROLL; ++u) {
      const int i = base + u * stride;
      dst[u] = nullptr;
      w[u] = par[u] = 0u;                           // scale = minimum = 0: a row of zeros
      if (i < total) {
        const int t = i / R, r = i - t * R;
        const int kv = r >= kv_heads, h = kv ? r - kv_heads : r;
        dst[u] = (kv ? v_out : k_out) + ((size_t)t * kv_heads + h) * HY_HEAD_DIM + 8 * l;
        const int slot = slots[t];
        const int blk = slot / HY_BLOCK, off = slot % HY_BLOCK;
        if (slot >= 0 && blk >= num_blocks) hy_flag(err, HY_ERR_BOUNDS);
        else if (slot >= 0) {
          const uint8_t* tile = cache + q4_tile(blk, h, kv, kv_heads);
          w[u] = __ldg(reinterpret_cast<const uint32_t*>(tile + off * Q4_ROW_BYTES) + l);
          par[u] = __ldg(reinterpret_cast<const uint32_t*>(tile + Q4_PARAM_OFF + off * Q4_PARAM_BYTES) +
                         (l >> 3));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < Q4_UNROLL; ++u)
      if (dst[u]) {
        const float2 p = __half22float2(q4_as_half2(par[u]));
        float x[8];
        q4_values(w[u], p.x, p.y, x);
        store8(dst[u], x);
      }
  }
}

// CTAs for `rows` rows: one pass of Q4_ROWS x Q4_UNROLL rows each, at most 8
// resident CTAs on each of 148 SMs (the kernels stride over the rest).
int q4_grid(long rows) {
  const long n = (rows + Q4_ROWS - 1) / Q4_ROWS;
  return (int)(n < 148 * 8 ? n : 148 * 8);
}

// The kernels count rows in 32 bits: longer calls go in slices of this many rows.
constexpr long Q4_SLICE_ROWS = 1L << 29;

}  // namespace

template <typename T>
static cudaError_t append_q4(const T* k, long ldk, const T* v, long ldv, int T_tokens, int kv_heads,
                             const int32_t* slots, uint8_t* cache, int num_blocks, int32_t* err,
                             cudaStream_t st) {
  const int step = (int)(Q4_SLICE_ROWS / (2 * kv_heads));
  for (int t = 0; t < T_tokens; t += step) {
    const int n = T_tokens - t < step ? T_tokens - t : step;
    const cudaError_t e = hy_launch(kv_append_q4_kernel<T>, dim3(q4_grid(2L * kv_heads * n)),
                                    dim3(Q4_THREADS), 0, st, k + (size_t)t * ldk, ldk,
                                    v + (size_t)t * ldv, ldv, n, kv_heads, slots + t, cache,
                                    num_blocks, err);
    if (e != cudaSuccess || n < step) return e;
  }
  return cudaSuccess;
}

cudaError_t hy_launch_kv_append_q4(int dtype, const void* k, long ldk, const void* v, long ldv,
                                   int T_tokens, int kv_heads, const int32_t* slots, void* cache,
                                   int num_blocks, int32_t* err, cudaStream_t st) {
  using B = __nv_bfloat16;
  if (dtype == 0)
    return append_q4((const B*)k, ldk, (const B*)v, ldv, T_tokens, kv_heads, slots,
                     (uint8_t*)cache, num_blocks, err, st);
  return append_q4((const float*)k, ldk, (const float*)v, ldv, T_tokens, kv_heads, slots,
                   (uint8_t*)cache, num_blocks, err, st);
}

template <typename T>
static cudaError_t read_q4(const uint8_t* cache, int num_blocks, int kv_heads,
                           const int32_t* slots, int T_tokens, T* k_out, T* v_out, int32_t* err,
                           cudaStream_t st) {
  const int step = (int)(Q4_SLICE_ROWS / (2 * kv_heads));
  for (int t = 0; t < T_tokens; t += step) {
    const int n = T_tokens - t < step ? T_tokens - t : step;
    const size_t at = (size_t)t * kv_heads * HY_HEAD_DIM;
    const cudaError_t e = hy_launch(kv_read_q4_kernel<T>, dim3(q4_grid(2L * kv_heads * n)),
                                    dim3(Q4_THREADS), 0, st, cache, num_blocks, kv_heads,
                                    slots + t, n, k_out + at, v_out + at, err);
    if (e != cudaSuccess || n < step) return e;
  }
  return cudaSuccess;
}

cudaError_t hy_launch_kv_read_q4(int dtype, const void* cache, int num_blocks, int kv_heads,
                                 const int32_t* slots, int T_tokens, void* k_out, void* v_out,
                                 int32_t* err, cudaStream_t st) {
  using B = __nv_bfloat16;
  if (dtype == 0)
    return read_q4((const uint8_t*)cache, num_blocks, kv_heads, slots, T_tokens, (B*)k_out,
                   (B*)v_out, err, st);
  return read_q4((const uint8_t*)cache, num_blocks, kv_heads, slots, T_tokens, (float*)k_out,
                 (float*)v_out, err, st);
}
