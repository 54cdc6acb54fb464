// Writing the 4-bit KV cache and reading it back.
//
// Both are one pass over rows of 128 (token, K or V, head): 8 lanes per row, 16
// dimensions (two code words) per lane, the 4 lanes of a half row agreeing on its
// minimum and maximum by two exchanges.  They do what hy_kv_append and a gather of its
// cache do (hayate/model/attention.py:52-54 keeps the cache in the model dtype; the
// reference has no quantised one).
//
// Bound by memory (a bf16 row moves 256 + 72 bytes: 8192 tokens of 8 heads are written in
// 11.8 us, 3.6 TB/s, from inputs in HBM, in 9.5 where the call before left them in L2, and
// 40001 tokens read back in 48.6 us, 4.3 TB/s, where filling the outputs alone takes 45.8)
// as long as the instructions per element stay few: the codes are rounded and collected by
// additions instead of conversions (which run at a quarter of the rate), read back by
// masks, and a thread's row of the token is found once, not per row.
#include "q4.cuh"

namespace {

constexpr int Q4_THREADS = 256;
constexpr int Q4_LANES = HY_HEAD_DIM / 16;            // lanes per row
constexpr int Q4_ROWS = Q4_THREADS / Q4_LANES;        // rows per CTA pass
// rows in flight per lane (8192 tokens of 8 heads written / read, from HBM: 12.7 / 12.5 us
// with 1, 11.8 / 10.8 with 2, 13.8 / 12.0 with 4)
constexpr int Q4_UNROLL = 2;

// min and max that are NaN if either operand is
HY_DEVICE float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
HY_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 16 consecutive elements as loaded; their values; and over the half row (lanes xor 1,
// 2) the minimum and maximum, NaN if any element is.
template <typename T> struct Raw16;
template <> struct Raw16<__nv_bfloat16> {
  uint4 a[2];
  HY_DEVICE void load(const __nv_bfloat16* p) {
    a[0] = __ldg(reinterpret_cast<const uint4*>(p));
    a[1] = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  }
  HY_DEVICE void get(float (&f)[16]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t u[4] = {a[h].x, a[h].y, a[h].z, a[h].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[8 * h + 2 * i] = __uint_as_float(u[i] << 16);
        f[8 * h + 2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    }
  }
  HY_DEVICE void range(const float (&)[16], float& lo, float& hi) const {
    const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(a);
    __nv_bfloat162 mn = v[0], mx = v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      mn = __hmin2_nan(mn, v[i]);
      mx = __hmax2_nan(mx, v[i]);
    }
    // (min, -max) of both halves of the registers, exchanged together
    const __nv_bfloat162 neg = __hneg2(mx);
    __nv_bfloat162 e = __hmin2_nan(__halves2bfloat162(__low2bfloat16(mn), __low2bfloat16(neg)),
                                   __halves2bfloat162(__high2bfloat16(mn), __high2bfloat16(neg)));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) e = __hmin2_nan(e, __shfl_xor_sync(0xffffffffu, e, o));
    lo = __low2float(e);
    hi = -__high2float(e);
  }
};
template <> struct Raw16<float> {
  float4 a[4];
  HY_DEVICE void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = __ldg(reinterpret_cast<const float4*>(p) + i);
  }
  HY_DEVICE void get(float (&f)[16]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[4 * i] = a[i].x;
      f[4 * i + 1] = a[i].y;
      f[4 * i + 2] = a[i].z;
      f[4 * i + 3] = a[i].w;
    }
  }
  HY_DEVICE void range(const float (&x)[16], float& lo, float& hi) const {
    lo = hi = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) {
      lo = min_nan(lo, x[i]);
      hi = max_nan(hi, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
  }
};

HY_DEVICE void store16(__nv_bfloat16* p, const float (&f)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    reinterpret_cast<uint4*>(p)[h] =
        make_uint4(pack_bf16(f[8 * h], f[8 * h + 1]), pack_bf16(f[8 * h + 2], f[8 * h + 3]),
                   pack_bf16(f[8 * h + 4], f[8 * h + 5]), pack_bf16(f[8 * h + 6], f[8 * h + 7]));
}
HY_DEVICE void store16(float* p, const float (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    reinterpret_cast<float4*>(p)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
}

// Code words of this lane's 16 values and its half row's (scale, minimum).  Every step
// is an IEEE fp32 operation, so the codes are the same whatever computes them.  The
// clamp of the values to +-Q4_LIMIT is the clamp of their range: beyond it a code is 0
// or 15 either way.
template <typename T>
HY_DEVICE uint2 quantise16(const Raw16<T>& raw, __half2& par) {
  float x[16], lo, hi;
  raw.get(x);
  raw.range(x, lo, hi);
  if (lo != lo) {                                       // a NaN somewhere: it reads back as NaN
    par = __half2half2(__ushort_as_half(0x7fff));
    return make_uint2(0u, 0u);
  }
  lo = fminf(fmaxf(lo, -Q4_LIMIT), Q4_LIMIT);
  hi = fminf(fmaxf(hi, -Q4_LIMIT), Q4_LIMIT);
  const __half scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  const __half low = __float2half_rn(lo);
  par = __halves2half2(scale, low);
  const float s = __half2float(scale), m = __half2float(low);
  const float inv = s > 0.f ? __fdiv_rn(1.0f, s) : 0.f; // a constant half row: codes 0
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // c + 2^23 rounds c to an integer, half to even, in the low bits; the words collect
    // 16 u + u' from nibble 7 down, and the exponents' multiples are taken off at the end
#pragma unroll
    for (int n = 7; n >= 0; --n) {
      const int i = 8 * h + (n < 4 ? 2 * n : 2 * (n - 4) + 1);
      const float c = fminf(fmaxf(__fmul_rn(__fsub_rn(x[i], m), inv), 0.f), 15.f);
      w[h] = w[h] * 16u + __float_as_uint(__fadd_rn(c, 8388608.0f));
    }
    w[h] -= 0x4b000000u;       // times 1 + 16 + .. + 16^7, of which all but 1 and 16 leave 32 bits
    w[h] -= 0xb0000000u;       // 16 x 0x4b000000
  }
  return make_uint2(w[0], w[1]);
}

// Rows of a CTA pass: 8 lanes each, `per` rows of a token (all its 2 kv_heads rows, or
// 32 at a time), as many tokens as fit.  With more than a pass per CTA, the passes in
// flight take neighbouring tokens, whose parameters share sectors (8192 tokens of 8
// heads, in L2: write 10.9 -> 9.8 us, read 10.7 -> 9.8); a short call spreads over the CTAs.
struct RowMap {
  int per, tokens, t, r;                                // this thread's token of the pass and row
  int first, near, stride;                              // the CTA's first token, from pass to pass in
                                                        // flight, from turn to turn
  HY_DEVICE RowMap(int kv_heads, int total) {
    const int row = threadIdx.x / Q4_LANES;
    per = min(2 * kv_heads, Q4_ROWS);
    tokens = Q4_ROWS / per;
    t = row / per;
    r = row - t * per;
    if (t >= tokens) r = 1 << 30;                       // a spare row of the pass
    const int all = (int)gridDim.x * tokens;
    const bool many = total > all;
    first = (int)blockIdx.x * tokens * (many ? Q4_UNROLL : 1);
    near = many ? tokens : all;
    stride = all * Q4_UNROLL;
  }
};

template <typename T>
__global__ void __launch_bounds__(Q4_THREADS) kv_append_q4_kernel(
    const T* __restrict__ k, long ldk, const T* __restrict__ v, long ldv, int tokens,
    int kv_heads, const int32_t* __restrict__ slots, uint8_t* __restrict__ cache, int num_blocks,
    int32_t* err) {
  hy_grid_wait();
  hy_grid_trigger();
  const int l = threadIdx.x % Q4_LANES, R = 2 * kv_heads;
  const RowMap map(kv_heads, tokens);
  // every lane of a warp makes the same trips: the exchanges need them all
  for (int rb = 0; rb < R; rb += map.per)
    for (int tb = map.first; tb < tokens; tb += map.stride) {
      const int r = rb + map.r, kv = r >= kv_heads, h = kv ? r - kv_heads : r;
      Raw16<T> raw[Q4_UNROLL];
      int slot[Q4_UNROLL];
#pragma unroll
      for (int u = 0; u < Q4_UNROLL; ++u) {
        const int t = tb + u * map.near + map.t;
        slot[u] = -1;
        if (r < R && t < tokens) {
          raw[u].load((kv ? v + (size_t)t * ldv : k + (size_t)t * ldk) + h * HY_HEAD_DIM + 16 * l);
          slot[u] = slots[t];
        } else {
          raw[u] = {};
        }
      }
#pragma unroll
      for (int u = 0; u < Q4_UNROLL; ++u) {
        __half2 par;
        const uint2 w = quantise16(raw[u], par);
        const uint32_t other = __shfl_xor_sync(0xffffffffu, q4_as_u32(par), Q4_LANES / 2);
        if (slot[u] < 0) continue;
        const int blk = slot[u] / HY_BLOCK, off = slot[u] % HY_BLOCK;
        if (blk >= num_blocks) {
          hy_flag(err, HY_ERR_BOUNDS);
          continue;
        }
        uint8_t* tile = cache + q4_tile(blk, h, kv, kv_heads);
        reinterpret_cast<uint2*>(tile + off * Q4_ROW_BYTES)[l] = w;
        if (l == 0)
          *reinterpret_cast<uint2*>(tile + Q4_PARAM_OFF + off * Q4_PARAM_BYTES) =
              make_uint2(q4_as_u32(par), other);
      }
    }
}

// The 8 values of word i (dimensions 8i.., in order) with the scale times 2^0, 2^-4, ..
// 2^-16: nibbles 0-4 are taken where they stand, at 16^j times their code, nibbles 5-7
// after one shift.  The products are exact, so the sum is the only rounding.
HY_DEVICE void read_word(uint32_t w, const float (&s)[5], float low, float* x) {
  const uint32_t w12 = w >> 12;
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const int at = n < 5 ? n : n - 3;                   // nibble position in w or w12
    const float c = __uint_as_float(((n < 5 ? w : w12) & (15u << (4 * at))) | 0x4b000000u) - 8388608.0f;
    x[n < 4 ? 2 * n : 2 * (n - 4) + 1] = fmaf(c, s[at], low);
  }
}

template <typename T>
__global__ void __launch_bounds__(Q4_THREADS) kv_read_q4_kernel(
    const uint8_t* __restrict__ cache, int num_blocks, int kv_heads,
    const int32_t* __restrict__ slots, int tokens, T* __restrict__ k_out, T* __restrict__ v_out,
    int32_t* err) {
  hy_grid_wait();
  hy_grid_trigger();
  const int l = threadIdx.x % Q4_LANES, R = 2 * kv_heads;
  const RowMap map(kv_heads, tokens);
  for (int rb = 0; rb < R; rb += map.per) {
    const int r = rb + map.r, kv = r >= kv_heads, h = kv ? r - kv_heads : r;
    if (r >= R) continue;
    T* out = (kv ? v_out : k_out) + h * HY_HEAD_DIM + 16 * l;
    for (int tb = map.first + map.t; tb < tokens; tb += map.stride) {
      uint2 w[Q4_UNROLL];
      uint32_t par[Q4_UNROLL];
#pragma unroll
      for (int u = 0; u < Q4_UNROLL; ++u) {
        const int t = tb + u * map.near;
        w[u] = make_uint2(0u, 0u);
        par[u] = 0u;                                    // scale = minimum = 0: a row of zeros
        const int slot = t < tokens ? slots[t] : -1;
        const int blk = slot / HY_BLOCK, off = slot % HY_BLOCK;
        if (slot >= 0 && blk >= num_blocks) hy_flag(err, HY_ERR_BOUNDS);
        else if (slot >= 0) {
          const uint8_t* tile = cache + q4_tile(blk, h, kv, kv_heads);
          w[u] = __ldg(reinterpret_cast<const uint2*>(tile + off * Q4_ROW_BYTES) + l);
          par[u] = __ldg(reinterpret_cast<const uint32_t*>(tile + Q4_PARAM_OFF + off * Q4_PARAM_BYTES) +
                         l / (Q4_LANES / 2));
        }
      }
#pragma unroll
      for (int u = 0; u < Q4_UNROLL; ++u) {
        const int t = tb + u * map.near;
        if (t < tokens) {
          const float2 p = __half22float2(q4_as_half2(par[u]));
          const float s[5] = {p.x, p.x * 0x1p-4f, p.x * 0x1p-8f, p.x * 0x1p-12f, p.x * 0x1p-16f};
          float x[16];
          read_word(w[u].x, s, p.y, x);
          read_word(w[u].y, s, p.y, x + 8);
          store16(out + (size_t)t * kv_heads * HY_HEAD_DIM, x);
        }
      }
    }
  }
}

// CTAs for `tokens` tokens: one pass each, at most 8 resident CTAs on each of 148 SMs
// (the kernels stride over the rest).
int q4_grid(int tokens, int kv_heads) {
  const int per = 2 * kv_heads < Q4_ROWS ? 2 * kv_heads : Q4_ROWS, pass = Q4_ROWS / per;
  const long n = ((long)tokens + pass - 1) / pass;
  return (int)(n < 148 * 8 ? n : 148 * 8);
}

// The kernels count tokens in 32 bits, strides past the end included: longer calls go in
// slices of this many.
constexpr int Q4_SLICE = 1 << 28;

}  // namespace

template <typename T>
static cudaError_t append_q4(const T* k, long ldk, const T* v, long ldv, int T_tokens, int kv_heads,
                             const int32_t* slots, uint8_t* cache, int num_blocks, int32_t* err,
                             cudaStream_t st) {
  for (long t = 0; t < T_tokens; t += Q4_SLICE) {
    const int n = T_tokens - t < Q4_SLICE ? (int)(T_tokens - t) : Q4_SLICE;
    const cudaError_t e = hy_launch(kv_append_q4_kernel<T>, dim3(q4_grid(n, kv_heads)),
                                    dim3(Q4_THREADS), 0, st, k + (size_t)t * ldk, ldk,
                                    v + (size_t)t * ldv, ldv, n, kv_heads, slots + t, cache,
                                    num_blocks, err);
    if (e != cudaSuccess) return e;
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
  for (long t = 0; t < T_tokens; t += Q4_SLICE) {
    const int n = T_tokens - t < Q4_SLICE ? (int)(T_tokens - t) : Q4_SLICE;
    const size_t at = (size_t)t * kv_heads * HY_HEAD_DIM;
    const cudaError_t e = hy_launch(kv_read_q4_kernel<T>, dim3(q4_grid(n, kv_heads)),
                                    dim3(Q4_THREADS), 0, st, cache, num_blocks, kv_heads,
                                    slots + t, n, k_out + at, v_out + at, err);
    if (e != cudaSuccess) return e;
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
