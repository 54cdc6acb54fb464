// Varlen paged GQA attention over the 4-bit KV cache (layout: q4.cuh).
//
// Semantics as attention.cu: the j-th query token of sequence i sits at position
// prefix_i + j (prefix_i = seq_len_k_i - q_len_i) and attends to keys
// [0, prefix_i + j] of its own sequence (hayate/model/attention.py:52-64 with the
// masks of hayate/model/qwen.py:66-106); here a key or value is what its codes
// stand for, scale * code + minimum.
//
// bf16 runs the work items of hy_attention_plan (attention.cu) on the tensor cores.
// Decode items (one query token): CTAs take 8 consecutive items at a time, two of
// their 16 warps per item; each warp streams its blocks (2304 bytes: K and V of one
// block and head are adjacent) through its own ring of bulk copies, expands the
// codes to fp16 in registers, in the operand layout of mma.sync, and keeps a running
// maximum and sum.  The CTA merges its warps' partials in shared memory, so that a
// sequence split over many items leaves one partial per 8 items in the workspace;
// the CTA that finishes a (sequence, head) last joins those.
// fp32 runs a scalar kernel.
#include "attention.cuh"
#include "q4.cuh"

#include <math.h>

namespace {

constexpr int NW = 16;                                    // warps per CTA
constexpr int NT = NW * 32;
constexpr int CHUNK = NW / 2;                             // decode items a CTA takes at a time
static_assert(CHUNK == HY_PLAN_WARPS, "a per-CTA decode pair's items fit one chunk");
#ifndef HY_Q4_STAGES
#define HY_Q4_STAGES 4
#endif
constexpr int NS = HY_Q4_STAGES;                          // blocks in flight per warp
constexpr int BLK_BYTES = 2 * Q4_TILE_BYTES;              // K and V tile of one block and head
constexpr int RING_BYTES = NS * BLK_BYTES;
constexpr int PART_FLOATS = HY_GROUP * HY_HEAD_DIM + 2 * HY_GROUP;   // O [4][128], then (m, l) [4]
constexpr int DEC_SMEM = NW * (RING_BYTES + PART_FLOATS * 4);
constexpr float RESCALE_LOG2 = 8.0f;                      // see decode_range

struct Args {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const uint8_t* cache;   // this layer's tiles
  int q_heads, kv_heads, num_blocks, layer;
  const int32_t* block_tables;
  int bt_pitch;
  const int32_t* seq_bt_row;
  const int32_t* cu_q;
  const int32_t* seq_lens_k;
  float scale_log2;
  int32_t* err;
};

struct Shared {
  uint64_t bar[NW][NS];
  int chunk;              // the CTA's next chunk of decode items
  int last;               // bit j: this CTA finished pair j of its two open ones
};

// Row of the score matrix S^T (row r or r + 8 of the 16-key block) -> key of the
// block.  Any order of the 16 keys is right as long as K's rows, the weights and V
// agree; this one puts the four keys that lane (r, c) takes from V, and the two
// neighbouring rows it takes from K, in different halves of the 32 shared-memory
// banks (a key's 64 bytes of codes are half of them).
HY_DEVICE int key_of(int c, int e, int h) {               // row 2 c + e + 8 h, c < 4
  return ((c ^ e) & 1) | (e << 1) | (h << 2) | ((c >> 1) << 3);
}

// One warp: attention of query token `tok`, KV head g (4 query heads) over key
// blocks [lo, hi) of a sequence of kv_len keys.  Scores are computed transposed,
// S^T = K Q^T (16 keys x 8 columns, 4 of them heads), and so is the output, O^T = V^T
// P^T: the codes then fill the 16-row operand of mma.sync, where the 4 heads
// alone would leave three quarters of it empty, at half the instructions.
// On return lane (r, c) = (lane / 4, lane % 4) with c < 2 holds, for heads
// 2c + k (k = 0, 1), the unnormalised output at dimensions 8 r + i (+64) as
// o[i / 2 + 4 (i % 2)][k (+2)], and m[k], l[k]: the running maximum (log2 units) and
// this lane's part of the sum (l sums over the 8 lanes of equal c).
// The maximum is only raised when a score exceeds it by more than 2^8 (weights stay
// far below fp16's 65504), so that most blocks need no exchange between lanes.
// Returns false if a wait ran out.
__device__ bool decode_range(const Args& a, uint8_t* ring, uint64_t* bars, uint32_t& phase,
                             const int32_t* bt, int tok, int g, int lo, int hi, int kv_len,
                             float (&o)[8][4], float (&m)[2], float (&l)[2]) {
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int n = hi - lo;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  m[0] = m[1] = -INFINITY;
  l[0] = l[1] = 0.f;
  if (n <= 0) return true;

  // block ids 32 at a time, one per lane, the next 32 loaded ahead
  auto id_at = [&](int j) {
    const int b = lo + j;
    return j < n && b < a.bt_pitch ? __ldg(bt + b) : -1;
  };
  int ids = id_at(lane), ids_next = id_at(32 + lane);
  auto issue = [&](int j) {                               // the whole warp; j in issue order
    if (j > 0 && (j & 31) == 0) {
      ids = ids_next;
      ids_next = id_at(j + 32 + lane);
    }
    int blk = __shfl_sync(0xffffffffu, ids, j & 31);
    if (lane == 0) {
      if (blk < 0 || blk >= a.num_blocks) {
        hy_flag(a.err, HY_ERR_BOUNDS);
        blk = 0;
      }
      const int s = j % NS;
      fence_proxy_async();
      mbar_arrive_expect_tx(&bars[s], BLK_BYTES);
      bulk_load(ring + s * BLK_BYTES, a.cache + q4_tile(blk, g, 0, a.kv_heads), BLK_BYTES,
                &bars[s]);
    }
  };
  for (int j = 0; j < NS && j < n; ++j) issue(j);

  // Q: lane (r, c) holds head r's dimensions 32 c .. 32 c + 31 (rows 4-7: zero)
  uint32_t qb[4][4];
  float mult[2];
  {
    float x[32], amax = 0.f, down, up;
    const __nv_bfloat16* qp = a.q + ((size_t)tok * a.q_heads + g * HY_GROUP + r) * HY_HEAD_DIM + 32 * c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 u = r < HY_GROUP ? *reinterpret_cast<const uint4*>(qp + 8 * i) : make_uint4(0, 0, 0, 0);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
        x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(x[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    q4_query_scale(amax, down, up);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        qb[i][j] = q4_as_u32(__floats2half2_rn(x[8 * i + 2 * j] * down, x[8 * i + 2 * j + 1] * down));
    mult[0] = a.scale_log2 * __shfl_sync(0xffffffffu, up, 8 * c);        // head 2 c: lanes of row 2 c
    mult[1] = a.scale_log2 * __shfl_sync(0xffffffffu, up, 8 * c + 4);
  }

  const int keyA = key_of(r >> 1, r & 1, 0), keyB = keyA | 4;            // this lane's score rows
  bool ok = true;
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const int s = i % NS;
    const bool w_ok = mbar_wait(&bars[s], (phase >> s) & 1u, a.err);
    if (__any_sync(0xffffffffu, !w_ok)) { ok = false; break; }
    phase ^= 1u << s;
    const uint8_t* kt = ring + s * BLK_BYTES;
    const uint8_t* vt = kt + Q4_TILE_BYTES;

    // S^T = K Q^T
    float sc[4] = {0.f, 0.f, 0.f, 0.f};
    {
      const uint4 wa = *reinterpret_cast<const uint4*>(kt + keyA * Q4_ROW_BYTES + 16 * c);
      const uint4 wb = *reinterpret_cast<const uint4*>(kt + keyB * Q4_ROW_BYTES + 16 * c);
      const __half2 pa = *reinterpret_cast<const __half2*>(kt + Q4_PARAM_OFF + keyA * Q4_PARAM_BYTES + 4 * (c >> 1));
      const __half2 pb = *reinterpret_cast<const __half2*>(kt + Q4_PARAM_OFF + keyB * Q4_PARAM_BYTES + 4 * (c >> 1));
      const __half2 sa = __low2half2(pa), ma = __high2half2(pa);
      const __half2 sb = __low2half2(pb), mb = __high2half2(pb);
      const uint32_t ua[4] = {wa.x, wa.y, wa.z, wa.w}, ub[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t xa[4], xb[4];
        q4_expand(ua[w], sa, ma, xa);
        q4_expand(ub[w], sb, mb, xb);
        mma_f16_16816(sc, xa[0], xb[0], xa[1], xb[1], qb[w][0], qb[w][1]);
        mma_f16_16816(sc, xa[2], xb[2], xa[3], xb[3], qb[w][2], qb[w][3]);
      }
    }
    const int kbase = (lo + i) * HY_BLOCK, left = kv_len - kbase;
    const bool tail = left < HY_BLOCK;                    // only the last block is partial
    float x[4] = {sc[0] * mult[0], sc[1] * mult[1], sc[2] * mult[0], sc[3] * mult[1]};
    if (tail) {
      if (keyA >= left) x[0] = x[1] = -INFINITY;
      if (keyB >= left) x[2] = x[3] = -INFINITY;
    }
    float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
    const bool grow = mx[0] > m[0] + RESCALE_LOG2 || mx[1] > m[1] + RESCALE_LOG2;
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], d));
        const float m_new = fmaxf(m[k], mx[k]);
        const float alpha = m_new == -INFINITY ? 1.f : ex2_ftz(m[k] - m_new);
        m[k] = m_new;
        l[k] *= alpha;
#pragma unroll
        for (int j = 0; j < 8; ++j) { o[j][k] *= alpha; o[j][2 + k] *= alpha; }
      }
    }
    const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
    x[0] = ex2_ftz(x[0] - m0);
    x[1] = ex2_ftz(x[1] - m1);
    x[2] = ex2_ftz(x[2] - m0);
    x[3] = ex2_ftz(x[3] - m1);
    l[0] += x[0] + x[2];
    l[1] += x[1] + x[3];
    // P^T as the 16 x 8 operand: weights in fp16 (2^-11; their sum l stays fp32)
    const uint32_t b0 = movmatrix_trans(q4_as_u32(__floats2half2_rn(x[0], x[1])));
    const uint32_t b1 = movmatrix_trans(q4_as_u32(__floats2half2_rn(x[2], x[3])));

    // O^T += V^T P^T: words r and 8 + r (dimensions 8 r .. and 64 + 8 r ..) of four keys
    uint32_t xv[2][2][4];                                 // [half of the keys][low, high nibbles]
#pragma unroll
    for (int half = 0; half < 2; ++half) {                // dimensions 0-63, then 64-127: rows r, r + 8
      uint32_t y[2][2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k0 = key_of(c, 0, h), k1 = key_of(c, 1, h);
        const uint32_t w0 = *reinterpret_cast<const uint32_t*>(vt + k0 * Q4_ROW_BYTES + 32 * half + 4 * r);
        const uint32_t w1 = *reinterpret_cast<const uint32_t*>(vt + k1 * Q4_ROW_BYTES + 32 * half + 4 * r);
        uint32_t p0 = *reinterpret_cast<const uint32_t*>(vt + Q4_PARAM_OFF + k0 * Q4_PARAM_BYTES + 4 * half);
        uint32_t p1 = *reinterpret_cast<const uint32_t*>(vt + Q4_PARAM_OFF + k1 * Q4_PARAM_BYTES + 4 * half);
        if (tail) {                                       // rows past the end hold anything
          if (k0 >= left) p0 = 0u;
          if (k1 >= left) p1 = 0u;
        }
        const __half2 s2 = q4_as_half2(__byte_perm(p0, p1, 0x5410));
        const __half2 m2 = q4_as_half2(__byte_perm(p0, p1, 0x7632));
        q4_expand(__byte_perm(w0, w1, 0x5410), s2, m2, y[h][0]);
        q4_expand(__byte_perm(w0, w1, 0x7632), s2, m2, y[h][1]);
      }
      if (half == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j) xv[h][e][j] = y[h][e][j];
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_f16_16816(o[4 * e + j], xv[0][e][j], y[0][e][j], xv[1][e][j], y[1][e][j], b0, b1);
      }
    }
    __syncwarp();                                         // the stage is read
    if (i + NS < n) issue(i + NS);
  }
  if (!ok) {                                              // copies in flight land before the CTA exits
    for (int s = 0; s < NS; ++s) mbar_wait(&bars[s], (phase >> s) & 1u, nullptr);
    return false;
  }
  return true;
}

// The CTA runs decode items [i0, i0 + cnt), cnt <= CHUNK: warp w takes half w % 2
// of item w / 2's blocks; then thread t merges head t / 128, dimension t % 128 of every
// (sequence, head) among them.  A pair whose items are all here is done; of the
// others (the first and the last at most) one partial per chunk goes to the slot of
// its first item in the chunk, and the CTA whose count completes the pair joins the
// partials.  Returns false if a wait ran out.
__device__ bool decode_chunk(const Args& a, const PlanView& v, int i0, int cnt, uint8_t* payload,
                             Shared& sh, uint32_t& phase) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  float* parts = reinterpret_cast<float*>(payload + NW * RING_BYTES);
  bool ok = true;
  if ((warp >> 1) < cnt) {
    const int item = i0 + (warp >> 1);
    const int4 it = v.dec[2 * item], info = v.dec[2 * item + 1];
    const int seq = it.x, g = it.y, mid = (it.z + it.w + 1) >> 1;
    const int32_t* bt = a.block_tables + (size_t)(a.seq_bt_row ? a.seq_bt_row[seq] : seq) * a.bt_pitch;
    float o[8][4], m[2], l[2];
    ok = decode_range(a, payload + warp * RING_BYTES, sh.bar[warp], phase, bt, info.x, g,
                      (warp & 1) ? mid : it.z, (warp & 1) ? it.w : mid, info.y, o, m, l);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[k] += __shfl_xor_sync(0xffffffffu, l[k], d);
    float* pw = parts + warp * PART_FLOATS;
    if (c < 2) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float* ph = pw + (2 * c + k) * HY_HEAD_DIM + 8 * r;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float4* p4 = reinterpret_cast<float4*>(ph + 64 * half);
          p4[0] = make_float4(o[0][2 * half + k], o[4][2 * half + k], o[1][2 * half + k], o[5][2 * half + k]);
          p4[1] = make_float4(o[2][2 * half + k], o[6][2 * half + k], o[3][2 * half + k], o[7][2 * half + k]);
        }
        if (r == 0) {
          pw[HY_GROUP * HY_HEAD_DIM + 2 * (2 * c + k)] = m[k];
          pw[HY_GROUP * HY_HEAD_DIM + 2 * (2 * c + k) + 1] = l[k];
        }
      }
    }
  }
  if (__syncthreads_or(!ok)) return false;

  const int head = tid >> 7, d = tid & 127;
  int open_first[2] = {-1, -1}, open_ns[2], open_cnt[2], n_open = 0;
  for (int j = 0; j < cnt;) {
    const int4 it = v.dec[2 * (i0 + j)], info = v.dec[2 * (i0 + j) + 1];
    const int ns = info.z, first = info.w;
    const int run = min(cnt - j, first + ns - (i0 + j));  // items of this pair in the chunk
    float M = -INFINITY;
    for (int w = 2 * j; w < 2 * (j + run); ++w)
      M = fmaxf(M, parts[w * PART_FLOATS + HY_GROUP * HY_HEAD_DIM + 2 * head]);
    const float Mu = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc = 0.f;
    for (int w = 2 * j; w < 2 * (j + run); ++w) {
      const float* pw = parts + w * PART_FLOATS;
      const float wt = ex2_ftz(pw[HY_GROUP * HY_HEAD_DIM + 2 * head] - Mu);
      L = fmaf(wt, pw[HY_GROUP * HY_HEAD_DIM + 2 * head + 1], L);
      acc = fmaf(wt, pw[tid], acc);
    }
    if (run == ns) {
      a.out[((size_t)info.x * a.q_heads + it.y * HY_GROUP + head) * HY_HEAD_DIM + d] =
          __float2bfloat16_rn(acc / L);
    } else {
      __stcg(v.part_o + (size_t)(i0 + j) * (HY_GROUP * HY_HEAD_DIM) + tid, acc);
      if (d == 0) __stcg(v.part_ml + (size_t)(i0 + j) * HY_GROUP + head, make_float2(M, L));
      open_first[n_open & 1] = first;
      open_ns[n_open & 1] = ns;
      open_cnt[n_open & 1] = run;
      ++n_open;
    }
    j += run;
  }
  if (n_open == 0) {
    __syncthreads();                                      // parts are read
    return true;
  }
  __threadfence();                                        // this CTA's partials, before the count
  __syncthreads();
  if (tid == 0) {
    int last = 0;
    for (int k = 0; k < n_open; ++k) {
      const int4 it = v.dec[2 * open_first[k]];
      int* ctr = &v.counters[it.x * a.kv_heads + it.y];
      if (atomicAdd(ctr, open_cnt[k]) + open_cnt[k] == open_ns[k]) {
        last |= 1 << k;
        *ctr = 0;                                         // for the next launch on this plan
      }
    }
    sh.last = last;
  }
  __syncthreads();
  const int last = sh.last;
  __threadfence();                                        // the others' partials, after the count
  for (int k = 0; k < n_open; ++k) {
    if (!((last >> k) & 1)) continue;
    const int first = open_first[k], end = first + open_ns[k];
    const int4 it = v.dec[2 * first], info = v.dec[2 * first + 1];
    // partials stand at the pair's first item and at every chunk boundary inside it
    auto next = [](int i) { return (i / CHUNK + 1) * CHUNK; };
    float M = -INFINITY;
    for (int i = first; i < end; i = next(i))
      M = fmaxf(M, __ldcg(v.part_ml + (size_t)i * HY_GROUP + head).x);
    const float Mu = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc = 0.f;
#pragma unroll 4
    for (int i = first; i < end; i = next(i)) {
      const float2 ml = __ldcg(v.part_ml + (size_t)i * HY_GROUP + head);
      const float wt = ex2_ftz(ml.x - Mu);
      L = fmaf(wt, ml.y, L);
      acc = fmaf(wt, __ldcg(v.part_o + (size_t)i * (HY_GROUP * HY_HEAD_DIM) + tid), acc);
    }
    a.out[((size_t)info.x * a.q_heads + it.y * HY_GROUP + head) * HY_HEAD_DIM + d] =
        __float2bfloat16_rn(acc / L);
  }
  return true;
}

__global__ void __launch_bounds__(NT, 1) attn_q4_kernel(Args a, PlanView v) {
  __shared__ Shared sh;
  extern __shared__ __align__(128) uint8_t payload[];
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int w = 0; w < NW; ++w)
      for (int s = 0; s < NS; ++s) mbar_init(&sh.bar[w][s], 1);
    fence_mbar_init();
  }
  __syncthreads();
  hy_grid_wait();
  hy_grid_trigger();
  const uint64_t keep = l2_keep_policy();
  const int n_dec = ld_keep(v.header + 1, keep), n_pairs = ld_keep(v.header + 4, keep);
  uint32_t phase = 0;
  (void)warp;
  if (n_pairs > 0) {                                      // a (sequence, KV head) pair per CTA
    for (int p = blockIdx.x; p < n_pairs; p += gridDim.x) {
      const int seq = p / a.kv_heads, g = p - seq * a.kv_heads;
      const int2 si = v.seqinfo[seq];                     // first item, items per head
      if (si.y > 0 && !decode_chunk(a, v, si.x + g * si.y, si.y, payload, sh, phase)) return;
    }
    return;
  }
  const int chunks = (n_dec + CHUNK - 1) / CHUNK;
  if (chunks <= (int)gridDim.x) {                         // one round: no counters
    if ((int)blockIdx.x < chunks)
      decode_chunk(a, v, blockIdx.x * CHUNK, min(CHUNK, n_dec - (int)blockIdx.x * CHUNK), payload,
                   sh, phase);
    return;
  }
  int* grab = v.grab + HY_GRAB_INTS * (a.layer & 63);
  bool ok = true;
  for (;;) {
    if (threadIdx.x == 0) sh.chunk = ok ? atomicAdd(&grab[0], 1) : chunks;
    __syncthreads();
    const int k = sh.chunk;
    __syncthreads();
    if (k >= chunks) break;
    ok = decode_chunk(a, v, k * CHUNK, min(CHUNK, n_dec - k * CHUNK), payload, sh, phase);
  }
  if (threadIdx.x == 0) {                                 // the last CTA out resets the counters
    __threadfence();
    if (atomicAdd(&grab[1], 1) == (int)gridDim.x - 1) {
      atomicExch(&grab[0], 0);
      atomicExch(&grab[2], 0);
      atomicExch(&grab[1], 0);
    }
  }
}

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
    const int32_t* __restrict__ seq_lens_k, int S, float scale, bool skip_decodes, int32_t* err) {
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
    if (skip_decodes && cu_q[seq + 1] - cu_q[seq] == 1) continue;
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
                          bool skip_decodes, int32_t* err, cudaStream_t st) {
  const long blocks = ((long)tokens * q_heads + 7) / 8;
  return hy_launch(attn_q4_scalar_kernel<T>, dim3((int)(blocks < 148L * 32 ? blocks : 148L * 32)),
                   dim3(256), 0, st, static_cast<const T*>(q), static_cast<T*>(out), tokens,
                   q_heads, kv_heads, cache_layer, num_blocks, block_tables, bt_pitch, seq_bt_row,
                   cu_q, seq_lens_k, S, scale, skip_decodes, err);
}

}  // namespace

cudaError_t hy_launch_attn_q4_fp32(const void* q, void* out, int tokens, int q_heads, int kv_heads,
                                   const void* cache_layer, int num_blocks,
                                   const int32_t* block_tables, int bt_pitch,
                                   const int32_t* seq_bt_row, const int32_t* cu_q,
                                   const int32_t* seq_lens_k, int S, float scale, int32_t* err,
                                   cudaStream_t st) {
  return launch_scalar<float>(q, out, tokens, q_heads, kv_heads,
                              static_cast<const uint8_t*>(cache_layer), num_blocks, block_tables,
                              bt_pitch, seq_bt_row, cu_q, seq_lens_k, S, scale, false, err, st);
}

cudaError_t hy_launch_attn_q4_bf16(const void* q, void* out, int tokens, int q_heads, int kv_heads,
                                   const void* cache_layer, int num_blocks, int layer,
                                   const int32_t* block_tables, int bt_pitch,
                                   const int32_t* seq_bt_row, const int32_t* cu_q,
                                   const int32_t* seq_lens_k, int S, float scale,
                                   const PlanDims& dims, void* ws, int32_t* err, int dev,
                                   cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(attn_q4_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       DEC_SMEM);
  if (e != cudaSuccess) return e;
  Args a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.cache = static_cast<const uint8_t*>(cache_layer);
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.num_blocks = num_blocks;
  a.layer = layer;
  a.block_tables = block_tables;
  a.bt_pitch = bt_pitch;
  a.seq_bt_row = seq_bt_row;
  a.cu_q = cu_q;
  a.seq_lens_k = seq_lens_k;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err = err;
  e = hy_launch(attn_q4_kernel, dim3(hy_attn_num_sms(dev)), dim3(NT), DEC_SMEM, st, a,
                hy_attn_plan_view(ws, dims));
  if (e != cudaSuccess) return e;
  return launch_scalar<__nv_bfloat16>(q, out, tokens, q_heads, kv_heads, a.cache, num_blocks,
                                      block_tables, bt_pitch, seq_bt_row, cu_q, seq_lens_k, S,
                                      scale, true, err, st);
}
