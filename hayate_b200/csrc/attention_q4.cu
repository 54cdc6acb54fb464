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
// Prefill items (64 query tokens x one KV head, 256 score rows) run on tcgen05: four
// warps expand key tiles to fp16 operands in shared memory, one warp per 128-row
// sub-tile issues the products, two warpgroups run the softmax.
// fp32 runs a scalar kernel.
#include "attention.cuh"
#include "attention_pieces.cuh"
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

// Prefill: warps 0-3 / 4-7 softmax of sub-tile 0 / 1, 8-11 expand, 12 / 13 issue the
// products of sub-tile 0 / 1.  Sub-tile X, row r: query head 4 g + 2 X + r / 64, token
// t0 + r % 64.  Q is [column half][128 rows][64] per sub-tile, a K or V ring slot [column
// half][64 keys][64], rows of 128 bytes with the 128-byte swizzle: the K-major operand
// of S = Q K^T and the MN-major operand of P V.
constexpr int EXP_WARP = 8, MMA_WARP = 12;
constexpr int PS = 4;                                     // K and V ring slots
constexpr int Q_BYTES = 128 * HY_HEAD_DIM * 2;            // Q of one sub-tile: 32 KB
constexpr int KV_BYTES = PRE_KEYS * HY_HEAD_DIM * 2;      // K or V of one tile: 16 KB
constexpr int K_OFF = 2 * Q_BYTES, V_OFF = K_OFF + PS * KV_BYTES;
constexpr int PRE_SMEM = V_OFF + PS * KV_BYTES;           // 192 KB
constexpr int SMEM_BYTES = (PRE_SMEM > DEC_SMEM ? PRE_SMEM : DEC_SMEM) + 1024;   // + alignment
// TMEM columns: two S buffers per sub-tile, P (fp16 pairs) written over the first half
// of its S; O at 256 + 128 X.
constexpr uint32_t TMEM_COLS = 512, TM_O = 256;
HY_DEVICE uint32_t tm_s(int X, uint32_t b) { return 64u * (2u * X + b); }

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
  // prefill; ring barriers complete once per use of their slot, the others once
  // per key tile (per use of their S buffer), qfull once per item
  uint64_t full[PS];      // K and V of a tile expanded (one arrival per expanding warp)
  uint64_t free_[PS];     // both P V products of the slot's tile are done
  uint64_t sfull[2][2];   // S_X[b] complete
  uint64_t pfull[2][2];   // P_X[b] written (one arrival per softmax warp)
  uint64_t odone[2];      // O_X += P_X V complete
  uint64_t drain[2];      // error path: everything an issuing warp issued is complete
  uint64_t qfull;         // Q written (one arrival per softmax warp)
  uint32_t tmem_base;
  int pre_item, pre_last;
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

// ------------------------------------------------------------------ prefill item
struct PreItem {
  int seq, g, t0, row0, nrows, prefix, kv_len, kv_end, tlo, thi, w;
};
HY_DEVICE PreItem pre_item_geom(const Args& a, const PlanView& v, int item) {
  const int4 it = v.pre_sorted[item];
  PreItem p;
  p.seq = it.x;
  p.g = it.y;
  p.t0 = it.z;
  p.w = it.w;
  p.row0 = a.cu_q[p.seq];
  const int q_len = a.cu_q[p.seq + 1] - p.row0;
  p.kv_len = a.seq_lens_k[p.seq];
  p.prefix = p.kv_len - q_len;
  p.nrows = min(PRE_QROWS, q_len - p.t0);
  p.kv_end = p.prefix + p.t0 + p.nrows;                   // keys its last row sees
  pre_piece_range(p.w, (p.kv_end + PRE_KEYS - 1) / PRE_KEYS, p.tlo, p.thi);
  return p;
}

// Expanding warps: thread t of 128 takes row t % 64 of every key tile's K (t < 64) or
// V: its 64 code bytes and parameters from global memory, the next tile's loaded
// ahead, to 256 bytes of fp16 in the ring.  Rows past the item's keys become zeros:
// their scores are masked, and a zero weight times a zero adds nothing.
struct RowCodes {
  uint4 w[4];
  uint32_t par[2];
};
HY_DEVICE int tile_block(const Args& a, const PreItem& P, const int32_t* bt, int pos) {
  if (pos >= P.kv_end) return -1;
  const int b = pos / HY_BLOCK;
  const int id = b < a.bt_pitch ? __ldg(bt + b) : -1;
  if (id >= 0 && id < a.num_blocks) return id;
  hy_flag(a.err, HY_ERR_BOUNDS);
  return -1;
}
HY_DEVICE void load_row(const Args& a, const PreItem& P, int part, int pos, int blk, RowCodes& x) {
  if (blk < 0) {
    x.w[0] = x.w[1] = x.w[2] = x.w[3] = make_uint4(0, 0, 0, 0);
    x.par[0] = x.par[1] = 0u;
    return;
  }
  const uint8_t* tile = a.cache + q4_tile(blk, P.g, part, a.kv_heads);
  const uint4* src = reinterpret_cast<const uint4*>(tile + (pos % HY_BLOCK) * Q4_ROW_BYTES);
#pragma unroll
  for (int i = 0; i < 4; ++i) x.w[i] = src[i];
  const uint2 p = *reinterpret_cast<const uint2*>(tile + Q4_PARAM_OFF + (pos % HY_BLOCK) * Q4_PARAM_BYTES);
  x.par[0] = p.x;
  x.par[1] = p.y;
}
HY_DEVICE void expand_row(const RowCodes& x, uint8_t* slot, int key) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const __half2 sm = q4_as_half2(x.par[half]);
    const __half2 s2 = __low2half2(sm), m2 = __high2half2(sm);
    uint8_t* row = slot + half * (KV_BYTES / 2) + key * 128;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 q = x.w[2 * half + (i >> 2)];
      const uint32_t w = (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
      uint32_t y[4];
      q4_expand(w, s2, m2, y);
      *reinterpret_cast<uint4*>(row + ((i ^ (key & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
}

// One prefill item, all warps of the CTA (roles as above).  The products, barriers
// and softmax follow attention.cu's prefill: S(t + 1) is issued while the softmax
// works on S(t); S(t) may overwrite its buffer because P V(t - 2) was issued before it
// by the same thread; the softmax writes P(t) over S(t) and waits for P V(t - 1) only
// to rescale O.  c = c0 + t counts key tiles over all items of the launch.
// Returns false if a wait ran out; the roles then drain what they issued.
__device__ bool prefill_item(const Args& a, const PlanView& v, int item, uint8_t* payload,
                             Shared& sh, uint32_t tmem, uint32_t& ctr, uint32_t qpar) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PreItem P = pre_item_geom(a, v, item);
  const int ntiles = P.thi - P.tlo;
  const uint32_t sbase = smem_u32(payload);
  const uint32_t c0 = ctr;
  ctr += ntiles;
  bool ok = true;

  if (warp >= EXP_WARP && warp < MMA_WARP) {
    const int t128 = tid - EXP_WARP * 32, part = t128 >> 6, key = t128 & 63;
    const int32_t* bt = a.block_tables + (size_t)(a.seq_bt_row ? a.seq_bt_row[P.seq] : P.seq) * a.bt_pitch;
    uint8_t* ring = payload + (part ? V_OFF : K_OFF);
    RowCodes cur, nxt;
    int pos = P.tlo * PRE_KEYS + key;
    load_row(a, P, part, pos, tile_block(a, P, bt, pos), nxt);
    int blk = ntiles > 1 ? tile_block(a, P, bt, pos + PRE_KEYS) : -1;
    for (int t = 0; t < ntiles; ++t) {
      cur = nxt;
      pos += PRE_KEYS;
      if (t + 1 < ntiles) load_row(a, P, part, pos, blk, nxt);
      if (t + 2 < ntiles) blk = tile_block(a, P, bt, pos + PRE_KEYS);
      const uint32_t c = c0 + t, slot = c % PS;
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.free_[slot], ((c / PS) & 1) ^ 1, a.err));
      if (!ok) break;
      expand_row(cur, ring + slot * KV_BYTES, key);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.full[slot]);
    }
  } else if (warp == MMA_WARP || warp == MMA_WARP + 1) {
    const int X = warp - MMA_WARP;
    if (lane == 0) {
      constexpr uint32_t ID_S = tc_idesc_f16(128, PRE_KEYS, false);
      constexpr uint32_t ID_O = tc_idesc_f16(128, HY_HEAD_DIM, true);
      const uint64_t dQ = tc_desc_sw128(sbase + X * Q_BYTES, 16, 1024);
      ok = mbar_wait(&sh.qfull, qpar, a.err);
      tc_fence_after();
      for (int t = 0; t <= ntiles && ok; ++t) {
        if (t < ntiles) {                                 // S_X(t) = Q_X K_t^T
          const uint32_t c = c0 + t, slot = c % PS;
          ok = mbar_wait(&sh.full[slot], (c / PS) & 1, a.err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t dK = tc_desc_sw128(sbase + K_OFF + slot * KV_BYTES, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < HY_HEAD_DIM / 16; ++kk)
            tc_mma_bf16(tmem + tm_s(X, c & 1),
                        dQ + (uint64_t)((((kk >> 2) * (Q_BYTES / 2)) + (kk & 3) * 32) >> 4),
                        dK + (uint64_t)((((kk >> 2) * (KV_BYTES / 2)) + (kk & 3) * 32) >> 4), ID_S,
                        kk > 0);
          tc_commit(&sh.sfull[X][c & 1]);
        }
        if (t > 0) {                                      // O_X += P_X(t - 1) V_{t-1}
          const uint32_t c = c0 + t - 1, slot = c % PS;
          ok = mbar_wait(&sh.pfull[X][c & 1], (c >> 1) & 1, a.err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t dV = tc_desc_sw128(sbase + V_OFF + slot * KV_BYTES, KV_BYTES / 2, 1024);
#pragma unroll
          for (int kk = 0; kk < PRE_KEYS / 16; ++kk)
            tc_mma_bf16_ta(tmem + TM_O + 128 * X, tmem + tm_s(X, c & 1) + 8 * kk,
                           dV + (uint64_t)((kk * 2048) >> 4), ID_O, (t > 1 || kk > 0));
          tc_commit(&sh.odone[X]);
          tc_commit(&sh.free_[slot]);
        }
      }
      if (!ok) {                                          // let every issued product finish
        tc_commit(&sh.drain[X]);
        mbar_wait(&sh.drain[X], 0, nullptr);
      }
    }
    __syncwarp();
  } else if (warp < EXP_WARP) {                           // softmax: thread = row = TMEM lane
    const int X = warp >> 2, r = (warp & 3) * 32 + lane, j = r & 63;
    const int head = P.g * HY_GROUP + 2 * X + (r >> 6);
    const size_t at = ((size_t)(P.row0 + P.t0 + j) * a.q_heads + head) * HY_HEAD_DIM;
    const bool real = j < P.nrows;
    float sl2;                                            // scale to log2 units of this row
    {                                                     // Q row r in fp16 (q4_query_scale)
      uint4 u[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        u[i] = real ? reinterpret_cast<const uint4*>(a.q + at)[i] : make_uint4(0, 0, 0, 0);
      float amax = 0.f, down, up;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float lo = __uint_as_float(w[k] << 16), hi = __uint_as_float(w[k] & 0xffff0000u);
          amax = fmax3f(amax, fabsf(lo), fabsf(hi));
        }
      }
      q4_query_scale(amax, down, up);
      // not 0 (a scale of 0, a row of tiny elements): masked scores are -inf times it,
      // and the scores it multiplies, at most 2^24, stay 0 to fp32 either way
      sl2 = fmaxf(a.scale_log2 * up, 1e-30f);
      uint8_t* row = payload + X * Q_BYTES + r * 128;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
        uint32_t y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          y[k] = q4_as_u32(__floats2half2_rn(__uint_as_float(w[k] << 16) * down,
                                             __uint_as_float(w[k] & 0xffff0000u) * down));
        *reinterpret_cast<uint4*>(row + (i >> 3) * (Q_BYTES / 2) + (((i & 7) ^ (r & 7)) << 4)) =
            make_uint4(y[0], y[1], y[2], y[3]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.qfull);
    }
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_base + TM_O + 128 * X;
    const int lim = P.prefix + P.t0 + j;                  // last key row r may see
    float m = NEG_INF, l = 0.f;                           // m in scaled log2 units
    for (int t = 0; t < ntiles && ok; ++t) {
      const uint32_t c = c0 + t;
      const uint32_t tS = tmem + lane_base + tm_s(X, c & 1);
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.sfull[X][c & 1], (c >> 1) & 1, a.err));
      if (!ok) break;
      tc_fence_after();
      float s[64];
      tmem_ld32(tS, *reinterpret_cast<float(*)[32]>(&s[0]));
      tmem_ld32(tS + 32, *reinterpret_cast<float(*)[32]>(&s[32]));
      tmem_wait_ld();
      const int kb = (P.tlo + t) * PRE_KEYS;
      if (kb + PRE_KEYS - 1 > P.prefix + P.t0) {          // the tile reaches the diagonal or the end
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (kb + i > lim || kb + i >= P.kv_end) s[i] = NEG_INF;
      }
      float mxs[8];                                       // 8 independent chains
#pragma unroll
      for (int k = 0; k < 8; ++k) mxs[k] = fmax3f(s[k], s[8 + k], s[16 + k]);
#pragma unroll
      for (int i = 24; i < 56; i += 16)
#pragma unroll
        for (int k = 0; k < 8; ++k) mxs[k] = fmax3f(mxs[k], s[i + k], s[i + 8 + k]);
#pragma unroll
      for (int k = 0; k < 8; ++k) mxs[k] = fmaxf(mxs[k], s[56 + k]);
      const float mx = sl2 * fmax3f(fmax3f(mxs[0], mxs[1], mxs[2]), fmax3f(mxs[3], mxs[4], mxs[5]),
                                    fmaxf(mxs[6], mxs[7]));
      const bool grow = mx > m + RESCALE_LOG2;
      if (__any_sync(0xffffffffu, grow)) {
        const float mnew = grow ? mx : m;
        const float alpha = mnew == NEG_INF ? 1.f : ex2_ftz(m - mnew);
        l *= alpha;
        m = mnew;
        if (t > 0) {                                      // O holds tiles < t: wait for P V(t - 1)
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.odone[X], (c & 1) ^ 1, a.err));
          tc_fence_after();
#pragma unroll 1
          for (int cc = 0; cc < 4; ++cc) {
            float o[32];
            tmem_ld32(tO + 32 * cc, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= alpha;
            tmem_st32(tO + 32 * cc, o);
          }
          tmem_wait_st();
        }
      }
      const float mneg = (m == NEG_INF) ? 0.f : -m;
      const float2 sl2v = make_float2(sl2, sl2), mnegv = make_float2(mneg, mneg);
      uint32_t pk[32];
      float2 ls[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                      make_float2(0.f, 0.f)};
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float2 x = __ffma2_rn(make_float2(s[2 * i], s[2 * i + 1]), sl2v, mnegv);
        const float p0 = ex2_ftz(x.x), p1 = ex2_ftz(x.y);
        ls[i & 3] = __fadd2_rn(ls[i & 3], make_float2(p0, p1));
        pk[i] = q4_as_u32(__floats2half2_rn(p0, p1));
      }
      l += ((ls[0].x + ls[0].y) + (ls[1].x + ls[1].y)) + ((ls[2].x + ls[2].y) + (ls[3].x + ls[3].y));
      tmem_st32u(tS, pk);                                 // P(t) over the first 32 columns of S(t)
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.pfull[X][c & 1]);
    }
    if (ok) {                                             // epilogue: O_X complete
      const uint32_t c = c0 + ntiles - 1;
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.odone[X], c & 1, a.err));
      tc_fence_after();
    }
    const bool store = ok && real;
    __nv_bfloat16* op = a.out + at;
    if (P.w != 0) {                                       // a piece: every softmax thread takes part
      ok = prefill_piece_finish(v, P.w, X * 128 + r, tO, m, l, ok, store ? op : nullptr,
                                sh.pre_last);
    } else if (ok) {
      const float inv = 1.f / l;
#pragma unroll 1
      for (int cc = 0; cc < 4; ++cc) {
        float o[32];
        tmem_ld32(tO + 32 * cc, o);                       // warp-collective: every lane loads
        tmem_wait_ld();
        if (store) {
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<uint4*>(op + 32 * cc + 8 * q4) =
                make_uint4(pack_bf16(o[8 * q4 + 0] * inv, o[8 * q4 + 1] * inv),
                           pack_bf16(o[8 * q4 + 2] * inv, o[8 * q4 + 3] * inv),
                           pack_bf16(o[8 * q4 + 4] * inv, o[8 * q4 + 5] * inv),
                           pack_bf16(o[8 * q4 + 6] * inv, o[8 * q4 + 7] * inv));
        }
      }
    }
  }
  tc_fence_before();
  if (__syncthreads_or(!ok)) ok = false;
  return ok;
}

// Decode items, in whichever way suits their number.  Returns false if a wait ran out.
__device__ bool decode_items(const Args& a, const PlanView& v, int n_pre, int n_dec, int n_pairs,
                             uint8_t* payload, Shared& sh) {
  uint32_t phase = 0;
  if (n_pairs > 0) {                                      // a (sequence, KV head) pair per CTA
    if ((int)blockIdx.x >= n_pairs) return true;
    const int seq = (int)blockIdx.x / a.kv_heads, g = (int)blockIdx.x - seq * a.kv_heads;
    const int2 si = v.seqinfo[seq];                       // first item, items per head
    return si.y == 0 || decode_chunk(a, v, si.x + g * si.y, si.y, payload, sh, phase);
  }
  const int chunks = (n_dec + CHUNK - 1) / CHUNK;
  if (n_pre == 0 && chunks <= (int)gridDim.x) {           // one round: no counters
    if ((int)blockIdx.x >= chunks) return true;
    const int i0 = (int)blockIdx.x * CHUNK;
    return decode_chunk(a, v, i0, min(CHUNK, n_dec - i0), payload, sh, phase);
  }
  int* grab = v.grab + HY_GRAB_INTS * (a.layer & 63);
  for (;;) {
    if (threadIdx.x == 0) sh.chunk = atomicAdd(&grab[0], 1);
    __syncthreads();
    const int k = sh.chunk;
    __syncthreads();
    if (k >= chunks) return true;
    if (!decode_chunk(a, v, k * CHUNK, min(CHUNK, n_dec - k * CHUNK), payload, sh, phase))
      return false;
  }
}

__global__ void __launch_bounds__(NT, 1) attn_q4_kernel(Args a, PlanView v) {
  __shared__ Shared sh;
  extern __shared__ uint8_t dyn_smem[];
  uint8_t* payload = dyn_smem + ((1024u - (smem_u32(dyn_smem) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int w = 0; w < NW; ++w)
      for (int s = 0; s < NS; ++s) mbar_init(&sh.bar[w][s], 1);
    for (int s = 0; s < PS; ++s) {
      mbar_init(&sh.full[s], MMA_WARP - EXP_WARP);
      mbar_init(&sh.free_[s], 2);                         // one commit per MMA warp
    }
    for (int x = 0; x < 2; ++x) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&sh.sfull[x][b], 1);
        mbar_init(&sh.pfull[x][b], 4);
      }
      mbar_init(&sh.odone[x], 1);
      mbar_init(&sh.drain[x], 1);
    }
    mbar_init(&sh.qfull, EXP_WARP);
    fence_mbar_init();
  }
  __syncthreads();
  hy_grid_wait();
  hy_grid_trigger();
  const uint64_t keep = l2_keep_policy();
  const int n_pre = ld_keep(v.header, keep), n_dec = ld_keep(v.header + 1, keep);
  const int n_pairs = ld_keep(v.header + 4, keep);
  int* grab = v.grab + HY_GRAB_INTS * (a.layer & 63);
  bool ok = true;
  if ((int)blockIdx.x < n_pre) {                          // the first n_pre CTAs take prefill items
    if (warp == 0) {
      tmem_alloc(&sh.tmem_base, TMEM_COLS);
      tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem_base;
    uint32_t tile_ctr = 0;
    for (uint32_t n = 0; ok; ++n) {
      if (threadIdx.x == 0) sh.pre_item = atomicAdd(&grab[2], 1);
      __syncthreads();
      const int k = sh.pre_item;
      __syncthreads();
      if (k >= n_pre) break;
      ok = prefill_item(a, v, k, payload, sh, tmem, tile_ctr, n & 1);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      tmem_dealloc(tmem, TMEM_COLS);
    }
  }
  if (ok) decode_items(a, v, n_pre, n_dec, n_pairs, payload, sh);
  __syncthreads();
  if ((n_pre > 0 || n_dec > CHUNK * (int)gridDim.x) && threadIdx.x == 0) {
    __threadfence();                                      // the last CTA out resets the counters
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

cudaError_t hy_launch_attn_q4_fp32(const void* q, void* out, int tokens, int q_heads, int kv_heads,
                                   const void* cache_layer, int num_blocks,
                                   const int32_t* block_tables, int bt_pitch,
                                   const int32_t* seq_bt_row, const int32_t* cu_q,
                                   const int32_t* seq_lens_k, int S, float scale, int32_t* err,
                                   cudaStream_t st) {
  return launch_scalar<float>(q, out, tokens, q_heads, kv_heads,
                              static_cast<const uint8_t*>(cache_layer), num_blocks, block_tables,
                              bt_pitch, seq_bt_row, cu_q, seq_lens_k, S, scale, err, st);
}

cudaError_t hy_launch_attn_q4_bf16(const void* q, void* out, int q_heads, int kv_heads,
                                   const void* cache_layer, int num_blocks, int layer,
                                   const int32_t* block_tables, int bt_pitch,
                                   const int32_t* seq_bt_row, const int32_t* cu_q,
                                   const int32_t* seq_lens_k, int S, float scale,
                                   const PlanDims& dims, void* ws, int32_t* err, int dev,
                                   cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(attn_q4_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       SMEM_BYTES);
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
  return hy_launch(attn_q4_kernel, dim3(hy_attn_num_sms(dev)), dim3(NT), SMEM_BYTES, st, a,
                   hy_attn_plan_view(ws, dims));
}
