// Varlen paged GQA attention over the 4-bit KV cache (layout: q4.cuh).
//
// Semantics as attention.cu: the j-th query token of sequence i sits at position
// prefix_i + j (prefix_i = seq_len_k_i - q_len_i) and attends to keys
// [0, prefix_i + j] of its own sequence (hayate/model/attention.py:52-64 with the
// masks of hayate/model/qwen.py:66-106); here a key or value is what its codes
// stand for, scale * code + minimum.
//
// bf16 runs on the tensor cores, in two kernels.  The decode kernel takes steps of one
// query token per sequence: the key blocks of all (sequence, head) pairs, one after the
// other, are dealt evenly over every warp of the grid; a warp streams its blocks (2304
// bytes: K and V of one block and head are adjacent) through a ring of bulk copies and
// feeds their codes to mma.sync as they are (4 query heads would fill 3 % of a tcgen05
// tile); warps of a CTA merge what they share in shared memory, CTAs through the
// workspace.  Bound by the cache's bytes: 256 sequences of 4096 keys take 214 to 231 us
// from run to run, 5.2 to 5.6 TB/s (of 6.5 for a copy); a launch costs about 9 us beside
// its blocks, of which the smallest steps consist (one sequence of 600 keys 8.85 us; of
// 40960 keys 19.8).
// The other kernel adds prefill items (64 query tokens x one KV head, 256 score rows) on
// tcgen05: four warps expand key tiles to fp16 operands in shared memory, one warp per
// 128-row sub-tile issues the products, two warpgroups run the softmax.  Bound by the
// softmax and the products taking turns in a sub-tile (two sub-tiles overlap): 16 chunks
// of 512 tokens with 4096 keys take 565 to 593 us back to back, 870 to 910 TFLOP/s (55 % of
// a large bf16 product's burst rate; the bf16 cache's kernel 618 beside 565).
// Key tiles of 128, with one S buffer per sub-tile, ran the same in 793 us.
// fp32 runs a kernel of its own on the fp32 units.
#include "attention.cuh"
#include "attention_pieces.cuh"
#include "q4.cuh"

#include <atomic>
#include <float.h>
#include <limits.h>
#include <math.h>

namespace {

constexpr int NW = 16;                                    // warps per CTA
constexpr int NT = NW * 32;
constexpr int BLK_BYTES = 2 * Q4_TILE_BYTES;              // K and V tile of one block and head
constexpr int STAGE_BYTES = 2 * BLK_BYTES;                // a decode warp takes two blocks at a time
constexpr int NS = 2;                                     // stages of a decode warp's ring
constexpr int RING_BYTES = NS * STAGE_BYTES;
// a warp's partial result of one (sequence, head): O [4][128], then (m, l) [4]
constexpr int PART_FLOATS = HY_GROUP * HY_HEAD_DIM + 2 * HY_GROUP;
constexpr int DEC_SMEM = NW * (RING_BYTES + 2 * PART_FLOATS * 4) + 1024;   // + alignment
constexpr float RESCALE_LOG2 = 8.0f;                      // see decode_warp
// A weight is 2^(score mult - m), m the running maximum in log2 units, by one multiply-add.
// m is rounded to fp32, which scales all weights alike, by next to nothing while |m| is
// at most this (2^-24 of it is 2^-4).  Past it the factor could leave fp16's range: the
// threshold above which m is raised is then the largest score itself, without slack, and
// the weights are 2^((score - threshold) mult), in a branch that ordinary rows never enter.
constexpr float FAR_LOG2 = 1048576.0f;
HY_DEVICE float raise_above(float score, float m, float mult) {
  return fabsf(m) <= FAR_LOG2 ? (m + RESCALE_LOG2) / mult : score;
}
// What scores (of a query row scaled by 1 / up) are multiplied with: log2 units.  Not 0 (a
// scale of 0, a row of tiny elements): masked scores are -inf times it.  Not infinite:
// where it would be, scores that differ are so far apart that a smaller factor gives the
// same weights.
HY_DEVICE float score_mult(float scale_log2, float up) {
  return fminf(fmaxf(scale_log2 * up, 1e-30f), FLT_MAX);
}

// Prefill: warps 0-3 / 4-7 softmax of sub-tile 0 / 1, 8-11 expand, 12 / 13 issue the
// products of sub-tile 0 / 1, 14 deals out items and loads Q.  Sub-tile X, row r: query
// head 4 g + 2 X + r / 64, token t0 + r % 64.  Q is [column half][128 rows][64] per
// sub-tile, a K or V ring slot [column half][64 keys][64], rows of 128 bytes with the
// 128-byte swizzle: the K-major operand of S = Q K^T and the MN-major operand of P V.
constexpr int EXP_WARP = 8, MMA_WARP = 12, ITEM_WARP = 14;
constexpr int ITEM_READERS = 14;                          // the warps before ITEM_WARP
constexpr int PS = 4;                                     // K and V ring slots
constexpr int Q_BYTES = 128 * HY_HEAD_DIM * 2;            // Q of one sub-tile: 32 KB
constexpr int KV_BYTES = PRE_KEYS * HY_HEAD_DIM * 2;      // K or V of one tile: 16 KB
constexpr int K_OFF = 2 * Q_BYTES, V_OFF = K_OFF + PS * KV_BYTES;
constexpr int PRE_SMEM = V_OFF + PS * KV_BYTES;           // 192 KB
constexpr int MIXED_SMEM = PRE_SMEM + 1024 > DEC_SMEM ? PRE_SMEM + 1024 : DEC_SMEM;
// TMEM columns: two S buffers per sub-tile, P (fp16 pairs) written over the first half
// of its S; O at 256 + 128 X.
constexpr uint32_t TMEM_COLS = 512, TM_O = 256;
HY_DEVICE uint32_t tm_s(int X, uint32_t b) { return 64u * (2u * X + b); }

struct Args {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const uint8_t* cache;   // this layer's tiles
  int q_heads, kv_heads, num_blocks, layer, num_seqs, num_tokens;
  int block_cap;          // hy_dec_block_cap
  const int32_t* block_tables;
  int bt_pitch;
  const int32_t* seq_bt_row;
  float scale_log2;
  int32_t* err;
};

// A prefill item (or a key-range piece of one): query tokens t0 .. t0 + nrows - 1 of a
// sequence, KV head g, key tiles [tlo, thi).
struct PreItem {
  int seq, g, t0, row0, nrows, prefix, kv_end, tlo, thi, w;   // seq -1: no more items
};

// A place in the flattened list of key blocks (sequence, head, block) of the step's
// decode sequences, with what a warp needs of the sequence.  Warps keep theirs in shared
// memory: it is read once per pair, and the key loop needs the registers.
struct Cursor {
  int seq, g, b, nb;                                      // block b of nb
  int first, tok, kv_len, row;                            // of the sequence, see SeqInfo
};

// 1 / x of a power of two whose inverse is normal.
HY_DEVICE float pow2_inverse(float x) { return __int_as_float(0x7f000000 - __float_as_int(x)); }

// Maximum over the warp; NaN only if every lane's is.
HY_DEVICE float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

// What a warp leaves of a pair that it did not finish alone.
struct Part {
  int pair;               // sequence * kv_heads + head, -1: none
  int blocks, nb;         // blocks that it covers, blocks of the pair
  int first;              // the pair's first block in the flattened list
  int tok;                // query row
};

// Where the partials of an open pair are: units u0 .. u1, u0's in its second slot if the
// pair starts inside it; and the pair's first row of the output.
struct Join {
  int u0, u1, inside, row;
};

struct Shared {
  uint64_t bar[NW][NS];
  int unit;               // the CTA's next unit of decode work
  int last;               // bit j: this CTA finished pair j of its two open ones
  Join join[2];
  Part part[2 * NW];      // each warp's two parts, in block order
  Cursor cur[NW][2];      // each warp's pair computed, and next block to load
  // prefill; ring barriers complete once per use of their slot, sfull, pfull and odone
  // once per use of their S buffer, the others once per item
  uint64_t full[PS];      // K and V of a tile expanded (one arrival per expanding warp)
  uint64_t free_[PS];     // both P V products of the slot's tile are done
  uint64_t sfull[2][2];   // S_X[b] complete
  uint64_t pfull[2][2];   // P_X[b] written (one arrival per softmax warp)
  uint64_t odone[2][2];   // O_X += P_X[b] V complete
  uint64_t drain[2];      // error path: everything an issuing warp issued is complete
  uint64_t qraw;          // Q landed as bf16 (TMA transaction bytes)
  uint64_t qfull;         // Q is fp16 (one arrival per softmax warp)
  uint64_t ofree[2];      // O_X is read out (one arrival per softmax warp)
  uint64_t qfree;         // both sub-tiles' last S is done (one commit each)
  uint64_t itemfull;      // item[n % 2] is the CTA's item n
  uint64_t itemfree;      // every warp has read it (one arrival each)
  uint64_t expdone;       // the item's last tile is about to be expanded (one arrival per
                          // expanding warp)
  PreItem item[2];
  int nan_at[2][2];       // [item n % 2][half]: the first key whose value is NaN there
  uint32_t tmem_base;
  int pre_last;
};

// Row of the score matrix S^T (row r or r + 8 of the 16-key block) -> key of the
// block.  Any order of the 16 keys is right as long as K's rows, the weights and V
// agree; this one puts the four keys that lane (r, c) takes from V, and the two
// neighbouring rows it takes from K, in different halves of the 32 shared-memory
// banks (a key's 64 bytes of codes are half of them).
HY_DEVICE int key_of(int c, int e, int h) {               // row 2 c + e + 8 h, c < 4
  return ((c ^ e) & 1) | (e << 1) | (h << 2) | ((c >> 1) << 3);
}

// A word's nibbles as fp16 pairs without any arithmetic: nibble n in bits 0-3 of a half
// is the subnormal n 2^-24, in bits 4-7 it is 16 n 2^-24; the tensor core multiplies
// subnormals exactly.  x[0], x[2] hold n, x[1], x[3] 16 n (pairs as in q4_expand).
HY_DEVICE void q4_bits(uint32_t w, uint32_t (&x)[4]) {
  const uint32_t w8 = w >> 8;
  x[0] = w & 0x000f000fu;
  x[1] = w & 0x00f000f0u;
  x[2] = w8 & 0x000f000fu;
  x[3] = w8 & 0x00f000f0u;
}

// What a sequence is to the decode: its first block in the list of all sequences' key
// blocks, query row, key length and block-table row.  All but the last are the plan's, so
// that they agree with its counts of blocks whatever the caller's arrays hold by now.
struct SeqInfo {
  int first, tok, kv_len, row;
};
HY_DEVICE SeqInfo seq_info(const Args& a, const PlanView& v, int seq) {
  const int4 s = v.seqs[seq];
  return SeqInfo{s.x, s.y, s.z, a.seq_bt_row ? a.seq_bt_row[seq] : seq};
}
// The workspace's plan.  One of other sequences or capacities (or none), or of query rows
// that q does not have, is reported and holds no work.
HY_DEVICE HyPlan load_plan(const Args& a, const PlanView& v) {
  const uint64_t keep = l2_keep_policy();
  const int4 x = ld_keep(reinterpret_cast<const int4*>(v.header + 8), keep);
  const int4 y = ld_keep(reinterpret_cast<const int4*>(v.header + 12), keep);
  const int bad = x.z != a.num_seqs || x.w != v.key ? HY_ERR_PLAN
                  : y.z < 0 || y.w > a.num_tokens ? HY_ERR_BOUNDS : 0;
  if (bad) {
    if (threadIdx.x == 0) hy_flag(a.err, bad);
    return HyPlan{};
  }
  return HyPlan{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
}
// The search of cursor_at begins with sequences `top_step` apart, one per lane; they are
// loaded before the kernel knows whether it has decode work.
HY_DEVICE int top_step(const Args& a) {
  int step = 1;
  while ((long)step * 32 < a.num_seqs) step *= 32;
  return step;
}

HY_DEVICE SeqInfo seq_top(const Args& a, const PlanView& v) {
  return seq_info(a, v, (int)min((threadIdx.x & 31) * (long)top_step(a), a.num_seqs - 1L));
}

HY_DEVICE void cursor_sequence(const Args& a, Cursor& k, const SeqInfo& s) {
  k.first = s.first;
  k.tok = s.tok;
  k.kv_len = s.kv_len;
  k.nb = min((s.kv_len + HY_BLOCK - 1) / HY_BLOCK, a.block_cap);   // as the plan counts them
  k.row = s.row;
}
// The place of flattened block f: the last sequence that starts at or before it, found
// by the whole warp 32 sequences (or runs of 32^n) at a time.
HY_DEVICE Cursor cursor_at(const Args& a, const PlanView& v, const SeqInfo& top, int f) {
  const int lane = threadIdx.x & 31;
  int lo = 0;
  SeqInfo s = top;
  for (int step = top_step(a);; step >>= 5) {
    const long i = lo + (long)lane * step;
    const bool le = i < a.num_seqs && s.first * a.kv_heads <= f;
    const int at = 31 - __clz(__ballot_sync(0xffffffffu, le) | 1u);
    lo += at * step;
    if (step == 1) {
      s = SeqInfo{__shfl_sync(0xffffffffu, s.first, at), __shfl_sync(0xffffffffu, s.tok, at),
                  __shfl_sync(0xffffffffu, s.kv_len, at), __shfl_sync(0xffffffffu, s.row, at)};
      break;
    }
    s = seq_info(a, v, (int)min(lo + (long)lane * (step >> 5), a.num_seqs - 1L));
  }
  Cursor k;
  k.seq = lo;
  cursor_sequence(a, k, s);
  const int in = f - s.first * a.kv_heads;
  k.g = in / k.nb;
  k.b = in - k.g * k.nb;
  return k;
}
// Step to the next (sequence, head) once all blocks of this one are passed.
HY_DEVICE void cursor_next_pair(const Args& a, const PlanView& v, Cursor& k) {
  k.b = 0;
  if (++k.g < a.kv_heads) return;
  k.g = 0;
  do {
    ++k.seq;
  } while (v.seqs[k.seq + 1].x == v.seqs[k.seq].x);
  cursor_sequence(a, k, seq_info(a, v, k.seq));
}

// One warp: n_blocks key blocks of the flattened list from cur[0] (= cur[1]) on, pair by
// pair, two blocks (32 keys) at a time.
//
// Scores are computed transposed, S^T = K Q^T (16 keys x 8 columns, the 4 heads twice),
// and so is the output, O^T = V^T P^T: the codes then fill the 16-row operand of
// mma.sync, where the 4 heads alone would leave three quarters of it empty.  The codes
// enter the products as they are (q4_bits), and the parameters outside them:
//   score = sum over halves of scale_K (code . q) + minimum_K (sum of q)
//   out   = sum over keys of (p scale_V) code + p minimum_V
// so that an expanded value costs 5/8 of an instruction and keys are exact.  The
// minima of K meet the sums of q in a product of their own (the sums as two fp16
// parts, 22 bits); p and p scale_V are rounded to fp16 (2^-11 each), the output to bf16.
// p scale_V is kept inside fp16's normal range by a power of two vs: p is at most 2^8
// (the maximum is only raised when a score exceeds it by more than that, so that most
// blocks need no exchange between lanes), scale_V vs at most 2^7.
// The 8 columns hold the 4 heads twice: the products with V use the second ones for the
// odd dimensions.  Lane (r, c) = (lane / 4, lane % 4) ends with heads 2 (c % 2) + k (k = 0,
// 1) at dimensions 8 r + 2 i + c / 2 of either half.  ring_pos: the ring's next stage, ring_par the
// parity of its next pass.  Returns false if a wait ran out.
HY_DEVICE bool decode_warp(const Args& a, const PlanView& v, Cursor (&cur)[2], int n_blocks, uint8_t* ring_ptr,
                           float* part, Part* parts, uint64_t* bars,
                           uint32_t& ring_pos, uint32_t& ring_par) {
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  if (n_blocks == 0) return true;
  const uint32_t ring = smem_u32(ring_ptr);
  int to_load = n_blocks, left = n_blocks;
  uint4 qraw[4];                                          // this lane's part of Q
  auto load_q = [&]() {
    const __nv_bfloat16* qp =
        a.q + ((size_t)cur[0].tok * a.q_heads + cur[0].g * HY_GROUP + (r & 3)) * HY_HEAD_DIM + 16 * c;
#pragma unroll
    for (int i = 0; i < 4; ++i) qraw[i] = *reinterpret_cast<const uint4*>(qp + 64 * (i >> 1) + 8 * (i & 1));
  };
  load_q();

  // Loads: the ids of the next blocks of a pair, up to 32, are held one per lane as the
  // address of the block's tiles, and each lane issues its own block's copy in turn.
  const uint8_t* src = nullptr;
  int turn = 0, run = 0;                                  // lane whose block is next, blocks held
  uint32_t put = ring_pos;
  auto issue = [&]() {
    if (to_load == 0) return;
    if (run == 0) {
      Cursor ld = cur[1];
      if (ld.b == ld.nb) cursor_next_pair(a, v, ld);
      turn = 0;
      run = min(min(32, to_load), ld.nb - ld.b);
      int blk = lane < run && ld.b + lane < a.bt_pitch
                    ? __ldg(a.block_tables + (size_t)ld.row * a.bt_pitch + ld.b + lane) : -1;
      if (blk < 0 || blk >= a.num_blocks) {
        if (lane < run) hy_flag(a.err, HY_ERR_BOUNDS);
        blk = 0;
      }
      src = a.cache + q4_tile(blk, ld.g, 0, a.kv_heads);
      ld.b += run;
      __syncwarp();                                       // cur[1] is read
      if (lane == 0) cur[1] = ld;
      __syncwarp();
    }
    const int n = min(2, run);
    if (lane == turn) mbar_arrive_expect_tx(&bars[put], n * BLK_BYTES);
    __syncwarp();
    if ((unsigned)(lane - turn) < (unsigned)n) {
      fence_proxy_async();
      bulk_load(ring_ptr + put * STAGE_BYTES + (lane - turn) * BLK_BYTES, src, BLK_BYTES, &bars[put]);
    }
    turn += n;
    run -= n;
    to_load -= n;
    put = put + 1 == NS ? 0 : put + 1;
  };
#pragma unroll 1
  for (int j = 0; j < NS; ++j) issue();

  // shared-memory offsets of this lane inside a block's tiles: its two K rows (the second
  // four keys on) and the first of its four V keys of either kind
  const int keyA = key_of(r >> 1, r & 1, 0);
  const uint32_t k_off = keyA * Q4_ROW_BYTES + 8 * c, p_off = Q4_PARAM_OFF + keyA * Q4_PARAM_BYTES;
  const uint32_t v_off0 = Q4_TILE_BYTES + key_of(c, 0, 0) * Q4_ROW_BYTES + 4 * r;
  const uint32_t v_off1 = Q4_TILE_BYTES + key_of(c, 1, 0) * Q4_ROW_BYTES + 4 * r;
  constexpr uint32_t ROW4 = 4 * Q4_ROW_BYTES, PAR4 = 4 * Q4_PARAM_BYTES;
  // column r of P^T: its key's weight where the row of the pair is the column's parity
  const uint32_t sel0 = r < 4 ? 0x4410u : 0x1044u, sel1 = r < 4 ? 0x4432u : 0x3244u;
  uint32_t get = ring_pos, par = ring_par;
  bool ok = true, first_pair = true;
  int pending = 0;
#pragma unroll 1
  while (left > 0) {
    const int n = min(left, cur[0].nb - cur[0].b);        // this pair's blocks in the range
    left -= n;
    // those that are full: the pair's last one may not be
    const int full = cur[0].b + n == cur[0].nb && (cur[0].kv_len & (HY_BLOCK - 1)) ? n - 1 : n;
    // Q in fp16 (q4_query_scale): lane (r, c) holds head r's words 2 c, 2 c + 1 (dimensions
    // 16 c ..) of both halves; rows 4-7 repeat rows 0-3.  Codes in bits 0-3 meet 2^14 q, codes
    // in bits 4-7 2^10 q, so that a score comes out as 2^-10 code . q.
    uint32_t qb[2][2][4], qs = 0u;                        // qs: the operand of the sums of q
    float mult[2];                                        // scale to log2 units of heads 2 c + k
    {
      float x[32], amax = 0.f, down, up;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w[4] = {qraw[i].x, qraw[i].y, qraw[i].z, qraw[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
          x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmax3f(amax, fabsf(x[2 * i]), fabsf(x[2 * i + 1]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      q4_query_scale(amax, down, up);
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = (j & 1) ? 1024.f : 16384.f;     // after down: their product may overflow
          const __half2 h = __floats2half2_rn(x[8 * i + 2 * j] * down * f, x[8 * i + 2 * j + 1] * down * f);
          qb[i >> 1][i & 1][j] = q4_as_u32(h);
          const float2 back = __half22float2(h);          // what the product sees, times 2^-10
          sum[i >> 1] += (back.x + back.y) * ((j & 1) ? 0x1p-20f : 0x1p-24f);
        }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        sum[hf] += __shfl_xor_sync(0xffffffffu, sum[hf], 1);
        sum[hf] += __shfl_xor_sync(0xffffffffu, sum[hf], 2);
      }
      // times 2^8, the rest of what their 2^-10 is short of fp16's normal range: the minima
      // meet (hi, hi) in lanes c = 0 and (lo, lo) in lanes c = 1, and the result is taken
      // times 2^-8
      const __half2 hi = __floats2half2_rn(sum[0] * 256.f, sum[1] * 256.f);
      const float2 back = __half22float2(hi);
      const __half2 lo = __floats2half2_rn(sum[0] * 256.f - back.x, sum[1] * 256.f - back.y);
      qs = c == 0 ? q4_as_u32(hi) : c == 1 ? q4_as_u32(lo) : 0u;
      mult[0] = score_mult(a.scale_log2 * 1024.f, __shfl_sync(0xffffffffu, up, 8 * c));
      mult[1] = score_mult(a.scale_log2 * 1024.f, __shfl_sync(0xffffffffu, up, 8 * c + 4));
    }
    float o[4][4];                                        // O^T, in 2^-24 / vs (odd m-tiles 2^-20 / vs)
    float z[2][2] = {{0.f, 0.f}, {0.f, 0.f}};             // [half][k]: sum of p times V's minimum
    float m[2] = {-INFINITY, -INFINITY};                  // running maximum (log2 units)
    float thr[2] = {-INFINITY, -INFINITY};                // score at which it is raised
    float l[2] = {0.f, 0.f};                              // this lane's part of the sum
    __half2 vs1 = q4_as_half2(0x3c003c00u);               // (vs, 1)
    __half vcap = __ushort_as_half(0xbc00);               // the largest scale that vs fits: -1, none yet
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

#pragma unroll 1
    for (int i = 0; i < n; i += 2) {
      if (!__all_sync(0xffffffffu, mbar_try_wait(&bars[get], par)) &&
          !__all_sync(0xffffffffu, mbar_wait(&bars[get], par, a.err))) {
        ok = false;
        pending = left + n - i - to_load;                 // blocks not waited for
        break;
      }
      const uint32_t st = ring + get * STAGE_BYTES;
      const uint32_t k_at = st + k_off, p_at = st + p_off, v_at0 = st + v_off0, v_at1 = st + v_off1;
      float x[2][4];                                      // scores of (keyA, keyB) x 2 heads, per block
      uint2 va[2], vb[2];                                 // V's parameters of keyA, keyB
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        // S^T = K Q^T, one accumulator per half of the dimensions
        const uint32_t kb = k_at + b * BLK_BYTES, pb = p_at + b * BLK_BYTES;
        float sc[3][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const uint2 wa = lds64(kb + 32 * hf), wb = lds64(kb + 32 * hf + ROW4);
          uint32_t xa[4], xb[4];
          q4_bits(wa.x, xa);
          q4_bits(wb.x, xb);
          mma_f16_16816(sc[hf], xa[0], xb[0], xa[1], xb[1], qb[hf][0][0], qb[hf][0][1]);
          mma_f16_16816(sc[hf], xa[2], xb[2], xa[3], xb[3], qb[hf][0][2], qb[hf][0][3]);
          q4_bits(wa.y, xa);
          q4_bits(wb.y, xb);
          mma_f16_16816(sc[hf], xa[0], xb[0], xa[1], xb[1], qb[hf][1][0], qb[hf][1][1]);
          mma_f16_16816(sc[hf], xa[2], xb[2], xa[3], xb[3], qb[hf][1][2], qb[hf][1][3]);
        }
        const uint2 pa = lds64(pb), pc = lds64(pb + PAR4);
        mma_f16_16816(sc[2], __byte_perm(pa.x, pa.y, 0x7632), __byte_perm(pc.x, pc.y, 0x7632), 0u, 0u, qs, 0u);
        const float a0 = __low2float(q4_as_half2(pa.x)), a1 = __low2float(q4_as_half2(pa.y));
        const float c0 = __low2float(q4_as_half2(pc.x)), c1 = __low2float(q4_as_half2(pc.y));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[b][e] = fmaf(a0, sc[0][e], fmaf(a1, sc[1][e], 0x1p-8f * sc[2][e]));
          x[b][2 + e] = fmaf(c0, sc[0][2 + e], fmaf(c1, sc[1][2 + e], 0x1p-8f * sc[2][2 + e]));
        }
        va[b] = lds64(pb + Q4_TILE_BYTES);
        vb[b] = lds64(pb + Q4_TILE_BYTES + PAR4);
      }
      if (i + 2 > full) {                                 // keys past the end: their rows hold anything
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int keys = i + b < full ? HY_BLOCK : i + b < n ? cur[0].kv_len & (HY_BLOCK - 1) : 0;
          if (keyA >= keys) { x[b][0] = x[b][1] = -INFINITY; va[b] = make_uint2(0u, 0u); }
          if (keyA + 4 >= keys) { x[b][2] = x[b][3] = -INFINITY; vb[b] = make_uint2(0u, 0u); }
        }
      }
      float mx[2] = {fmax3f(x[0][0], x[0][2], fmaxf(x[1][0], x[1][2])),
                     fmax3f(x[0][1], x[0][3], fmaxf(x[1][1], x[1][3]))};
      const __half2 smax2 = __hmax2(
          __hmax2(__hmax2(q4_as_half2(va[0].x), q4_as_half2(va[0].y)), __hmax2(q4_as_half2(vb[0].x), q4_as_half2(vb[0].y))),
          __hmax2(__hmax2(q4_as_half2(va[1].x), q4_as_half2(va[1].y)), __hmax2(q4_as_half2(vb[1].x), q4_as_half2(vb[1].y))));
      const bool grow = mx[0] > thr[0] || mx[1] > thr[1] || __hgt(__low2half(smax2), vcap);
      if (__any_sync(0xffffffffu, grow)) {
        const float smax = warp_max(__low2float(smax2));
        float vr = 1.f;                                   // change of vs
        if (smax > __half2float(vcap)) {                  // vs = 2^(6 - exponent), at most 2^15
          const int e = min(max((__float_as_int(smax) >> 23) & 255, 118), 254) - 127;
          const float vs = __int_as_float((6 - e + 127) << 23);
          vr = __half2float(vcap) < 0.f ? 1.f : vs * pow2_inverse(__low2float(vs1));
          vs1 = __floats2half2_rn(vs, 1.f);
          vcap = __float2half_rn(__int_as_float((e + 127) << 23) * 1.9990234375f);   // the last below 2^(e + 1)
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], d));
          const float m_mx = mx[e] * mult[e], m_new = fmaxf(m[e], m_mx);
          const float alpha = m_new == -INFINITY ? 1.f : ex2_ftz(m[e] - m_new);
          if (mx[e] > thr[e] || m_mx > m[e]) thr[e] = raise_above(mx[e], m_new, mult[e]);
          m[e] = m_new;
          l[e] *= alpha;
          z[0][e] *= alpha;
          z[1][e] *= alpha;
          const float ao = alpha * vr;
#pragma unroll
          for (int j = 0; j < 4; ++j) { o[j][e] *= ao; o[j][2 + e] *= ao; }
        }
      }
      float ms[2] = {m[0] == -INFINITY ? 0.f : -m[0], m[1] == -INFINITY ? 0.f : -m[1]};
      if (fmaxf(fabsf(ms[0]), fabsf(ms[1])) > FAR_LOG2) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (fabsf(ms[e]) > FAR_LOG2) {
            x[0][e] -= thr[e];
            x[0][2 + e] -= thr[e];
            x[1][e] -= thr[e];
            x[1][2 + e] -= thr[e];
            ms[e] = 0.f;
          }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[b][e] = ex2_ftz(fmaf(x[b][e], mult[e & 1], ms[e & 1]));
        l[0] += x[b][0] + x[b][2];
        l[1] += x[b][1] + x[b][3];
        const __half2 pa = __floats2half2_rn(x[b][0], x[b][1]), pc = __floats2half2_rn(x[b][2], x[b][3]);
        // O^T += V^T (scale P)^T, a half of the dimensions and 8 keys at a time.  A register
        // of V^T is what q4_bits leaves of a key's word: an even and the next odd
        // dimension, contracted together; the even one's outputs are columns 0-3, whose P
        // is 0 where the odd one's codes are, the odd one's columns 4-7 the other way
        // round.  Nibbles of equal weight share an m-tile (rows 0-7 nibble e, rows 8-15
        // nibble e + 2 of words 0-7).
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const __half2 ua = q4_as_half2(hf ? va[b].y : va[b].x), uc = q4_as_half2(hf ? vb[b].y : vb[b].x);
          const float na = __high2float(ua), nc = __high2float(uc);
          z[hf][0] = fmaf(x[b][0], na, fmaf(x[b][2], nc, z[hf][0]));
          z[hf][1] = fmaf(x[b][1], na, fmaf(x[b][3], nc, z[hf][1]));
          const uint32_t pt[2] = {
              movmatrix_trans(q4_as_u32(__hmul2(pa, __low2half2(__hmul2(ua, vs1))))),
              movmatrix_trans(q4_as_u32(__hmul2(pc, __low2half2(__hmul2(uc, vs1)))))};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t y0[4], y1[4];                        // keys of rows 2 c, 2 c + 1 (+ 8 h)
            q4_bits(lds32(v_at0 + b * BLK_BYTES + 32 * hf + ROW4 * h), y0);
            q4_bits(lds32(v_at1 + b * BLK_BYTES + 32 * hf + ROW4 * h), y1);
            const uint32_t p0 = __byte_perm(pt[h], 0u, sel0), p1 = __byte_perm(pt[h], 0u, sel1);
            mma_f16_16816(o[2 * hf], y0[0], y0[2], y1[0], y1[2], p0, p1);
            mma_f16_16816(o[2 * hf + 1], y0[1], y0[3], y1[1], y1[3], p0, p1);
          }
        }
      }
      if (++get == NS) {
        get = 0;
        par ^= 1u;
      }
      __syncwarp();                                       // the stage is read
      issue();
    }
    if (!ok) break;

    // the pair's result, or a partial of it
    Cursor k = cur[0];
    const bool whole = n == k.nb;
    const int slot = first_pair ? 0 : 1;
    float inv[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
        z[0][e] += __shfl_xor_sync(0xffffffffu, z[0][e], d);
        z[1][e] += __shfl_xor_sync(0xffffffffu, z[1][e], d);
      }
      inv[e] = whole ? 1.f / l[e] : 1.f;
    }
    const float per_vs = pow2_inverse(__low2float(vs1));
    const float unit0 = 0x1p24f * per_vs, unit1 = 0x1p20f * per_vs;   // m-tiles of bits 0-3, 4-7
    // lanes c < 2 hold the even dimensions of heads 2 c + k, lanes c + 2 the odd ones; the
    // former take the odd ones of k = 0, the latter the even ones of k = 1
    const bool odd = c >= 2;
    const int head = 2 * (c & 1) + odd;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {                       // nibble i: m-tile 2 hf + i % 2, row group i / 2
        float u[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
          u[k] = fmaf(o[2 * hf + (i & 1)][2 * (i >> 1) + k], (i & 1) ? unit1 : unit0, z[hf][k]) * inv[k];
        const float got = __shfl_xor_sync(0xffffffffu, odd ? u[0] : u[1], 2);
        y[2 * i] = odd ? got : u[0];
        y[2 * i + 1] = odd ? u[1] : got;
      }
      const int at = head * HY_HEAD_DIM + 64 * hf + 8 * r;
      if (whole) {
        *reinterpret_cast<uint4*>(a.out + ((size_t)k.tok * a.q_heads + k.g * HY_GROUP) * HY_HEAD_DIM + at) =
            make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
      } else {
        float4* p4 = reinterpret_cast<float4*>(part + slot * PART_FLOATS + at);
        p4[0] = make_float4(y[0], y[1], y[2], y[3]);
        p4[1] = make_float4(y[4], y[5], y[6], y[7]);
      }
    }
    if (!whole && r == 0)
      *reinterpret_cast<float2*>(part + slot * PART_FLOATS + HY_GROUP * HY_HEAD_DIM + 2 * head) =
          make_float2(odd ? m[1] : m[0], odd ? l[1] : l[0]);
    if (!whole && lane == 0)
      parts[slot] = Part{k.seq * a.kv_heads + k.g, n, k.nb, k.first * a.kv_heads + k.g * k.nb, k.tok};
    first_pair = false;
    if (left > 0) {
      cursor_next_pair(a, v, k);
      __syncwarp();                                       // cur[0] is read
      if (lane == 0) cur[0] = k;
      __syncwarp();
      load_q();
    }
  }
  if (!ok && pending > 0) {                               // copies in flight land before the CTA exits
    do {
      mbar_wait(&bars[get], par, nullptr);
      if (++get == NS) {
        get = 0;
        par ^= 1u;
      }
    } while (get != put);
  }
  ring_pos = get;
  ring_par = par;
  return ok;
}

struct Units {            // `total` blocks in n units whose sizes differ by at most one
  int n, size, more;      // the first `more` units have size + 1 blocks
  HY_DEVICE Units(int total, int units) : n(units), size(total / units), more(total - size * units) {}
  HY_DEVICE int start(int u) const { return u * size + min(u, more); }
  HY_DEVICE int of(int f) const {                         // the unit that holds block f
    return f < more * (size + 1) ? f / (size + 1) : more + (f - more * (size + 1)) / size;
  }
};

// The CTA runs the key blocks of one unit: its warps take equal parts, then merge, a head
// each, every pair that no warp finished alone.  A pair that reaches out of the unit (its
// first or last) leaves one partial in the workspace (slot 2 unit, or 2 unit + 1 where the
// pair starts inside the unit), and the CTA whose count of blocks completes a pair joins
// its partials, in their order whoever comes last.  Returns false if a wait ran out.
// alone: the unit is the n blocks of one pair, k; else blocks f0 .. f0 + n - 1.
HY_DEVICE bool decode_unit(const Args& a, const PlanView& v, const Units& units, int unit, bool alone,
                           Cursor k, int f0, int n, const SeqInfo& top, uint8_t* payload, Shared& sh,
                           uint32_t& ring_pos, uint32_t& ring_par) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* parts = reinterpret_cast<float*>(payload + NW * RING_BYTES);
  if (lane < 2) sh.part[2 * warp + lane].pair = -1;
  const int per = n / NW, more = n - per * NW;            // the first `more` warps take one more
  const int at = warp * per + min(warp, more), count = per + (warp < more);
  if (alone) k.b = at;
  else if (count > 0) k = cursor_at(a, v, top, f0 + at);
  if (lane < 2) sh.cur[warp][lane] = k;
  __syncwarp();
  const bool ok = decode_warp(a, v, sh.cur[warp], count, payload + warp * RING_BYTES,
                              parts + warp * 2 * PART_FLOATS, sh.part + 2 * warp, sh.bar[warp],
                              ring_pos, ring_par);
  if (__syncthreads_or(!ok)) return false;

  // Lane j of every warp looks after part j: parts of one pair are neighbours (but for
  // empty ones between them).  Warps 4 i + h, i = 0..3, take head h of every fourth pair.
  static_assert(2 * NW == 32 && NW == 4 * HY_GROUP, "one part per lane, four warps per head");
  const int head = warp & 3;
  const int my_pair = sh.part[lane].pair, my_blocks = sh.part[lane].blocks;
  const float2 ml = my_pair < 0 ? make_float2(-INFINITY, 0.f)
                                  : *reinterpret_cast<const float2*>(
                                        parts + lane * PART_FLOATS + HY_GROUP * HY_HEAD_DIM + 2 * head);
  unsigned todo = __ballot_sync(0xffffffffu, my_pair >= 0);
  int open_at[2], open_blocks[2], n_open = 0;             // pairs that reach out: first part, blocks here
  for (int turn = 0; todo; ++turn) {
    const int i = __ffs(todo) - 1;
    const Part& part = sh.part[i];                        // its pair, number of blocks, query row
    const int pair = part.pair, nb = part.nb;
    const bool in = my_pair == pair;
    const unsigned group = __ballot_sync(0xffffffffu, in);
    todo &= ~group;
    const int blocks = __reduce_add_sync(0xffffffffu, in ? my_blocks : 0);
    if (blocks != nb) {
      open_at[n_open & 1] = i;
      open_blocks[n_open & 1] = blocks;
      ++n_open;
    }
    if ((turn & 3) != (warp >> 2)) continue;              // warp-uniform
    const float M = warp_max(in ? ml.x : -INFINITY);
    const float wt = in ? ex2_ftz(ml.x - (M == -INFINITY ? 0.f : M)) : 0.f;
    float L = wt * ml.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (unsigned g = group; g;) {                        // four parts in flight
      float w[4];
      float4 p[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int j = g ? __ffs(g) - 1 : i;
        w[t] = g ? __shfl_sync(0xffffffffu, wt, j) : 0.f;
        p[t] = *reinterpret_cast<const float4*>(parts + j * PART_FLOATS + head * HY_HEAD_DIM + 4 * lane);
        g &= g - 1;
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        acc.x = fmaf(w[t], p[t].x, acc.x);
        acc.y = fmaf(w[t], p[t].y, acc.y);
        acc.z = fmaf(w[t], p[t].z, acc.z);
        acc.w = fmaf(w[t], p[t].w, acc.w);
      }
    }
    const int seq = pair / a.kv_heads, g = pair - seq * a.kv_heads;
    if (blocks == nb) {
      const float inv = __fdividef(1.f, L);
      *reinterpret_cast<uint2*>(a.out + ((size_t)part.tok * a.q_heads + g * HY_GROUP + head) * HY_HEAD_DIM + 4 * lane) =
          make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
    } else {
      const size_t slot = 2 * unit + (part.first > f0);
      __stcg(reinterpret_cast<float4*>(v.part_o + (slot * HY_GROUP + head) * HY_HEAD_DIM) + lane, acc);
      if (lane == 0) __stcg(v.part_ml + slot * HY_GROUP + head, make_float2(M, L));
    }
  }
  if (n_open == 0) {
    __syncthreads();                                      // parts are read
    return true;
  }
  __syncthreads();
  if (warp == 0) {
    __threadfence();                                      // this CTA's partials, before the count
    bool mine_last = false;
    if (lane < n_open) {
      const int mine_blocks = lane == 0 ? open_blocks[0] : open_blocks[1];
      const Part& p = sh.part[lane == 0 ? open_at[0] : open_at[1]];
      int* ctr = &v.counters[p.pair];
      mine_last = atomicAdd(ctr, mine_blocks) + mine_blocks == p.nb;
      if (mine_last) *ctr = 0;                            // for the next launch on this plan
    }
    sh.last = (int)__ballot_sync(0xffffffffu, mine_last);
    __threadfence();                                      // the others' partials, after the count
  } else if (warp == 1 && lane < n_open) {                // meanwhile, should this CTA be the last
    const Part& p = sh.part[lane == 0 ? open_at[0] : open_at[1]];
    const int u0 = units.of(p.first);
    sh.join[lane] = Join{u0, units.of(p.first + p.nb - 1), p.first > units.start(u0),
                         p.tok * a.q_heads + p.pair % a.kv_heads * HY_GROUP};
  }
  __syncthreads();
  const int last = sh.last;
  if (last == 0) return true;
  for (int j = 0; j < n_open; ++j) {
    if (!((last >> j) & 1)) continue;
    // warps 4 i + h, i = 0..3, take every fourth partial's head h, one float4 per lane
    const Join at = sh.join[j];
    const int u0 = at.u0, u1 = at.u1, quarter = warp >> 2;
    auto slot = [&](int u) { return (size_t)(2 * u + (u == u0 ? at.inside : 0)); };
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = u0 + quarter; c0 <= u1; c0 += 128) {    // 32 partials (none is empty), one weight per lane
      const int cnt = min(32, (u1 - c0) / 4 + 1);
      float4 po[8];                                       // 8 partials in flight, beside the weights
      auto load8 = [&](int i) {
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (i + t < cnt)
            po[t] = __ldcg(reinterpret_cast<const float4*>(
                               v.part_o + (slot(c0 + 4 * (i + t)) * HY_GROUP + head) * HY_HEAD_DIM) + lane);
          else po[t] = make_float4(0.f, 0.f, 0.f, 0.f);
      };
      load8(0);
      const float2 e = lane < cnt ? __ldcg(v.part_ml + slot(c0 + 4 * lane) * HY_GROUP + head)
                                  : make_float2(-INFINITY, 0.f);
      const float m_new = warp_max(fmaxf(M, e.x));
      const float mu = m_new == -INFINITY ? 0.f : m_new, old = ex2_ftz(M - mu);
      const float w = ex2_ftz(e.x - mu);
      float lw = w * e.y;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, o);
      L = fmaf(L, old, lw);
      acc = make_float4(acc.x * old, acc.y * old, acc.z * old, acc.w * old);
      for (int i = 0; i < cnt; i += 8) {
        if (i > 0) load8(i);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float wt = __shfl_sync(0xffffffffu, w, (i + t) & 31);
          acc.x = fmaf(wt, po[t].x, acc.x);
          acc.y = fmaf(wt, po[t].y, acc.y);
          acc.z = fmaf(wt, po[t].z, acc.z);
          acc.w = fmaf(wt, po[t].w, acc.w);
        }
      }
      M = m_new;
    }
    // the four quarters, through shared memory (the warps' parts are read)
    float* mine4 = parts + (quarter * HY_GROUP + head) * (HY_HEAD_DIM + 4);
    *reinterpret_cast<float4*>(mine4 + 4 * lane) = acc;
    if (lane == 0) *reinterpret_cast<float2*>(mine4 + HY_HEAD_DIM) = make_float2(M, L);
    __syncthreads();
    if (quarter == 0) {
      float mm[4], ll[4], m_all = -INFINITY, sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float2 e = *reinterpret_cast<const float2*>(parts + (t * HY_GROUP + head) * (HY_HEAD_DIM + 4) + HY_HEAD_DIM);
        mm[t] = e.x;
        ll[t] = e.y;
        m_all = fmaxf(m_all, e.x);
      }
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float w = ex2_ftz(mm[t] - (m_all == -INFINITY ? 0.f : m_all));
        const float4 x = *reinterpret_cast<const float4*>(parts + (t * HY_GROUP + head) * (HY_HEAD_DIM + 4) + 4 * lane);
        sum = fmaf(w, ll[t], sum);
        o.x = fmaf(w, x.x, o.x);
        o.y = fmaf(w, x.y, o.y);
        o.z = fmaf(w, x.z, o.z);
        o.w = fmaf(w, x.w, o.w);
      }
      const float inv = __fdividef(1.f, sum);
      *reinterpret_cast<uint2*>(a.out + (size_t)(at.row + head) * HY_HEAD_DIM + 4 * lane) =
          make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
    }
    if (j == 0 && n_open > 1) __syncthreads();            // before the next pair's quarters
  }
  __syncthreads();                                        // sh.part is read
  return true;
}

// ------------------------------------------------------------------ prefill item
HY_DEVICE PreItem pre_item_geom(const Args& a, const PlanView& v, int item) {
  const int4 it = v.pre_sorted[item];
  PreItem p;
  p.seq = it.x;
  p.g = it.y;
  p.t0 = it.z;
  p.w = it.w;
  const int4 s = v.seqs[p.seq];
  p.row0 = s.y;
  const int q_len = v.seqs[p.seq + 1].y - p.row0;
  p.prefix = s.z - q_len;
  p.nrows = min(PRE_QROWS, q_len - p.t0);
  p.kv_end = p.prefix + p.t0 + p.nrows;                   // keys its last row sees
  pre_piece_range(p.w, (p.kv_end + PRE_KEYS - 1) / PRE_KEYS, p.tlo, p.thi);
  // a sequence longer than its block-table row: no tiles past the row (but one at least,
  // which the roles count on)
  const long row_tiles = ((long)a.bt_pitch * HY_BLOCK + PRE_KEYS - 1) / PRE_KEYS;
  if (p.thi > row_tiles) {
    hy_flag(a.err, HY_ERR_BOUNDS);
    p.thi = (int)max(row_tiles, 1L);
    p.tlo = min(p.tlo, p.thi - 1);
  }
  return p;
}

// Expanding warps: thread t of 128 takes row t % 64 of every key tile's K (t < 64) or
// V: its 64 code bytes and parameters from global memory, the next tile's loaded
// ahead, to 256 bytes of fp16 in the ring.  Rows past the item's keys become zeros:
// their scores are masked, and a zero weight times a zero adds nothing.  A half of V
// whose parameters are NaN (its codes are 0 then) is expanded to fp16's lowest number, so
// that a later token's does not reach the rows that do not see it; its key is noted, and
// the softmax warps write NaN where a row does see it.  (16 chunks of 512 tokens, when it
// was added: 393 us with this, 389 without; zeroing the half in a branch before it is
// expanded, 402.)
constexpr uint32_t VALUE_LEAST = 0xfbff0000u;             // parameters are at least (0, -65504)
constexpr uint32_t KEY_LEAST = 0x7fff7fffu;               // NaN: whatever they are
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
HY_DEVICE void expand_row(const RowCodes& x, uint8_t* slot, int key, uint32_t at_least) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const __half2 sm = __hmax2(q4_as_half2(x.par[half]), q4_as_half2(at_least));
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

// 64 columns of O become NaN in the lanes that say so (the whole warp takes part).
HY_DEVICE void nan_half(uint32_t t, bool on) {
#pragma unroll 1
  for (int i = 0; i < 64; i += 16) {
    float o[16];
    tmem_ld16(t + i, o);
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = on ? __int_as_float(0x7fffffff) : o[k];
    tmem_st16(t + i, o);
  }
  tmem_wait_st();
}

// The CTA's prefill items, taken from the counter `next` until there are no more.  Each
// role runs through the items at its own pace, ahead of the others as far as the
// barriers let it: the expanding warps fill the ring for the next item, whose Q is
// loaded as soon as the last score tile of this one is done, while the softmax warps
// write this one's output.
// The products, barriers and softmax follow attention.cu's prefill: S(t + 1) is issued
// while the softmax works on S(t); the softmax writes P(t) over S(t) and waits for
// P V(t - 1) only to rescale O.  c counts key tiles, n items, over the launch.
// Returns false if a wait ran out; the roles then drain what they issued.
__device__ bool prefill_all(const CUtensorMap* q_map, const Args& a, const PlanView& v, int n_pre,
                            int* next, uint8_t* payload, Shared& sh, uint32_t tmem) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t sbase = smem_u32(payload);
  bool ok = true;
  uint32_t c0 = 0;
  // the CTA's item n, for a whole warp
  auto item_at = [&](uint32_t n) {
    PreItem p;
    ok = __all_sync(0xffffffffu, mbar_wait(&sh.itemfull, n & 1, a.err));
    p = sh.item[n & 1];
    if (!ok) p.seq = -1;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.itemfree);
    return p;
  };

  if (warp == ITEM_WARP) {
    if (lane == 0) {
      for (uint32_t n = 0; ok; ++n) {
        // an item is taken when the loads of the last one are over, not before: others
        // may be free for it
        if (n > 0) ok = mbar_wait(&sh.expdone, (n - 1) & 1, a.err);
        if (!ok) break;
        const int k = atomicAdd(next, 1);
        PreItem N;
        if (k < n_pre) N = pre_item_geom(a, v, k);
        else N.seq = -1;
        if (n > 0) ok = mbar_wait(&sh.itemfree, (n - 1) & 1, a.err);
        if (!ok) break;
        sh.item[n & 1] = N;
        sh.nan_at[n & 1][0] = sh.nan_at[n & 1][1] = INT_MAX;
        mbar_arrive(&sh.itemfull);
        if (N.seq < 0) break;
        if (n > 0) ok = mbar_wait(&sh.qfree, (n - 1) & 1, a.err);
        if (!ok) break;
        fence_proxy_async();
        mbar_arrive_expect_tx(&sh.qraw, 2 * Q_BYTES);
        for (int X = 0; X < 2; ++X)
          tma_load_4d(payload + X * Q_BYTES, q_map, 0, N.row0 + N.t0, N.g * HY_GROUP + 2 * X, 0, &sh.qraw);
        ok = mbar_wait(&sh.qraw, n & 1, a.err);           // landed before this warp can leave
      }
    }
    __syncwarp();
  } else if (warp >= EXP_WARP && warp < MMA_WARP) {
    const int t128 = tid - EXP_WARP * 32, part = t128 >> 6, key = t128 & 63;
    uint8_t* ring = payload + (part ? V_OFF : K_OFF);
    for (uint32_t n = 0; ok; ++n) {
      const PreItem P = item_at(n);
      if (P.seq < 0) break;
      const int ntiles = P.thi - P.tlo;
      const int32_t* bt = a.block_tables + (size_t)(a.seq_bt_row ? a.seq_bt_row[P.seq] : P.seq) * a.bt_pitch;
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
        if (t == ntiles - 1 && lane == 0) mbar_arrive(&sh.expdone);
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.free_[slot], ((c / PS) & 1) ^ 1, a.err));
        if (!ok) break;
        expand_row(cur, ring + slot * KV_BYTES, key, part ? VALUE_LEAST : KEY_LEAST);
        // a minimum of NaN: above the scale's 16 bits, an exponent of ones and a mantissa
        if (max(cur.par[0] << 1, cur.par[1] << 1) >= 0xf8020000u && part) {
          for (int half = 0; half < 2; ++half)
            if ((half ? cur.par[1] : cur.par[0]) << 1 >= 0xf8020000u)
              atomicMin(&sh.nan_at[n & 1][half], pos - PRE_KEYS);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.full[slot]);
      }
      c0 += ntiles;
    }
  } else if (warp == MMA_WARP || warp == MMA_WARP + 1) {
    const int X = warp - MMA_WARP;
    constexpr uint32_t ID_S = tc_idesc_f16(128, PRE_KEYS, false);
    constexpr uint32_t ID_O = tc_idesc_f16(128, HY_HEAD_DIM, true);
    const uint64_t dQ = tc_desc_sw128(sbase + X * Q_BYTES, 16, 1024);
    for (uint32_t n = 0; ok; ++n) {
      const PreItem P = item_at(n);
      if (P.seq < 0) break;
      const int ntiles = P.thi - P.tlo;
      if (lane == 0) {
        ok = mbar_wait(&sh.qfull, n & 1, a.err);
        for (int t = 0; t <= ntiles && ok; ++t) {
          if (t < ntiles) {                               // S_X(t) = Q_X K_t^T
            const uint32_t c = c0 + t, slot = c % PS;
            ok = mbar_wait(&sh.full[slot], (c / PS) & 1, a.err);
            // S(t) goes over P(t - 2): products of different shapes are not ordered among
            // themselves, so the one that reads it is waited for (it was issued a softmax
            // tile ago; the wait also tells the softmax, which waits for S(t), that it is done)
            if (ok && c > 1) ok = mbar_wait(&sh.odone[X][c & 1], ((c - 2) >> 1) & 1, a.err);
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
            if (t == ntiles - 1) tc_commit(&sh.qfree);
          }
          if (t > 0) {                                    // O_X += P_X(t - 1) V_{t-1}
            const uint32_t c = c0 + t - 1, slot = c % PS;
            ok = mbar_wait(&sh.pfull[X][c & 1], (c >> 1) & 1, a.err);
            if (ok && t == 1 && n > 0) ok = mbar_wait(&sh.ofree[X], (n - 1) & 1, a.err);
            if (!ok) break;
            tc_fence_after();
            const uint64_t dV = tc_desc_sw128(sbase + V_OFF + slot * KV_BYTES, KV_BYTES / 2, 1024);
#pragma unroll
            for (int kk = 0; kk < PRE_KEYS / 16; ++kk)
              tc_mma_bf16_ta(tmem + TM_O + 128 * X, tmem + tm_s(X, c & 1) + 8 * kk,
                             dV + (uint64_t)((kk * 2048) >> 4), ID_O, (t > 1 || kk > 0));
            tc_commit(&sh.odone[X][c & 1]);
            tc_commit(&sh.free_[slot]);
          }
        }
        if (!ok) {                                        // let every issued product finish
          tc_commit(&sh.drain[X]);
          mbar_wait(&sh.drain[X], 0, nullptr);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      c0 += ntiles;
    }
  } else if (warp < EXP_WARP) {                           // softmax: thread = row = TMEM lane
    const int X = warp >> 2, r = (warp & 3) * 32 + lane, j = r & 63;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_base + TM_O + 128 * X;
    uint8_t* q_row = payload + X * Q_BYTES + r * 128;
    for (uint32_t n = 0;; ++n) {
      PreItem P = {};
      if (ok) P = item_at(n);
      if (ok && P.seq >= 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh.qraw, n & 1, a.err));
      // the softmax warps leave together: pieces of an item meet at a barrier of theirs
      if (named_sync_or(PRE_PIECE_BAR, PRE_ROWS, !ok)) ok = false;
      if (!ok || P.seq < 0) break;
      const int ntiles = P.thi - P.tlo;
      // Q row r to fp16 in place (q4_query_scale)
      float sl2;                                          // scale to log2 units of this row
      {
        float amax = 0.f, down, up;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint4 u = *reinterpret_cast<const uint4*>(q_row + (i >> 3) * (Q_BYTES / 2) + (((i & 7) ^ (r & 7)) << 4));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            amax = fmax3f(amax, fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xffff0000u)));
        }
        q4_query_scale(amax, down, up);
        sl2 = score_mult(a.scale_log2, up);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          uint4* at = reinterpret_cast<uint4*>(q_row + (i >> 3) * (Q_BYTES / 2) + (((i & 7) ^ (r & 7)) << 4));
          const uint4 u = *at;
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
          uint32_t y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            y[k] = q4_as_u32(__floats2half2_rn(__uint_as_float(w[k] << 16) * down,
                                               __uint_as_float(w[k] & 0xffff0000u) * down));
          *at = make_uint4(y[0], y[1], y[2], y[3]);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.qfull);
      }
      const int lim = min(P.prefix + P.t0 + j, P.kv_end - 1);   // last key row r may see
      float m = NEG_INF, l = 0.f;                         // m in scaled log2 units
      float thr = NEG_INF;                                // score above which it is raised
      for (int t = 0; t < ntiles; ++t) {
        const uint32_t c = c0 + t;
        const uint32_t tS = tmem + lane_base + tm_s(X, c & 1);
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.sfull[X][c & 1], (c >> 1) & 1, a.err));
        if (!ok) break;
        tc_fence_after();
        float s[64];
        float (&s_lo)[32] = *reinterpret_cast<float(*)[32]>(&s[0]);
        float (&s_hi)[32] = *reinterpret_cast<float(*)[32]>(&s[32]);
        tmem_ld32(tS, s_lo);
        tmem_ld32(tS + 32, s_hi);
        tmem_wait_ld(s_lo);
        tmem_wait_ld(s_hi);
        const int kb = (P.tlo + t) * PRE_KEYS;
        if (kb + PRE_KEYS - 1 > P.prefix + P.t0) {        // the tile reaches the diagonal or the end
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (kb + i > lim) s[i] = NEG_INF;
        }
        float mxs[8];                                     // 8 independent chains
#pragma unroll
        for (int k = 0; k < 8; ++k) mxs[k] = fmax3f(s[k], s[8 + k], s[16 + k]);
#pragma unroll
        for (int i = 24; i < 56; i += 16)
#pragma unroll
          for (int k = 0; k < 8; ++k) mxs[k] = fmax3f(mxs[k], s[i + k], s[i + 8 + k]);
#pragma unroll
        for (int k = 0; k < 8; ++k) mxs[k] = fmaxf(mxs[k], s[56 + k]);
        const float mx = fmax3f(fmax3f(mxs[0], mxs[1], mxs[2]), fmax3f(mxs[3], mxs[4], mxs[5]),
                                fmaxf(mxs[6], mxs[7]));
        const bool grow = mx > thr;
        if (__any_sync(0xffffffffu, grow)) {
          const float mnew = grow ? mx * sl2 : m;
          const float alpha = mnew == NEG_INF ? 1.f : ex2_ftz(m - mnew);
          l *= alpha;
          m = mnew;
          if (grow) thr = raise_above(mx, m, sl2);
          if (t > 0) {                                    // O holds tiles < t: wait for P V(t - 1)
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.odone[X][(c & 1) ^ 1], ((c - 1) >> 1) & 1, a.err));
            tc_fence_after();
#pragma unroll 1
            for (int cc = 0; cc < 8; ++cc) {
              float o[16];
              tmem_ld16(tO + 16 * cc, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= alpha;
              tmem_st16(tO + 16 * cc, o);
            }
            tmem_wait_st();
            if (!ok) break;
          }
        }
        float mneg = (m == NEG_INF) ? 0.f : -m;
        if (__any_sync(0xffffffffu, fabsf(mneg) > FAR_LOG2)) {
          const float off = fabsf(mneg) > FAR_LOG2 ? thr : 0.f;
#pragma unroll
          for (int i = 0; i < 64; ++i) s[i] -= off;
          mneg = fabsf(mneg) > FAR_LOG2 ? 0.f : mneg;
        }
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
        tmem_st32u(tS, pk);                               // P(t) over the first 32 columns of S(t)
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.pfull[X][c & 1]);
      }
      c0 += ntiles;
      if (ok) {                                           // epilogue: O_X complete
        const uint32_t c = c0 - 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.odone[X][c & 1], (c >> 1) & 1, a.err));
        tc_fence_after();
        for (int half = 0; half < 2; ++half)
          if (__any_sync(0xffffffffu, sh.nan_at[n & 1][half] <= lim))
            nan_half(tO + 64 * half, sh.nan_at[n & 1][half] <= lim);
      }
      // read again rather than held in registers over the tiles: no item takes the place
      // before these warps have read the next one
      const PreItem& E = sh.item[n & 1];
      const bool store = ok && j < E.nrows;               // rows past the chunk hold other tokens' Q
      __nv_bfloat16* op = a.out + ((size_t)(E.row0 + E.t0 + j) * a.q_heads + E.g * HY_GROUP + 2 * X + (r >> 6)) *
                                      HY_HEAD_DIM;
      const int piece = E.w;
      if (piece != 0) {                                   // a piece: every softmax thread takes part
        ok = prefill_piece_finish(v, piece, X * 128 + r, tO, m, l, ok, store ? op : nullptr, sh.pre_last);
      } else if (ok) {
        const float inv = 1.f / l;
#pragma unroll 1
        for (int cc = 0; cc < 4; ++cc) {
          float o[32];
          tmem_ld32(tO + 32 * cc, o);                     // warp-collective: every lane loads
          tmem_wait_ld(o);
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
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.ofree[X]);
    }
  }
  tc_fence_before();
  return !__syncthreads_or(!ok);
}

// The decode sequences of a step with prefill items: their key blocks in even shares that
// CTAs take as they become free (as many as plan_sides says; a share costs about 8 us
// beside its blocks: 4 chunks and 128 decodes took 135 us with a share per CTA, 145 with
// two smaller ones and 154 with three, all on one build).  Returns false if a wait ran out.
__device__ bool decode_shares(const Args& a, const PlanView& v, int shares, int blocks, uint8_t* payload,
                              Shared& sh) {
  uint32_t ring_pos = 0, ring_par = 0;
  const int total = blocks * a.kv_heads;                  // below 2^31: the host checks the tables' size
  if (total == 0) return true;
  const Units units(total, shares);
  int* grab = v.grab + HY_GRAB_INTS * (a.layer & 63);
  for (;;) {
    if (threadIdx.x == 0) sh.unit = atomicAdd(&grab[0], 1);
    __syncthreads();
    const int u = sh.unit;
    __syncthreads();
    if (u >= units.n) return true;
    const int f0 = units.start(u);
    if (!decode_unit(a, v, units, u, false, Cursor{}, f0, units.start(u + 1) - f0, seq_top(a, v), payload,
                     sh, ring_pos, ring_par))
      return false;
  }
}

// The sequence of query row `tok`: the last that starts at or before it.
HY_DEVICE int seq_of_row(const Args& a, const PlanView& v, int tok) {
  int lo = 0, hi = a.num_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v.seqs[mid].y <= tok) lo = mid; else hi = mid;
  }
  return lo;
}

// Steps that may hold prefill chunks (more query rows than sequences).
__global__ void __launch_bounds__(NT, 1) attn_q4_kernel(const __grid_constant__ CUtensorMap q_map,
                                                          Args a, PlanView v) {
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
        mbar_init(&sh.odone[x][b], 1);
      }
      mbar_init(&sh.drain[x], 1);
      mbar_init(&sh.ofree[x], EXP_WARP / 2);
    }
    mbar_init(&sh.qraw, 1);
    mbar_init(&sh.qfull, EXP_WARP);
    mbar_init(&sh.qfree, 2);
    mbar_init(&sh.itemfull, 1);
    mbar_init(&sh.itemfree, ITEM_READERS);
    mbar_init(&sh.expdone, MMA_WARP - EXP_WARP);
    fence_mbar_init();
  }
  __syncthreads();
  hy_grid_wait();
  hy_grid_trigger();
  const HyPlan plan = load_plan(a, v);
  if (plan.work <= 0 && plan.blocks == 0) return;         // every CTA: no counter is touched
  int* grab = v.grab + HY_GRAB_INTS * (a.layer & 63);
  bool ok = true;
  if ((int)blockIdx.x < plan.pre_ctas) {                     // these CTAs take prefill items
    if (warp == 0) {
      tmem_alloc(&sh.tmem_base, TMEM_COLS);
      tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem_base;
    ok = prefill_all(&q_map, a, v, plan.work, &grab[2], payload, sh, tmem);
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      tmem_dealloc(tmem, TMEM_COLS);
    }
  }
  if (ok) decode_shares(a, v, plan.shares, plan.blocks, payload, sh);
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();                                      // the last CTA out resets the counters
    if (atomicAdd(&grab[1], 1) == (int)gridDim.x - 1) {
      atomicExch(&grab[0], 0);
      atomicExch(&grab[2], 0);
      atomicExch(&grab[1], 0);
    }
  }
}

// Steps of no more query rows than sequences, which are decode steps but for sequences
// without a token: without the prefill's code a launch takes 2 us less (one sequence of 600
// keys 8.9 us, 11.1 by the other kernel, one of 40960 19.9 and 22.3).  The key blocks are
// dealt evenly over the CTAs; a small step's pairs (the plan's choice) go one to a CTA,
// which merges them in shared memory, unless there are at most 16, of more than 64 blocks
// on average over all sequences, those without a token included (8 pairs of 64 / 96 / 128
// blocks dealt 8.8 / 9.1 / 9.4 us, a CTA each 9.8 / 11.7 / 13.5; 16 of 64 / 128 9.6 / 10.7
// and 9.8 / 13.5; 32 of 128 13.9 and 13.7; 80 of 38 13.7 and 9.3).  The average overlooks
// a long sequence beside a short one: 8 pairs of 120 blocks and 8 of 1 take 13.3, 9.1 if
// dealt.  Rows of longer chunks that such a step may hold all the same are taken one (row,
// head) at a time, a CTA each.
__global__ void __launch_bounds__(NT, 1) attn_q4_decode_kernel(Args a, PlanView v) {
  __shared__ Shared sh;
  extern __shared__ uint8_t dyn_smem[];
  uint8_t* payload = dyn_smem + ((1024u - (smem_u32(dyn_smem) & 1023u)) & 1023u);
  if (threadIdx.x < NW * NS) {
    mbar_init(&sh.bar[0][0] + threadIdx.x, 1);
    fence_mbar_init();
  }
  __syncthreads();
  hy_grid_wait();
  hy_grid_trigger();
  const SeqInfo top = seq_top(a, v);                      // with the header: needed by most steps
  const HyPlan plan = load_plan(a, v);
  int n_pairs = max(-plan.work, 0);
  const int total = plan.blocks * a.kv_heads;             // below 2^31, see decode_shares
  if (n_pairs <= 16 && total > 64 * n_pairs) n_pairs = 0;       // few, not short: dealt after all
  uint32_t ring_pos = 0, ring_par = 0;
  const Units units(total, (int)gridDim.x);
  const int shares = n_pairs > 0 ? n_pairs : total > 0 ? units.n : 0;
  const long n = shares + (plan.work > 0 ? (long)plan.end_row * a.kv_heads : 0);
  for (long u = blockIdx.x; u < n; u += gridDim.x) {
    const bool alone = n_pairs > 0 || u >= shares;
    Cursor k = {};
    int f0 = 0, blocks;
    if (alone) {
      const int i = (int)(u < shares ? u : u - shares) / a.kv_heads;
      k.g = (int)(u < shares ? u : u - shares) - i * a.kv_heads;
      k.seq = u < shares ? i : seq_of_row(a, v, i);
      SeqInfo s = seq_info(a, v, k.seq);
      const int q_len = v.seqs[k.seq + 1].y - s.tok;
      bool take = q_len == 1;                             // (of a plan that fits)
      if (u >= shares) {                                  // row i, which sees kv_len - (rows after it) keys
        take = q_len > 1 && i >= s.tok;
        s.kv_len -= s.tok + q_len - 1 - i;
        s.tok = i;
      }
      if (take) cursor_sequence(a, k, s);
      blocks = take ? k.nb : 0;                           // the others are not this unit's
    } else {
      f0 = units.start((int)u);
      blocks = units.start((int)u + 1) - f0;
    }
    if (!decode_unit(a, v, units, (int)u, alone, k, f0, blocks, top, payload, sh, ring_pos, ring_par)) return;
  }
}

// ------------------------------------------------------------------ fp32 path
// fp32 throughout, for the parity engine.  A CTA takes one (query token, KV head): its
// four query heads share every key and value read (188 rows of 2 KV heads with 60 to 700
// keys: 17 us, bound by the instructions per value; a pair of dimensions shares most).  The
// warps take 32 keys at a time in turn: one key per lane for the scores (the whole 128-long product in a lane, no exchange
// between lanes), four dimensions per lane for the values; each keeps a running maximum
// and sum, merged at the end.
constexpr int F_WARPS = 8, F_KEYS = 32;
struct F32Shared {
  float q[HY_GROUP][HY_HEAD_DIM];
  float2 p[F_WARPS][F_KEYS][HY_GROUP];                    // weights of a warp's 32 keys, each twice
  float o[F_WARPS][HY_GROUP][HY_HEAD_DIM];
  float2 ml[F_WARPS][HY_GROUP];
};

__global__ void __launch_bounds__(F_WARPS * 32) attn_q4_fp32_kernel(
    const float* __restrict__ q, float* __restrict__ out, int tokens, int q_heads, int kv_heads,
    const uint8_t* __restrict__ cache_layer, int num_blocks,
    const int32_t* __restrict__ block_tables, int bt_pitch,
    const int32_t* __restrict__ seq_bt_row, const int32_t* __restrict__ cu_q,
    const int32_t* __restrict__ seq_lens_k, int S, float scale, int32_t* err) {
  __shared__ F32Shared sh;
  hy_grid_wait();
  hy_grid_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long total = (long)cu_q[S] * kv_heads;            // rows past the last sequence stay
  if (cu_q[0] < 0 || cu_q[S] > tokens) {                  // rows that q does not have
    if (tid == 0) hy_flag(err, HY_ERR_BOUNDS);
    return;
  }
  for (long u = blockIdx.x; u < total; u += gridDim.x) {
    const int row = (int)(u / kv_heads), g = (int)(u % kv_heads);
    int lo = 0, hi = S;                     // seq = last i with cu_q[i] <= row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu_q[mid] <= row) lo = mid; else hi = mid;
    }
    const int seq = lo;
    if (row < cu_q[seq]) continue;                        // before the first sequence
    const int prefix = seq_lens_k[seq] - (cu_q[seq + 1] - cu_q[seq]);
    const int key_end = prefix + (row - cu_q[seq]) + 1;
    if (prefix < 0 || (long)key_end > (long)bt_pitch * HY_BLOCK) {
      if (tid == 0) hy_flag(err, HY_ERR_BOUNDS);
      continue;
    }
    const int32_t* bt = block_tables + (size_t)(seq_bt_row ? seq_bt_row[seq] : seq) * bt_pitch;
    const size_t at = ((size_t)row * q_heads + g * HY_GROUP) * HY_HEAD_DIM;
    __syncthreads();                        // the last unit's merge is over
    if (tid < HY_GROUP * HY_HEAD_DIM / 4)
      reinterpret_cast<float4*>(sh.q)[tid] = reinterpret_cast<const float4*>(q + at)[tid];
    __syncthreads();
    float m[HY_GROUP], l[HY_GROUP];
    float2 acc[HY_GROUP][2];
#pragma unroll
    for (int h = 0; h < HY_GROUP; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
      acc[h][0] = acc[h][1] = make_float2(0.f, 0.f);
    }
    for (int k0 = warp * F_KEYS; k0 < key_end; k0 += F_WARPS * F_KEYS) {
      const int key = k0 + lane, cnt = min(F_KEYS, key_end - k0);
      int blk = lane < cnt ? bt[key / HY_BLOCK] : 0;
      if (blk < 0 || blk >= num_blocks) {
        hy_flag(err, HY_ERR_BOUNDS);
        blk = 0;
      }
      const uint8_t* tile = cache_layer + q4_tile(blk, g, 0, kv_heads);
      float s[HY_GROUP];
      {
        const uint4* codes = reinterpret_cast<const uint4*>(tile + (key % HY_BLOCK) * Q4_ROW_BYTES);
        const uint2 par = *reinterpret_cast<const uint2*>(tile + Q4_PARAM_OFF + (key % HY_BLOCK) * Q4_PARAM_BYTES);
        float2 s2[HY_GROUP];                              // sums of even and odd dimensions
#pragma unroll
        for (int h = 0; h < HY_GROUP; ++h) s2[h] = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 w4 = codes[i];
          const float2 sm = __half22float2(q4_as_half2(i < 2 ? par.x : par.y));
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float2 x[4];
            q4_values(w == 0 ? w4.x : w == 1 ? w4.y : w == 2 ? w4.z : w4.w, sm.x, sm.y, x);
#pragma unroll
            for (int h = 0; h < HY_GROUP; ++h) {
              const float4* qp = reinterpret_cast<const float4*>(&sh.q[h][32 * i + 8 * w]);
              const float4 a = qp[0], b = qp[1];
              s2[h] = __ffma2_rn(make_float2(a.x, a.y), x[0], s2[h]);
              s2[h] = __ffma2_rn(make_float2(a.z, a.w), x[1], s2[h]);
              s2[h] = __ffma2_rn(make_float2(b.x, b.y), x[2], s2[h]);
              s2[h] = __ffma2_rn(make_float2(b.z, b.w), x[3], s2[h]);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < HY_GROUP; ++h) s[h] = s2[h].x + s2[h].y;
      }
      float p[HY_GROUP];
#pragma unroll
      for (int h = 0; h < HY_GROUP; ++h) {
        s[h] = lane < cnt ? s[h] * scale : -INFINITY;     // rows past the end hold anything
        float mx = s[h];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float m_new = fmaxf(m[h], mx), mu = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = expf(m[h] - mu);
        p[h] = expf(s[h] - mu);
        m[h] = m_new;
        l[h] = fmaf(l[h], alpha, p[h]);                   // this lane's part of the sum
#pragma unroll
        for (int d = 0; d < 2; ++d) acc[h][d] = __fmul2_rn(acc[h][d], make_float2(alpha, alpha));
      }
      float4* pw = reinterpret_cast<float4*>(sh.p[warp][lane]);
      pw[0] = make_float4(p[0], p[0], p[1], p[1]);
      pw[1] = make_float4(p[2], p[2], p[3], p[3]);
      __syncwarp();
      // this lane's 4 dimensions (4 lane ..) of each key's value: half a code word
      const int sh8 = 8 * (lane & 1);
      for (int half = 0; half < 2; ++half) {              // a block of 16 keys each
        const int b = __shfl_sync(0xffffffffu, blk, 16 * half), n = min(HY_BLOCK, cnt - 16 * half);
        const uint8_t* vt = cache_layer + q4_tile(b, g, 1, kv_heads);
        const uint8_t* w_at = vt + 4 * (lane >> 1);
        const uint8_t* p_at = vt + Q4_PARAM_OFF + 4 * (lane >> 4);
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(w_at + j * Q4_ROW_BYTES) >> sh8;
          const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(p_at + j * Q4_PARAM_BYTES));
          const float2 scale2 = make_float2(sm.x, sm.x), low2 = make_float2(sm.y, sm.y);
          // nibbles j, j + 1 and, 16 bits up, their partners
          const float2 x0 = __ffma2_rn(q4_nibbles(w, 0), scale2, low2), x1 = __ffma2_rn(q4_nibbles(w, 4), scale2, low2);
          const float4* pj = reinterpret_cast<const float4*>(sh.p[warp][16 * half + j]);
          const float4 pa = pj[0], pb = pj[1];
          const float2 ph[HY_GROUP] = {make_float2(pa.x, pa.y), make_float2(pa.z, pa.w), make_float2(pb.x, pb.y),
                                       make_float2(pb.z, pb.w)};
#pragma unroll
          for (int h = 0; h < HY_GROUP; ++h) {
            acc[h][0] = __ffma2_rn(ph[h], x0, acc[h][0]);
            acc[h][1] = __ffma2_rn(ph[h], x1, acc[h][1]);
          }
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int h = 0; h < HY_GROUP; ++h) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
      if (lane == 0) sh.ml[warp][h] = make_float2(m[h], l[h]);
      *reinterpret_cast<float4*>(&sh.o[warp][h][4 * lane]) = make_float4(acc[h][0].x, acc[h][0].y, acc[h][1].x, acc[h][1].y);
    }
    __syncthreads();
    for (int i = tid; i < HY_GROUP * HY_HEAD_DIM; i += F_WARPS * 32) {
      const int h = i / HY_HEAD_DIM, d = i % HY_HEAD_DIM;
      float M = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < F_WARPS; ++w) M = fmaxf(M, sh.ml[w][h].x);
      const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int w = 0; w < F_WARPS; ++w) {
        const float wt = expf(sh.ml[w][h].x - mu);
        L = fmaf(wt, sh.ml[w][h].y, L);
        o = fmaf(wt, sh.o[w][h][d], o);
      }
      out[at + i] = o / L;
    }
  }
}

}  // namespace

cudaError_t hy_launch_attn_q4_fp32(const void* q, void* out, int tokens, int q_heads, int kv_heads,
                                   const void* cache_layer, int num_blocks,
                                   const int32_t* block_tables, int bt_pitch,
                                   const int32_t* seq_bt_row, const int32_t* cu_q,
                                   const int32_t* seq_lens_k, int S, float scale, int32_t* err,
                                   cudaStream_t st) {
  const long units = (long)tokens * kv_heads;
  return hy_launch(attn_q4_fp32_kernel, dim3((int)(units < 148L * 32 ? units : 148L * 32)),
                   dim3(F_WARPS * 32), 0, st, static_cast<const float*>(q), static_cast<float*>(out),
                   tokens, q_heads, kv_heads, static_cast<const uint8_t*>(cache_layer), num_blocks,
                   block_tables, bt_pitch, seq_bt_row, cu_q, seq_lens_k, S, scale, err);
}

cudaError_t hy_launch_attn_q4_bf16(const CUtensorMap* q_map, const void* q, void* out, int tokens,
                                   int q_heads, int kv_heads,
                                   const void* cache_layer, int num_blocks, int layer,
                                   const int32_t* block_tables, int bt_pitch,
                                   const int32_t* seq_bt_row, int S, float scale,
                                   const PlanDims& dims, void* ws, int32_t* err, int dev,
                                   cudaStream_t st) {
  static std::atomic<bool> attr_set[64];                  // per device, set on its first call
  if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(attn_q4_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         MIXED_SMEM);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(attn_q4_decode_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DEC_SMEM);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
  }
  Args a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.cache = static_cast<const uint8_t*>(cache_layer);
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.num_blocks = num_blocks;
  a.layer = layer;
  a.num_seqs = S;
  a.num_tokens = tokens;
  a.block_cap = hy_dec_block_cap(S, kv_heads);
  a.block_tables = block_tables;
  a.bt_pitch = bt_pitch;
  a.seq_bt_row = seq_bt_row;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err = err;
  const dim3 grid(hy_attn_num_sms(dev)), block(NT);
  const PlanView v = hy_attn_plan_view(ws, dims);
  if (q_map == nullptr) return hy_launch(attn_q4_decode_kernel, grid, block, DEC_SMEM, st, a, v);
  return hy_launch(attn_q4_kernel, grid, block, MIXED_SMEM, st, *q_map, a, v);
}
