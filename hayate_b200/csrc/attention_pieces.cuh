// Prefill items and their key-range pieces: what the plan, the bf16 cache's kernel
// and the 4-bit cache's kernel share.
#pragma once

#include "attention.cuh"
#include "common.cuh"

namespace {

constexpr float NEG_INF = -INFINITY;
constexpr int PRE_QROWS = 64;                                    // query tokens per prefill item
constexpr int PRE_KEYS = 64;                                     // keys per tile
constexpr int PRE_ROWS = HY_GROUP * PRE_QROWS;                   // score rows of an item: 256
constexpr int PRE_PIECE_BAR = 1;                                 // named barrier of the softmax warps

// Split prefill items: a step with fewer prefill items (64 query tokens x one
// KV head) than SMs cuts the long ones into pieces over equal key-tile ranges,
// at least PRE_SPLIT_MIN tiles each, so that the pieces fill the idle SMs;
// each piece leaves its unnormalised O, running max and sum in the workspace
// and the last piece to finish merges them.  Without this such a step waits
// for its longest items (one 512-token chunk after 3584 cached tokens: 64
// items of 57-64 key tiles, 84 SMs idle: 80.0 us uncut, 57.6 us cut).  A
// step with at least as many items as SMs, or with decode work for the idle
// SMs, is not cut: a piece costs a second Q load, a 128 KB partial and its
// share of the merge (~25k cycles per cut item, measured), more than the
// balance gains there (4 chunks of 512: 80.6 us uncut, 93.0 us cut to the
// tiles per SM; one chunk beside 256 decode sequences: 704 us uncut, 732 us
// cut).
#ifndef HY_PRE_SPLIT_MIN
#define HY_PRE_SPLIT_MIN 16
#endif
constexpr int PRE_SPLIT_MIN = HY_PRE_SPLIT_MIN;                  // key tiles
constexpr int PRE_MAX_PIECES = 31;
constexpr int PRE_PART_F4 = 32 * 256;                            // float4 of O per piece

// A sequence that the plan takes: keys for all its query tokens, and no more of them
// than any pool holds (2^28; the plan sums the tiles of up to an item per SM in 32 bits).
constexpr int SEQ_MAX_KEYS = 1 << 28;
HY_DEVICE bool seq_fits(int q, int kv) { return q >= 0 && kv >= q && kv <= SEQ_MAX_KEYS; }

// key tiles of the prefill item at query offset t0 of a sequence of q query
// tokens and kv keys
HY_DEVICE int pre_item_tiles(int kv, int q, int t0) {
  return (kv - q + t0 + min(PRE_QROWS, q - t0) + PRE_KEYS - 1) / PRE_KEYS;
}
HY_DEVICE int pre_pieces(int nt, int cap) {
  return nt > cap ? min(PRE_MAX_PIECES, (nt + cap - 1) / cap) : 1;
}
// An item's w field: 0 for a whole item, else (pieces << 26) | (piece << 20) |
// the first partial slot of the item (its pieces use consecutive slots).
HY_DEVICE int pre_piece_code(int ns, int sp, int slot) { return (ns << 26) | (sp << 20) | slot; }
HY_DEVICE int pre_code_pieces(int w) { return (w >> 26) & 31; }
HY_DEVICE int pre_code_piece(int w) { return (w >> 20) & 63; }
HY_DEVICE int pre_code_slot(int w) { return w & 0xFFFFF; }
// key tiles [lo, hi) that the item (w) of nt key tiles covers
HY_DEVICE void pre_piece_range(int w, int nt, int& lo, int& hi) {
  if (w == 0) { lo = 0; hi = nt; return; }
  const int ns = pre_code_pieces(w), sp = pre_code_piece(w);
  lo = sp * nt / ns;
  hi = (sp + 1) * nt / ns;
}

// The end of one piece of a split prefill item, run by all PRE_ROWS
// softmax threads (thread rr holds row rr of the item's 256 rows): the row's
// unnormalised O (TMEM column base tO) and (m, l) go to the piece's partial
// slot; the piece that finishes last (counted at the item's first slot)
// merges every piece's partials into the output row op (nullptr: a padding row)
// and resets the count.  Piece s weighs 2^(m_s - M), M the largest m_s.
// pre_last is shared memory.  Returns whether every thread's waits succeeded.
HY_DEVICE bool prefill_piece_finish(const PlanView& v, int w, int rr, uint32_t tO, float m,
                                     float l, bool ok, __nv_bfloat16* op, int& pre_last) {
  const int ns = pre_code_pieces(w), sp = pre_code_piece(w), slot = pre_code_slot(w);
  const bool all_ok = !named_sync_or(PRE_PIECE_BAR, PRE_ROWS, !ok);
  if (all_ok) {
    float4* po = v.pre_part_o + (size_t)(slot + sp) * PRE_PART_F4 + rr;
#pragma unroll 1
    for (int cc = 0; cc < 4; ++cc) {
      float o[32];
      tmem_ld32(tO + 32 * cc, o);
      tmem_wait_ld(o);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        __stcg(po + (cc * 8 + k) * 256,
               make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]));
    }
    __stcg(v.pre_part_ml + (size_t)(slot + sp) * 256 + rr, make_float2(m, l));
    __threadfence();                            // this row's partial, before the count
  }
  named_sync(PRE_PIECE_BAR, PRE_ROWS);
  if (threadIdx.x == 0) pre_last = all_ok && atomicAdd(&v.pre_ctr[slot], 1) == ns - 1;
  named_sync(PRE_PIECE_BAR, PRE_ROWS);
  if (!pre_last) return all_ok;
  __threadfence();                              // the other pieces' partials, after the count
  const float2* ml = v.pre_part_ml + (size_t)slot * 256 + rr;
  float M = NEG_INF;
#pragma unroll 4
  for (int s = 0; s < ns; ++s) M = fmaxf(M, __ldcg(ml + s * 256).x);
  float L = 0.f;
#pragma unroll 4
  for (int s = 0; s < ns; ++s) {
    const float2 e = __ldcg(ml + s * 256);
    L += e.y * (M == NEG_INF ? 0.f : ex2_ftz(e.x - M));
  }
  const float inv = 1.f / L;
#pragma unroll 1
  for (int cc = 0; cc < 4; ++cc) {
    float acc[32];
#pragma unroll
    for (int k = 0; k < 32; ++k) acc[k] = 0.f;
    // two pieces per round: their 16 loads are in flight together
#pragma unroll 1
    for (int s = 0; s < ns; s += 2) {
      const int s1 = min(s + 1, ns - 1);
      const float w0 = M == NEG_INF ? 0.f : ex2_ftz(__ldcg(ml + s * 256).x - M);
      const float w1 = (s1 == s || M == NEG_INF) ? 0.f : ex2_ftz(__ldcg(ml + s1 * 256).x - M);
      const float4* p0 = v.pre_part_o + (size_t)(slot + s) * PRE_PART_F4 + cc * 8 * 256 + rr;
      const float4* p1 = v.pre_part_o + (size_t)(slot + s1) * PRE_PART_F4 + cc * 8 * 256 + rr;
      float4 f0[8], f1[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f0[k] = __ldcg(p0 + k * 256);
        f1[k] = __ldcg(p1 + k * 256);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        acc[4 * k] += w0 * f0[k].x + w1 * f1[k].x;
        acc[4 * k + 1] += w0 * f0[k].y + w1 * f1[k].y;
        acc[4 * k + 2] += w0 * f0[k].z + w1 * f1[k].z;
        acc[4 * k + 3] += w0 * f0[k].w + w1 * f1[k].w;
      }
    }
    if (op) {
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        uint4 pk4;
        pk4.x = pack_bf16(acc[8 * q4 + 0] * inv, acc[8 * q4 + 1] * inv);
        pk4.y = pack_bf16(acc[8 * q4 + 2] * inv, acc[8 * q4 + 3] * inv);
        pk4.z = pack_bf16(acc[8 * q4 + 4] * inv, acc[8 * q4 + 5] * inv);
        pk4.w = pack_bf16(acc[8 * q4 + 6] * inv, acc[8 * q4 + 7] * inv);
        *reinterpret_cast<uint4*>(op + 32 * cc + 8 * q4) = pk4;
      }
    }
  }
  if (threadIdx.x == 0) v.pre_ctr[slot] = 0;   // for the next launch on this plan
  return all_ok;
}

}  // namespace
