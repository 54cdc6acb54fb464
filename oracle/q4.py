"""Plain specification of the 4-bit KV cache -- TEST INFRASTRUCTURE ONLY.

Tiles, codes and parameters as ``include/hayate_b200.h`` defines them for
``hy_kv_append_q4``.  The codes' arithmetic is numpy float32, one IEEE operation
at a time, so the kernel must match it byte for byte; attention is float64.
"""
from __future__ import annotations

import numpy as np

BLOCK, HEAD_DIM, HALF, GROUP = 16, 128, 64, 4
CODE_BYTES = BLOCK * HEAD_DIM // 2
TILE_BYTES = CODE_BYTES + BLOCK * 8
LIMIT = np.float32(32768.0)


def _dims_of_nibbles() -> np.ndarray:
    """dims[w, n]: the dimension that nibble n of word w holds."""
    w, n = np.meshgrid(np.arange(HEAD_DIM // 8), np.arange(8), indexing="ij")
    return 8 * w + np.where(n < 4, 2 * n, 2 * (n - 4) + 1)


DIMS = _dims_of_nibbles()


def quantise(x: np.ndarray):
    """float32 rows (..., 128) -> code bytes (..., 64) and fp16 parameters (..., 4)."""
    x = x.astype(np.float32)
    y = x.reshape(*x.shape[:-1], 2, HALF)
    nan = np.isnan(y).any(-1, keepdims=True)
    y = np.clip(np.where(np.isnan(y), np.float32(0), y), -LIMIT, LIMIT)
    lo, hi = y.min(-1, keepdims=True), y.max(-1, keepdims=True)
    low = lo.astype(np.float16)
    scale = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16)
    s = scale.astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        inv = np.where(s > 0, np.float32(1) / s, np.float32(0)).astype(np.float32)
        code = np.clip(np.rint((y - low.astype(np.float32)) * inv), 0, 15)
    code = np.where(nan, 0, code).astype(np.uint8).reshape(x.shape)
    bad = np.float16(np.nan)
    par = np.concatenate([np.where(nan, bad, scale), np.where(nan, bad, low)], -1)
    nib = code[..., DIMS].astype(np.uint32)                       # (..., word, nibble)
    words = (nib << (4 * np.arange(8, dtype=np.uint32))).sum(-1).astype("<u4")
    return (np.ascontiguousarray(words).view(np.uint8).reshape(*x.shape[:-1], HEAD_DIM // 2),
            par.reshape(*x.shape[:-1], 4))


def values(codes: np.ndarray, params: np.ndarray) -> np.ndarray:
    """float64 rows (..., 128) of code bytes (..., 64) and fp16 parameters (..., 4)."""
    words = np.ascontiguousarray(codes).view("<u4")
    nib = (words[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15
    code = np.empty((*codes.shape[:-1], HEAD_DIM), np.float64)
    code[..., DIMS] = nib
    p = params.astype(np.float64)
    out = code.reshape(*codes.shape[:-1], 2, HALF)
    out = out * p.reshape(*p.shape[:-1], 2, 2)[..., :1] + p.reshape(*p.shape[:-1], 2, 2)[..., 1:]
    return out.reshape(code.shape)


def tile_codes(cache: np.ndarray) -> np.ndarray:
    """View of the codes, (..., 16, 64)."""
    return cache[..., :CODE_BYTES].reshape(*cache.shape[:-1], BLOCK, HEAD_DIM // 2)


def tile_params(cache: np.ndarray) -> np.ndarray:
    """The parameters, fp16 (..., 16, 4) (a copy)."""
    p = np.ascontiguousarray(cache[..., CODE_BYTES:])
    return p.view(np.float16).reshape(*cache.shape[:-1], BLOCK, 4)


def append(cache_layer: np.ndarray, k: np.ndarray, v: np.ndarray, slots) -> None:
    """hy_kv_append_q4 on a numpy cache layer (blocks, heads, 2, TILE_BYTES), in place."""
    for t, slot in enumerate(slots):
        if slot < 0 or slot >= cache_layer.shape[0] * BLOCK:
            continue
        blk, off = divmod(int(slot), BLOCK)
        for part, x in enumerate((k, v)):
            codes, par = quantise(x[t])
            cache_layer[blk, :, part, 64 * off:64 * (off + 1)] = codes
            at = CODE_BYTES + 8 * off
            cache_layer[blk, :, part, at:at + 8] = np.ascontiguousarray(par).view(np.uint8)


def read(cache_layer: np.ndarray, slots):
    """float64 (k, v), each (tokens, heads, 128); zeros for slots outside the pool."""
    x = values(tile_codes(cache_layer), tile_params(cache_layer))   # (NB, heads, 2, 16, 128)
    s = np.asarray(slots)
    ok = (s >= 0) & (s < cache_layer.shape[0] * BLOCK)
    at = np.where(ok, s, 0)
    rows = np.where(ok[:, None, None, None], x[at // BLOCK, :, :, at % BLOCK], 0.0)
    return rows[:, :, 0], rows[:, :, 1]


def attention(q: np.ndarray, cache_layer: np.ndarray, tables: np.ndarray, q_lens, kv_lens,
              scale: float):
    """float64 causal attention (T, Hq, 128) and, per output row, what an error
    bound needs: sum of p (|v| + |minimum of v's half row|), the largest |scale| sum |q k| over visible keys,
    the number of visible keys and the largest |v|."""
    out = np.zeros(q.shape, np.float64)
    absv = np.zeros(q.shape, np.float64)
    reach = np.zeros(q.shape[:2], np.float64)
    keys = np.zeros(q.shape[:2], np.float64)
    vmax = np.zeros(q.shape[:2], np.float64)
    first = 0
    for i, (ql, kv) in enumerate(zip(q_lens, kv_lens)):
        x = None
        if ql:
            blocks = tables[i, :-(-kv // BLOCK)]
            par = tile_params(cache_layer[blocks])
            x = values(tile_codes(cache_layer[blocks]), par)
            low = np.repeat(np.abs(par[:, :, 1, :, 1::2].astype(np.float64)), HALF, -1)
            low = low.transpose(1, 0, 2, 3).reshape(low.shape[1], -1, HEAD_DIM)[:, :kv]
            x = x.transpose(1, 2, 0, 3, 4).reshape(x.shape[1], 2, -1, HEAD_DIM)[:, :, :kv]
        for h in range(q.shape[1] if ql else 0):
            k, v = x[h // GROUP]
            z = scale * (q[first:first + ql, h].astype(np.float64) @ k.T)
            r = abs(scale) * (np.abs(q[first:first + ql, h].astype(np.float64)) @ np.abs(k).T)
            hidden = np.arange(kv)[None] > (kv - ql + np.arange(ql))[:, None]
            z = np.where(hidden, -np.inf, z)
            p = np.exp(z - z.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[first:first + ql, h] = p @ v
            absv[first:first + ql, h] = p @ (np.abs(v) + low[h // GROUP])
            reach[first:first + ql, h] = np.where(hidden, 0, r).max(-1)
            keys[first:first + ql, h] = (~hidden).sum(-1)
            vmax[first:first + ql, h] = (np.abs(v) + low[h // GROUP]).max()
        first += ql
    return out, absv, reach, keys, vmax
