"""The 4-bit KV cache on the CPU: its specification and what the C ABI refuses."""
import ctypes

import numpy as np
import pytest
import torch

from hayate_b200 import _lib
from hayate_b200 import kernels as K
from oracle import q4


def test_codes_stay_within_half_a_step():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 128)) * 10 ** rng.uniform(-3, 3, (50, 1))).astype(np.float32)
    x += rng.standard_normal((50, 1)).astype(np.float32)
    codes, par = q4.quantise(x)
    back = q4.values(codes, par)
    step = np.repeat(par[:, 0::2].astype(np.float64), 64, -1)
    low = np.repeat(np.abs(par[:, 1::2].astype(np.float64)), 64, -1)
    # half a step, or at the ends of the range what the parameters' rounding cut off: 15 steps
    # rounded to fp16 and the minimum rounded to fp16 (2^-11 each), the subnormal fp16 step
    # of each, and the fp32 arithmetic of the codes (far below a code)
    cut = 15 * (step * 2.0 ** -11 + 2.0 ** -25) + low * 2.0 ** -11 + 2.0 ** -25
    assert (np.abs(back - x) <= step * (0.5 + 1e-5) + cut).all()


def test_spec_nibble_order():
    x = np.tile(np.arange(64, dtype=np.float32) % 16, 2)[None]     # step 1, minimum 0
    codes, par = q4.quantise(x)
    assert par.tolist() == [[1.0, 0.0, 1.0, 0.0]]
    w0 = int(codes[0, :4].view("<u4")[0])
    assert [(w0 >> (4 * n)) & 15 for n in range(8)] == [0, 2, 4, 6, 1, 3, 5, 7]
    assert np.array_equal(q4.values(codes, par), x)


def _aligned(n=8192):
    buf = ctypes.create_string_buffer(n + 16)
    return buf, (ctypes.addressof(buf) + 15) // 16 * 16


def test_append_and_read_refuse_bad_arguments():
    lib = _lib.load()
    keep, p = _aligned()

    def append(dtype=0, k=p, ldk=256, v=p, ldv=256, n=1, heads=2, slots=p, cache=p, nb=4):
        return lib.hy_kv_append_q4(dtype, k, ldk, v, ldv, n, heads, slots, cache, nb, None, None)

    def read(dtype=0, cache=p, nb=4, heads=2, slots=p, n=1, k=p, v=p):
        return lib.hy_kv_read_q4(dtype, cache, nb, heads, slots, n, k, v, None, None)

    assert append(n=0) == 0 and read(n=0) == 0                      # nothing to do
    for kw in (dict(dtype=2), dict(k=None), dict(v=None), dict(slots=None), dict(cache=None),
               dict(n=-1), dict(heads=0), dict(heads=1 << 20, ldk=1 << 28, ldv=1 << 28),
               dict(nb=0), dict(ldk=255), dict(ldv=128), dict(ldk=260), dict(k=p + 2),
               dict(v=p + 8), dict(cache=p + 4), dict(dtype=1, ldv=258)):
        assert append(**kw) == -1, kw
        assert lib.hy_get_last_error().startswith(b"hy_kv_append_q4")
    for kw in (dict(dtype=-1), dict(cache=None), dict(slots=None), dict(k=None), dict(v=None),
               dict(n=-5), dict(heads=0), dict(nb=-1), dict(k=p + 8), dict(cache=p + 8)):
        assert read(**kw) == -1, kw
        assert lib.hy_get_last_error().startswith(b"hy_kv_read_q4")


def test_attention_refuses_bad_arguments():
    lib = _lib.load()
    keep, p = _aligned()

    def call(dtype=1, q=p, out=p, n=1, qh=8, kh=2, cache=p, layers=2, nb=4, layer=0, bt=p, pitch=4,
             cu=p, kv=p, seqs=1, ws=p, ws_bytes=0, scale=0.1):
        return lib.hy_varlen_attention_q4(dtype, q, out, n, qh, kh, cache, layers, nb, layer, bt, pitch,
                                          None, cu, kv, seqs, scale, 4, 4, ws, ws_bytes, None, None)

    assert call(n=0) == 0
    for kw in (dict(dtype=3), dict(q=None), dict(out=None), dict(cache=None), dict(bt=None),
               dict(cu=None), dict(kv=None), dict(n=-1), dict(layers=0), dict(nb=0), dict(layer=2),
               dict(layer=-1), dict(pitch=0), dict(seqs=0), dict(q=p + 8), dict(out=p + 8),
               dict(cache=p + 8), dict(scale=-0.1), dict(scale=float("nan")),
               dict(scale=float("inf"))):
        assert call(**kw) == -1, kw
        assert lib.hy_get_last_error().startswith(b"hy_varlen_attention_q4")
    assert call(qh=6) == -3 and call(kh=0, qh=0) == -3


def test_wrappers_refuse_what_is_not_a_cache():
    cache = K.kv_cache_q4(1, 3, 2, device="cpu")
    assert tuple(cache.shape) == (1, 3, 2, 2, 1152) and q4.TILE_BYTES == K.Q4_TILE_BYTES
    k = torch.zeros(4, 2, 128)
    slots = torch.zeros(4, dtype=torch.int32)
    for bad in (cache, cache[0].float(), cache[0, :, :, :, :1024], cache[0].transpose(0, 1)):
        with pytest.raises(ValueError, match="4-bit cache"):
            K.kv_append_q4(k, k, slots, bad)
        with pytest.raises(ValueError, match="4-bit cache"):
            K.kv_read_q4(bad, slots, torch.float32)
    for kk, vv in ((k[:, :1], k), (k, k[..., :64]), (k, k.bfloat16())):
        with pytest.raises(ValueError, match="must be"):
            K.kv_append_q4(kk, vv, slots, cache[0])
    with pytest.raises(ValueError, match="contiguous"):
        K.kv_append_q4(k, torch.zeros(4, 128, 2).transpose(1, 2), slots, cache[0])
    with pytest.raises(ValueError, match="int32 CUDA"):      # a host slot list
        K.kv_append_q4(k, k, slots, cache[0])
    with pytest.raises(ValueError, match="4-bit cache"):
        K.varlen_attention_q4(k, k, cache[0], 0, slots, slots, slots, 1, 1, 4, None)


def test_engine_refuses_unknown_cache_types():
    from hayate_b200.config import EngineConfig, TINY
    from hayate_b200.model import Runner
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        Runner(TINY, EngineConfig(kv_cache_dtype="fp8"), torch.float32, torch.device("cpu"), None, [])


def test_attention_of_no_tokens_is_nothing_to_do():
    """An empty tensor's address is null."""
    lib = _lib.load()
    keep, p = _aligned()
    for dtype in (0, 1):
        assert lib.hy_varlen_attention_q4(dtype, None, None, 0, 8, 2, p, 2, 4, 0, p, 4, None, p, p, 1, 0.1, 4, 4,
                                          None, 0, None, None) == 0
        assert lib.hy_varlen_attention_q4(dtype, None, None, 0, 8, 2, None, 2, 4, 0, p, 4, None, p, p, 1, 0.1, 4,
                                          4, None, 0, None, None) == -1
