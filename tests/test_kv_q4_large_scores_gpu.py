"""The 4-bit cache's attention on queries of any size: what the result has to be is known whatever the
scores' roundings are (run on a B200)."""
import numpy as np
import pytest
import torch

from oracle import q4
from test_kv_q4_gpu import BF, F32, Batch

pytestmark = pytest.mark.gpu

LENS = [([1, 1, 1], [90, 33, 300]), ([1], [5003]), ([1] * 40, [700 - 9 * i for i in range(40)]),   # decode
        ([1, 3, 0, 0], [90, 200, 1, 1]), ([70], [300]), ([512], [4000]), ([1, 70, 1], [500, 300, 2000])]


@pytest.mark.parametrize("dt,power", [(BF, -90), (BF, 17), (BF, 100), (BF, 117), (BF, 122), (F32, -90), (F32, 17),
                                      (F32, 100)])
@pytest.mark.parametrize("lens", LENS)
def test_a_power_of_two_moves_between_queries_and_scale(lens, dt, power):
    """2^power q with 2^-power scale: every product is the same but for exponents, so every bit is."""
    b = Batch(*lens, 2, dt, seed=41)
    want = b.run()
    b.check(want)
    b.q = (b.q.double() * 2.0 ** power).to(dt)
    assert torch.equal(b.run(scale=128 ** -0.5 * 2.0 ** -power), want)


def plant(b, c, ties):
    """Query rows c times a key that they see, so that its score is ahead of all others by far more
    than scores are rounded.  With `ties`, another key has the same codes.  Returns what the rows'
    output is, the winning value or the winners' mean, and the |v| + |minimum| of the winners."""
    rng = np.random.default_rng(7)
    heads, layer = b.heads, b.cache[b.layer]
    want = np.zeros((b.T, 4 * heads, 128))
    size = np.zeros_like(want)
    codes, params = layer[..., :q4.CODE_BYTES], layer[..., q4.CODE_BYTES:]
    row = 0
    for i, (ql, kv) in enumerate(zip(b.q_lens, b.kv_lens)):
        at = lambda j: (b.tables[i, j // 16], j % 16)
        pair = None
        if ties and ql:
            seen = kv - ql + 1                          # keys that every row sees
            pair = seen // 5, seen - 1 - seen // 7
            (b0, o0), (b1, o1) = at(pair[0]), at(pair[1])
            codes[b1, :, 0, 64 * o1:64 * o1 + 64] = codes[b0, :, 0, 64 * o0:64 * o0 + 64]
            params[b1, :, 0, 8 * o1:8 * o1 + 8] = params[b0, :, 0, 8 * o0:8 * o0 + 8]
        blocks = b.tables[i, :-(-kv // 16)]
        par = q4.tile_params(layer[blocks])
        x = q4.values(q4.tile_codes(layer[blocks]), par)        # (blocks, heads, 2, 16, 128)
        low = np.repeat(np.abs(par[:, :, 1, :, 1::2].astype(np.float64)), 64, -1)
        for t in range(ql):
            n = kv - ql + t + 1
            for h in range(4 * heads):
                g = h // 4
                k = x[:, g, 0].reshape(-1, 128)[:n]
                v = x[:, g, 1].reshape(-1, 128)[:n]
                w = np.abs(v) + low[:, g].reshape(-1, 128)[:n]
                for _ in range(20):
                    win = list(pair) if pair else [int(rng.integers(n))]
                    q = torch.from_numpy(k[win[0]] * c).to(b.dt)
                    z = 128 ** -0.5 * (k @ q.double().numpy())
                    reach = 128 ** -0.5 * (np.abs(k) @ np.abs(q.double().numpy())).max()
                    rest = np.delete(z, win)
                    # a score is off by 2^-11 of its terms' sum at most, twice over; 2^-60 is left of a
                    # weight that is 42 behind
                    if rest.size == 0 or z[win[0]] - rest.max() > 4 * 2.0 ** -11 * reach + 42:
                        break
                else:
                    raise AssertionError("no key is ahead")
                b.q[row + t, h] = q
                want[row + t, h] = v[win].mean(0)
                size[row + t, h] = w[win].mean(0)
        row += ql
    return want, size


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("dt,c", [(BF, 1e3), (BF, 1e5), (BF, 1e8), (BF, 1e12), (BF, 1e30), (BF, 1e36), (F32, 1e3),
                                  (F32, 1e8), (F32, 1e30)])
@pytest.mark.parametrize("lens", [([1, 1, 1], [90, 33, 300]), ([1], [5003]), ([1] * 12, [700 - 9 * i for i in range(12)]),
                                  ([1, 3, 0, 0], [90, 200, 1, 1]), ([70], [300]), ([24], [4000])])
def test_the_winning_key_s_value_comes_out(lens, dt, c, ties):
    b = Batch(*lens, 2, dt, seed=42)
    want, size = plant(b, c, ties)
    out = b.run()[:b.T].double().cpu().numpy()
    # bf16: the weight and its product with the value's scale, or the value itself, are rounded to
    # fp16 (2^-11 each), the output to bf16 (8 significant bits: steps of 2^-7 of the leading
    # one, so half a step is up to 2^-8 of the value); fp32: a few roundings of 2^-24
    tol = 2.0 ** -8 * np.abs(want) + 2.02 * 2.0 ** -11 * size if dt == BF else 8 * 2.0 ** -24 * size
    assert np.isfinite(out).all()
    bad = np.abs(out - want) > tol * 1.01 + 1e-30
    assert bad.sum() == 0, (np.argwhere(bad)[:5], (np.abs(out - want) / tol).max())
