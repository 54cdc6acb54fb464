"""The 4-bit KV cache's kernels against their specification (run on a B200)."""
import numpy as np
import pytest
import torch

from hayate_b200 import kernels as K
from oracle import q4

pytestmark = pytest.mark.gpu
dev = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def i32(a):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32, device=dev).contiguous()


def rows(gen, *shape):
    """Near-normal rows with some strong dimensions and an offset per head."""
    x = torch.randn(*shape, 128, generator=gen)
    x = x * (0.5 + torch.rand(*shape[1:], 128, generator=gen))
    return x + 0.5 * torch.randn(*shape[1:], 1, generator=gen)


def random_cache(gen, layers, nb, heads):
    """A 4-bit cache written everywhere, as numpy."""
    x = rows(gen, layers * nb * 2 * 16, heads).view(layers, nb, 2, 16, heads, 128)
    x = x.permute(0, 1, 4, 2, 3, 5).numpy()
    codes, par = q4.quantise(x)
    return np.concatenate([codes.reshape(layers, nb, heads, 2, -1),
                           par.view(np.uint8).reshape(layers, nb, heads, 2, -1)], -1)


# ------------------------------------------------------------------ write, read
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (3, 8), (17, 2), (333, 3), (2500, 8)])
def test_append_bytes(dt, tokens, heads):
    g = torch.Generator().manual_seed(tokens + heads)
    nb = tokens // 16 + 5
    k = rows(g, tokens, heads).to(dt)
    qkv = torch.zeros(tokens, (6 * heads) * 128, dtype=dt)
    qkv[:, 5 * heads * 128:] = rows(g, tokens, heads).to(dt).flatten(1)
    slots = torch.randperm(nb * 16, generator=g)[:tokens].numpy().astype(np.int32)
    slots[1::7] = -1
    want = random_cache(g, 2, nb, heads)
    cache = torch.from_numpy(want.copy()).to(dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    dqkv = qkv.to(dev)
    v = dqkv[:, 5 * heads * 128:].unflatten(1, (heads, 128))    # strided tokens
    K.kv_append_q4(k.to(dev), v, i32(slots), cache[1], err=err)
    q4.append(want[1], k.float().numpy(), v.float().cpu().numpy(), slots)
    assert int(err.item()) == 0
    # every byte: the written rows, the rows beside them and the other layer
    assert np.array_equal(cache.cpu().numpy(), want)


@pytest.mark.parametrize("dt", [BF, F32])
def test_append_special_rows(dt):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(14, 2, 128, generator=g)
    x[0] = 0.0
    x[1] = 3.25                                # constant: scale 0
    x[2] *= 1e30                               # clamped
    x[3, :, 5] = float("inf")
    x[4, :, 70] = -float("inf")
    x[5] *= 1e-6                               # fp16-subnormal parameters
    x[6] *= 1e-38
    x[7] = -0.0
    x[8] = 1000.0 + torch.arange(128) % 3      # a small range on a large offset
    x[9] = torch.where(torch.arange(128) % 2 == 0, -32768.0, 32768.0)
    x[10] = torch.arange(128) % 16             # codes exactly on the grid
    x[11] = torch.arange(128) % 16 * 0.5 - 3.5
    x[12, 0, 3] = float("nan")
    x[13, 1, 100] = float("nan")
    x = x.to(dt)
    want = np.zeros((2, 2, 2, q4.TILE_BYTES), np.uint8)
    cache = torch.zeros(2, 2, 2, q4.TILE_BYTES, dtype=torch.uint8, device=dev)
    slots = np.arange(14, dtype=np.int32) + 3
    K.kv_append_q4(x.to(dev), x.flip(-1).contiguous().to(dev), i32(slots), cache)
    q4.append(want, x.float().numpy(), x.flip(-1).float().numpy(), slots)
    got = cache.cpu().numpy()
    assert np.array_equal(q4.tile_codes(got), q4.tile_codes(want))
    assert np.array_equal(q4.tile_params(got), q4.tile_params(want), equal_nan=True)
    back_k, back_v = K.kv_read_q4(cache, i32(slots), F32)
    nan_k = torch.isnan(back_k).cpu()
    assert nan_k[12, 0, :64].all() and nan_k[13, 1, 64:].all() and int(nan_k.sum()) == 128
    assert float(back_k[2].abs().max()) <= 32768.0 * (1 + 2.0 ** -10)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("tokens,heads", [(1, 2), (40, 8), (1000, 3)])
def test_read_values(dt, tokens, heads):
    g = torch.Generator().manual_seed(tokens)
    cache = random_cache(g, 1, 40, heads)[0]
    slots = torch.randint(-2, 40 * 16, (tokens,), generator=g).numpy()
    slots[0] = 40 * 16 - 1
    slots[-1] = slots[0]                         # a slot twice
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    k, v = K.kv_read_q4(torch.from_numpy(cache).to(dev), i32(slots), dt, err=err)
    for got, want in zip((k, v), q4.read(cache, slots)):
        # scale * code + minimum is one fp32 rounding, then one to dt; both are monotone
        # roundings of a value that fp32 holds but for its last bit
        assert torch.equal(got.cpu(), torch.from_numpy(want).float().to(dt))
    assert int(err.item()) == 0


def test_out_of_range_slots_are_reported_and_skipped():
    g = torch.Generator().manual_seed(3)
    start = random_cache(g, 1, 4, 2)[0]
    cache = torch.from_numpy(start.copy()).to(dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    k = rows(g, 3, 2).to(dev)
    K.kv_append_q4(k, k, i32([64, 2 ** 31 - 1, -2 ** 31]), cache, err=err)
    assert int(err.item()) == K.DEV_BOUNDS and np.array_equal(cache.cpu().numpy(), start)
    err.zero_()
    a, b = K.kv_read_q4(cache, i32([64, 5, -9]), F32, err=err)
    assert int(err.item()) == K.DEV_BOUNDS
    assert not a[0].any() and not b[0].any() and a[1].any() and not a[2].any()


def test_append_offsets_past_32_bits():
    """A layer larger than 4 GB: the last block's bytes."""
    heads, nb = 8, (1 << 32) // (8 * 2 * q4.TILE_BYTES) + 3
    cache = torch.zeros(nb, heads, 2, q4.TILE_BYTES, dtype=torch.uint8, device=dev)
    g = torch.Generator().manual_seed(4)
    k, v = rows(g, 2, heads), rows(g, 2, heads)
    slots = [nb * 16 - 1, 7]
    K.kv_append_q4(k.to(dev), v.to(dev), i32(slots), cache)
    a, b = K.kv_read_q4(cache, i32(slots), F32)
    for got, x in ((a, k), (b, v)):
        codes, par = q4.quantise(x.numpy())
        assert np.array_equal(got.cpu().numpy(), q4.values(codes, par).astype(np.float32))
    assert not cache[1:nb - 1].any()


# ------------------------------------------------------------------ attention
class Batch:
    def __init__(self, q_lens, kv_lens, heads, dt, layers=2, layer=1, seed=0, qscale=1.0, pad_rows=0):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.kv_lens, self.layer = list(q_lens), list(kv_lens), layer
        counts = [-(-kv // 16) for kv in kv_lens]
        nb = sum(counts) + 5
        self.cache = random_cache(g, layers, nb, heads)
        ids = torch.randperm(nb, generator=g).numpy()
        self.tables = np.full((len(counts), max(counts) + 1), -1, np.int32)
        at = 0
        for i, n in enumerate(counts):
            self.tables[i, :n] = ids[at:at + n]
            at += n
        # rows past each sequence's end hold what an earlier owner left: NaN here
        for i, kv in enumerate(kv_lens):
            if kv % 16:
                tile = self.cache[:, self.tables[i, kv // 16]]
                tile[..., q4.CODE_BYTES + 8 * (kv % 16):] = 0xff
        self.T = sum(q_lens)
        self.q = (torch.randn(self.T + pad_rows, 4 * heads, 128, generator=g) * qscale).to(dt)
        self.cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        self.heads, self.dt = heads, dt

    def run(self, scale=None, seq_bt_row=None, tables=None, err=None, out=None):
        S, T = len(self.q_lens), self.q.shape[0]
        err = torch.zeros(1, dtype=torch.int32, device=dev) if err is None else err
        q = self.q.to(dev)
        out = torch.full_like(q, 7.0) if out is None else out
        cu, kv = i32(self.cu), i32(self.kv_lens)
        ws = torch.zeros(K.attention_workspace_size(S, T, self.heads), dtype=torch.uint8, device=dev)
        K.attention_plan(cu, kv, S, self.heads, S, T, ws, err)
        K.varlen_attention_q4(q, out, torch.from_numpy(self.cache).to(dev), self.layer,
                              i32(self.tables if tables is None else tables), cu, kv, S, S, T, ws,
                              seq_bt_row=seq_bt_row, scale=scale, err=err)
        assert int(err.item()) == 0, K.describe_error(int(err.item()))
        return out

    def check(self, out, scale=None):
        scale = 128 ** -0.5 if scale is None else scale
        want, absv, reach, keys, vmax = q4.attention(
            self.q[:self.T].float().numpy(), self.cache[self.layer], self.tables, self.q_lens,
            self.kv_lens, scale)
        got = out[:self.T].double().cpu().numpy()
        odd = np.argwhere(~np.isfinite(got))
        assert len(odd) == 0, odd[:5]
        keys, vmax, reach = (a[..., None] for a in (keys, vmax, reach))
        if self.dt == F32:
            # fp32: dot products and sums of `keys` terms, each term rounded (2^-24); exp of
            # an argument off by `reach` roundings of the dot product's 128 terms
            tol = absv * (2.0 ** -23 * (keys + 8) + 2 * 132 * 2.0 ** -24 * (reach + 1)) + 1e-30
        else:
            # keys, values and weights (decode: weights times the value's scale, which meet codes
            # of up to |v| + |minimum|) are held in fp16 where the tensor cores take them (2^-11
            # relative each; weights below 2^-14 to 2^-25), scores move by 2^-11 of their
            # terms' sum; fp32 sums (2^-23 per term); the output is rounded once to bf16 (2^-8)
            shift = reach * 2.0 ** -11 * 1.1
            tol = (2.0 ** -8 * np.abs(want) + absv * (2 * 2.0 ** -11 + 2 * np.expm1(shift) +
                                                      2.0 ** -23 * (keys + 300 * (reach + 1))) +
                   keys * 2.0 ** -25 * vmax + 1e-30) * 1.01
        bad = np.abs(got - want) > tol
        assert bad.sum() == 0, (np.argwhere(bad)[:5], np.abs(got - want)[bad][:5], tol[bad][:5])


CASES = [
    ([1], [1]), ([1], [16]), ([1], [17]), ([2], [2]), ([5], [5]),
    ([1, 1, 1], [15, 33, 64]),
    ([1, 40, 1, 17], [300, 40, 2049, 100]),
    ([0, 3, 0, 1], [5, 19, 16, 40]),             # sequences with no query token
    ([64], [64]), ([65], [130]), ([130], [700]), ([200, 1, 64, 1], [200, 90, 1000, 1]),
    ([512], [1111]), ([33] * 6, [33 + 50 * i for i in range(6)]),
    ([1] * 37, [1 + 61 * i % 900 for i in range(37)]),
    ([1, 0, 1, 1, 0], [0 + 40, 9, 1, 200, 3]), ([1] * 70, [1 + 13 * i % 40 for i in range(70)]),
    ([1, 1], [5003, 37]), ([1] * 20, [2500 - 97 * i for i in range(20)]),   # pairs split over many CTAs
]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("heads", [1, 2, 8])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(case, heads, dt):
    q_lens, kv_lens = CASES[case]
    b = Batch(q_lens, kv_lens, heads, dt, seed=case)
    b.check(b.run())


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("qscale,scale", [(1e-3, None), (8.0, None), (1.0, 0.5), (1.0, 0.0)])
def test_attention_score_ranges(qscale, scale, dt):
    b = Batch([1, 70], [500, 300], 2, dt, seed=11, qscale=qscale)
    b.check(b.run(scale=scale), scale=scale)


@pytest.mark.parametrize("dt", [F32, BF])
def test_attention_query_row_ranges(dt):
    """Query rows of zeros, of the type's smallest and of very large elements beside ordinary ones."""
    b = Batch([1, 1, 70], [90, 33, 300], 2, dt, seed=13)
    b.q[0] = 0
    b.q[1, 3] *= 1e-38
    b.q[5] = 0
    b.q[6] *= 1e-38
    b.q[7] *= 1e-20
    b.q[8, :, ::2] *= 1e-6            # far below its row's largest element
    b.q[9] *= 1e5                     # past fp16's range
    b.check(b.run())


@pytest.mark.parametrize("dt", [F32, BF])
def test_attention_value_ranges(dt):
    """Rows whose scales differ by many orders of magnitude, constant rows (scale 0) among them."""
    for lens in (([1, 1], [900, 40]), ([70], [333])):
        b = Batch(*lens, 2, dt, seed=14)
        g = torch.Generator().manual_seed(15)
        par = q4.tile_params(b.cache)                    # (layers, blocks, heads, 2, 16, 4)
        f = 10.0 ** (torch.rand(par.shape[:-1], generator=g).numpy() * 7 - 5)[..., None]
        f[:, ::3] = 0.0                                  # whole blocks of zeros
        f[:, :, :, 0] = 1.0                              # keys as they are
        par = (par.astype(np.float64) * f).astype(np.float16)
        b.cache[..., q4.CODE_BYTES:] = par.view(np.uint8).reshape(*b.cache.shape[:-1], -1)
        for i, kv in enumerate(b.kv_lens):               # no NaN: they were scaled away above
            assert np.isfinite(par.astype(np.float64)[:, b.tables[i, :kv // 16]]).all()
        b.check(b.run())


@pytest.mark.parametrize("dt", [F32, BF])
def test_attention_rows_past_the_last_sequence_stay(dt):
    b = Batch([1, 3, 70], [30, 3, 170], 2, dt, seed=5, pad_rows=9)
    out = b.run()
    b.check(out)
    assert (out[b.T:] == 7.0).all()


@pytest.mark.parametrize("dt", [F32, BF])
def test_attention_block_table_rows(dt):
    """seq_bt_row: sequence i's blocks stand in another row of the table."""
    b = Batch([1, 3, 1], [30, 47, 170], 2, dt, seed=6)
    perm = [4, 0, 2]
    tables = np.full((6, b.tables.shape[1]), -1, np.int32)
    tables[perm] = b.tables
    b.check(b.run(seq_bt_row=i32(perm), tables=tables))


def test_attention_again_on_the_same_plan():
    """Every layer of a step reuses the plan and the workspace: the counters are back at zero after
    each call, in both layers, for split sequences and prefill chunks."""
    b = Batch([1, 1, 130], [5003, 37, 900], 2, BF, seed=12)
    S, T = len(b.q_lens), b.T
    q, cache, cu, kv = b.q.to(dev), torch.from_numpy(b.cache).to(dev), i32(b.cu), i32(b.kv_lens)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = torch.zeros(K.attention_workspace_size(S, T, 2), dtype=torch.uint8, device=dev)
    K.attention_plan(cu, kv, S, 2, S, T, ws, err)
    first = {}
    for rep in range(3):
        for layer in (0, 1):
            out = torch.zeros_like(q)
            K.varlen_attention_q4(q, out, cache, layer, i32(b.tables), cu, kv, S, S, T, ws, err=err)
            b.layer = layer
            b.check(out)
            if layer in first:
                # no result depends on which CTA came last
                assert torch.equal(out, first[layer])
            first[layer] = out
    assert int(err.item()) == 0


@pytest.mark.parametrize("dt", [F32, BF])
def test_attention_bad_block_is_reported(dt):
    b = Batch([1, 3], [40, 50], 2, dt, seed=7)
    b.tables[0, 1] = b.cache.shape[1]
    b.tables[1, 0] = -1
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    with pytest.raises(AssertionError, match="out of range"):
        b.run(err=err)
    assert int(err.item()) == K.DEV_BOUNDS


@pytest.mark.parametrize("dt", [F32, BF])
def test_write_then_attend(dt):
    """The cache as the step uses it: a prompt written in two chunks, then decode tokens one at
    a time, each attending to everything written before it."""
    g = torch.Generator().manual_seed(8)
    heads, nb, n = 2, 12, 75
    k, v = rows(g, n, heads).to(dt), rows(g, n, heads).to(dt)
    table = torch.randperm(nb, generator=g)[:-(-n // 16)].numpy()[None].astype(np.int32)
    slot = table[0][np.arange(n) // 16] * 16 + np.arange(n) % 16
    cache = K.kv_cache_q4(1, nb, heads)
    b = Batch([1], [1], heads, dt)
    b.layer, b.tables, at = 0, table, 0
    for step in (50, 21, 1, 1, 1, 1):
        s = slice(at, at + step)
        K.kv_append_q4(k[s].to(dev), v[s].to(dev), i32(slot[s]), cache[0])
        at += step
        b.cache = cache.cpu().numpy()
        b.q = torch.randn(step, 4 * heads, 128, generator=g).to(dt)
        b.T, b.q_lens, b.kv_lens, b.cu = step, [step], [at], np.array([0, step], np.int32)
        b.check(b.run())
    ref = np.zeros((nb, heads, 2, q4.TILE_BYTES), np.uint8)
    q4.append(ref, k.float().numpy(), v.float().numpy(), slot)
    assert np.array_equal(b.cache[0], ref)
