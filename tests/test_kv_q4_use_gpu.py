"""The 4-bit KV cache's kernels as a serving program calls them: captured, on other streams, on
shared workspaces, beside the bf16 cache's attention, at the far ends of the sizes (run on a B200)."""
import numpy as np
import pytest
import torch

from hayate_b200 import kernels as K
from oracle import q4
from test_kv_q4_gpu import BF, F32, Batch, dev, i32, random_cache, rows

pytestmark = pytest.mark.gpu


class Step:
    """One batch's tensors on the device, its plan and workspace."""

    def __init__(self, b, max_seqs=None, max_tokens=None, ws=None):
        self.b, self.S, self.T = b, len(b.q_lens), b.q.shape[0]
        self.max = (max_seqs or self.S, max_tokens or self.T)
        self.q, self.cache = b.q.to(dev), torch.from_numpy(b.cache).to(dev)
        self.tables, self.cu, self.kv = i32(b.tables), i32(b.cu), i32(b.kv_lens)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        self.ws = ws if ws is not None else torch.zeros(
            K.attention_workspace_size(*self.max, b.heads), dtype=torch.uint8, device=dev)
        self.out = torch.full_like(self.q, 7.0)

    def plan(self):
        K.attention_plan(self.cu, self.kv, self.S, self.b.heads, *self.max, self.ws, self.err)

    def attend(self, layer=None):
        K.varlen_attention_q4(self.q, self.out, self.cache, self.b.layer if layer is None else layer,
                              self.tables, self.cu, self.kv, self.S, *self.max, self.ws, err=self.err)

    def check(self):
        torch.cuda.synchronize()
        assert int(self.err.item()) == 0, K.describe_error(int(self.err.item()))
        self.b.check(self.out)


# ------------------------------------------------------------ NaN in places a row does not see
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("q_len,kv_len,at", [(70, 333, 300), (64, 64, 63), (130, 1000, 880), (1, 500, 100),
                                             (512, 4600, 4200)])
def test_nan_rows_reach_only_the_rows_that_see_them(q_len, kv_len, at, dt):
    """A NaN key makes every output of the query rows that see it NaN, a NaN in half of a value that
    half; the rows before, the other half and the other head keep the bits they have without it."""
    b = Batch([q_len], [kv_len], 2, dt, seed=at)
    clean = b.run()
    b.check(clean)
    first = at - (kv_len - q_len)                        # the first query row that sees key `at`
    sees = torch.arange(q_len, device=dev) >= first
    blk = b.tables[0, at // 16]
    for part, half in ((1, 0), (1, 1), (0, 1)):
        p = q4.CODE_BYTES + 8 * (at % 16) + 4 * half
        keep = b.cache[b.layer, blk, 1, part, p:p + 4].copy()
        b.cache[b.layer, blk, 1, part, p:p + 4] = np.frombuffer(np.float16([np.nan, np.nan]).tobytes(), np.uint8)
        out = b.run()
        b.cache[b.layer, blk, 1, part, p:p + 4] = keep
        want = torch.zeros(q_len, 8, 128, dtype=torch.bool, device=dev)
        want[sees, 4:, 64 * half if part else 0:64 * half + 64 if part else 128] = True
        assert torch.equal(torch.isnan(out), want), (part, half)
        assert torch.equal(out[~want], clean[~want]), (part, half)


# ------------------------------------------------------------ sizes
@pytest.mark.parametrize("heads,q_lens,kv_lens", [
    (1, [1] * 1100, [1 + 7 * i % 90 for i in range(1100)]),           # more sequences than CTAs and than 32^2
    (2, [1, 0, 3] * 120, [1 + i % 40 + (i % 3) * 2 for i in range(360)]),
    (1, [1] * 300 + [100], [1 + 11 * i % 300 for i in range(300)] + [900]),
    (2, [0] * 80 + [70, 1], [3] * 80 + [1500, 600]), (8, [0, 2, 0, 1, 2, 0, 1], [9, 2, 5, 700, 33, 1, 1]),
    (1, [1], [100003]), (1, [70], [30011]), (2, [1] * 33 + [5], [40] * 33 + [20000]),
])
def test_attention_many_and_long_sequences(heads, q_lens, kv_lens):
    b = Batch(q_lens, kv_lens, heads, BF, layers=1, layer=0, seed=len(q_lens))
    b.check(b.run())


def test_attention_many_sequences_fp32():
    b = Batch([1, 0, 2] * 70, [2 + i % 40 for i in range(210)], 1, F32, layers=1, layer=0, seed=3)
    b.check(b.run())


def test_attention_more_than_64_layers():
    """Layers 64 apart share the counters of the work they hand out."""
    b = Batch([1, 70, 1], [90, 200, 400], 1, BF, layers=66, seed=16)
    s = Step(b)
    s.plan()
    for layer in (0, 64, 1, 65, 64):
        s.attend(layer)
        b.layer = layer
        s.check()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("lens", [([1, 1], [40, 7]), ([70], [170]), ([1, 40], [90, 40])])
def test_attention_offsets_past_32_bits(lens, dt):
    """A layer of more than 4 GB: blocks at its end, in its second layer."""
    heads = 8
    b = Batch(*lens, heads, dt, layers=1, layer=0, seed=21)
    s = Step(b)
    n = b.cache.shape[1]
    nb = (1 << 32) // (heads * 2 * q4.TILE_BYTES) + n + 3
    big = torch.empty(2, nb, heads, 2, q4.TILE_BYTES, dtype=torch.uint8, device=dev)
    big[1, nb - n:] = s.cache[0]
    s.cache, s.tables = big, torch.where(s.tables >= 0, s.tables + (nb - n), -1).contiguous()
    s.plan()
    s.attend(1)
    s.check()


def test_padding_rows_behind_a_decode_step():
    """More rows than sequences, though every sequence decodes one token."""
    b = Batch([1, 1, 0, 1, 1], [5003, 37, 8, 1, 640], 2, BF, seed=25, pad_rows=9)
    s = Step(b)
    s.plan()
    for layer in (0, 1, 0):
        s.out.fill_(7.0)
        s.attend(layer)
        b.layer = layer
        s.check()
        assert (s.out[b.T:] == 7.0).all()


@pytest.mark.parametrize("q_lens,kv_lens", [
    ([512, 300] + [1] * 60, [2500, 900] + [100 + 61 * i for i in range(60)]),    # both kinds of work on most CTAs
    ([64] + [1] * 40, [64] + [4000 - 90 * i for i in range(40)]), ([512] * 4 + [1], [3000] * 4 + [50])])
def test_prefill_beside_decodes(q_lens, kv_lens):
    b = Batch(q_lens, kv_lens, 8, BF, layers=2, layer=0, seed=26)
    s = Step(b)
    s.plan()
    first = None
    for _ in range(6):
        s.out.fill_(7.0)
        s.attend()
        first = s.out.clone() if first is None else first
        assert torch.equal(s.out, first)
    s.check()


def test_capacities_above_the_batch():
    b = Batch([1, 40, 1], [300, 90, 17], 2, BF, seed=22, pad_rows=3)
    s = Step(b, max_seqs=200, max_tokens=4000)
    s.plan()
    s.attend()
    s.check()
    assert (s.out[b.T:] == 7.0).all()


# ------------------------------------------------------------ streams, graphs, shared workspaces
def test_two_streams_at_once():
    """Calls on two streams, each with its own workspace."""
    steps = [Step(Batch(*lens, 2, BF, seed=i)) for i, lens in enumerate(
        [([1] * 9, [3000 - 211 * i for i in range(9)]), ([130, 1], [700, 400])])]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                s.plan()
                s.attend()
    for s in steps:
        s.check()


def test_alternating_with_the_bf16_cache_on_one_plan():
    """Both caches' attention on the same plan and workspace, in turn: neither leaves the other
    counters or cached ids that it does not expect."""
    b = Batch([1, 1, 100], [2500, 37, 300], 2, BF, seed=24)
    s = Step(b)
    n = b.cache.shape[1]
    g = torch.Generator().manual_seed(1)
    dense = torch.randn(1, n, 2, 2, 16, 128, generator=g).to(BF).to(dev)
    alone = torch.zeros_like(s.q)

    def bf16(out):
        K.varlen_attention(s.q, out, dense, 0, s.tables, s.cu, s.kv, s.S, *s.max, s.ws, err=s.err)

    s.plan()
    bf16(alone)
    for _ in range(3):
        s.out.fill_(7.0)
        s.attend()
        s.check()
        got = torch.zeros_like(s.q)
        bf16(got)
        assert torch.equal(got, alone)
    s.plan()                                            # and the 4-bit cache's first
    s.attend()
    s.check()
    got = torch.zeros_like(s.q)
    bf16(got)
    assert torch.equal(got, alone)


@pytest.mark.parametrize("dt", [F32, BF])
def test_captured_step_replays_with_new_inputs(dt):
    """Write, plan, attention and read-back in a graph; a second graph of another batch on the same
    workspace and cache is replayed in between."""
    heads, nb = 2, 40
    g = torch.Generator().manual_seed(30)
    table = torch.randperm(nb, generator=g)[:36].view(3, 12).numpy().astype(np.int32)
    lens0 = [100, 20, 60]
    base = random_cache(g, 1, nb, heads)
    cache = torch.from_numpy(base.copy()).to(dev)
    tables = i32(table)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = torch.zeros(K.attention_workspace_size(3, 64, heads), dtype=torch.uint8, device=dev)

    class Graph:
        def __init__(self, q_lens):
            T = sum(q_lens)
            self.q_lens, self.T = q_lens, T
            self.k, self.v = (torch.zeros(T, heads, 128, dtype=dt, device=dev) for _ in range(2))
            self.q = torch.zeros(T, 4 * heads, 128, dtype=dt, device=dev)
            self.out = torch.zeros_like(self.q)
            self.slots, self.kv = i32([-1] * T), i32(q_lens)
            self.cu = i32(np.concatenate([[0], np.cumsum(q_lens)]))
            self.back = tuple(torch.zeros_like(self.k) for _ in range(2))
            self.run()                                   # as the engine does, once before the capture
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.run()

        def run(self):
            K.kv_append_q4(self.k, self.v, self.slots, cache[0], err=err)
            K.attention_plan(self.cu, self.kv, 3, heads, 3, 64, ws, err)
            K.varlen_attention_q4(self.q, self.out, cache, 0, tables, self.cu, self.kv, 3, 3, 64, ws, err=err)
            K.kv_read_q4(cache[0], self.slots, dt, *self.back, err=err)

    graphs = [Graph([1, 1, 1]), Graph([1, 30, 20])]
    lens = list(lens0)
    for turn in range(6):
        gr = graphs[turn % 2]
        k, v = rows(g, gr.T, heads).to(dt), rows(g, gr.T, heads).to(dt)
        q = torch.randn(gr.T, 4 * heads, 128, generator=g).to(dt)
        slots = np.concatenate([table[i][np.arange(n, n + m) // 16] * 16 + np.arange(n, n + m) % 16
                                for i, (n, m) in enumerate(zip(lens, gr.q_lens))]).astype(np.int32)
        lens = [n + m for n, m in zip(lens, gr.q_lens)]
        for dst, src in ((gr.k, k), (gr.v, v), (gr.q, q), (gr.slots, i32(slots)), (gr.kv, i32(lens))):
            dst.copy_(src)
        gr.graph.replay()
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        q4.append(base[0], k.float().numpy(), v.float().numpy(), slots)
        assert np.array_equal(cache.cpu().numpy(), base)
        for got, want in zip(gr.back, q4.read(base[0], slots)):
            assert torch.equal(got.cpu(), torch.from_numpy(want).float().to(dt))
        b = Batch([1], [1], heads, dt)
        b.cache, b.layer, b.tables, b.q, b.T = base, 0, table, q, gr.T
        b.q_lens, b.kv_lens = gr.q_lens, lens
        b.check(gr.out)
        if turn == 3:
            lens = list(lens0)                           # over the same slots again


# ------------------------------------------------------------ arguments
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("q_lens,kv_lens", [
    ([1, 3], [200, 30]), ([70, 1], [300, 30]), ([5, 1], [3, 30]), ([1, 1], [0, 30]), ([1, 1], [200000, 30]),
    ([70, 1], [1 << 24, 30]), ([1, 1], [2 ** 31 - 1, 30]), ([70, 70], [2 ** 31 - 1, 70]),
    ([70, 64], [2 ** 31 - 1, 64])])
def test_sequences_that_do_not_fit_are_reported(q_lens, kv_lens, dt):
    """Longer than the block-table row, or fewer keys than query tokens: reported, the others right."""
    b = Batch(q_lens, [min(kv, 64) for kv in kv_lens], 2, dt, seed=31)
    s = Step(b)
    s.tables = s.tables[:, :4].contiguous()
    s.kv = i32(kv_lens)
    s.plan()
    s.attend()
    assert int(s.err.item()) == K.DEV_BOUNDS
    if dt == BF and any(not q <= kv <= 1 << 28 for q, kv in zip(q_lens, kv_lens)):
        assert (s.out == 7.0).all()                      # the plan refuses the whole batch
    elif kv_lens[1] <= 64:                               # the second sequence fits its row
        b.kv_lens = [max(q_lens[0], min(kv_lens[0], 64)), kv_lens[1]]
        want = q4.attention(b.q.float().numpy(), b.cache[b.layer], b.tables, q_lens, b.kv_lens, 128 ** -0.5)[0]
        off = np.abs(s.out.double().cpu().numpy() - want)[q_lens[0]:].max()
        assert off < 0.05                                # values are a few units: not another sequence's


@pytest.mark.parametrize("dt", [F32, BF])
def test_read_into_given_tensors_and_nothing_to_do(dt):
    g = torch.Generator().manual_seed(32)
    cache = torch.from_numpy(random_cache(g, 1, 3, 2)[0]).to(dev)
    slots = i32([5, -1, 40])
    want = K.kv_read_q4(cache, slots, dt)
    ko, vo = (torch.full((3, 2, 128), 9.0, dtype=dt, device=dev) for _ in range(2))
    got = K.kv_read_q4(cache, slots, dt, ko, vo)
    assert got[0] is ko and got[1] is vo
    assert torch.equal(ko, want[0]) and torch.equal(vo, want[1])
    before = cache.clone()
    none = torch.zeros(0, 2, 128, dtype=dt, device=dev)
    K.kv_append_q4(none, none, slots[:0], cache)
    K.kv_append_q4(ko, vo, i32([-1, -1, -1]), cache)
    e, f = K.kv_read_q4(cache, slots[:0], dt)
    assert e.shape == f.shape == (0, 2, 128) and torch.equal(cache, before)


def test_bf16_attention_refuses_a_workspace_that_does_not_fit():
    s = Step(Batch([1, 3], [30, 40], 2, BF))
    s.plan()
    torch.cuda.synchronize()

    def call(ws=s.ws, seqs=2, max_seqs=2, max_tokens=4):
        K.varlen_attention_q4(s.q, s.out, s.cache, 0, s.tables, s.cu, s.kv, seqs, max_seqs, max_tokens, ws)

    call()
    for kw in (dict(ws=None), dict(ws=s.ws[:-256]), dict(ws=s.ws[16:]), dict(seqs=2, max_seqs=1),
               dict(max_tokens=3)):
        with pytest.raises(Exception):
            call(**kw)
    for bad in (s.cu[:2], s.cu.cpu(), s.cu.long()):
        with pytest.raises(ValueError):
            K.varlen_attention_q4(s.q, s.out, s.cache, 0, s.tables, bad, s.kv, 2, 2, 4, s.ws)
    with pytest.raises(ValueError):
        K.varlen_attention_q4(s.q, s.out, s.cache, 0, s.tables[:1], s.cu, s.kv, 2, 2, 4, s.ws)
    with pytest.raises(ValueError):
        K.varlen_attention_q4(s.q, s.out.float(), s.cache, 0, s.tables, s.cu, s.kv, 2, 2, 4, s.ws)
