"""The 4-bit cache's attention and its plan: rows that q does not have, workspaces that hold another
batch's plan or none, and sequences as the plan has them (run on a B200)."""
import pytest
import torch

from hayate_b200 import kernels as K
from hayate_b200._lib import HayateError
from test_kv_q4_gpu import BF, F32, Batch, dev, i32
from test_kv_q4_use_gpu import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("q_lens,kv_lens,rows", [
    ([1, 1, 1], [40, 33, 300], 2),                       # a CTA per pair
    ([1, 1, 1], [40, 33, 5000], 2),                      # pairs over several CTAs
    ([1, 3, 0, 0, 0], [40, 50, 9, 9, 9], 3),             # a longer chunk in a step of few rows
    ([70, 130], [300, 900], 100), ([64, 512], [64, 4000], 200),
    ([130, 1, 1, 1], [700, 40, 3000, 17], 131), ([130, 1, 1, 1], [700, 40, 3000, 17], 60),
])
def test_rows_that_q_does_not_have_are_reported(q_lens, kv_lens, rows, dt):
    """The sequences have more query tokens than q has rows, or rows before its first: nothing is
    written, behind out least of all, and the plan serves a whole q afterwards."""
    b = Batch(q_lens, kv_lens, 2, dt, seed=rows)
    s = Step(b)
    whole, guard, cu = s.q, torch.full_like(s.q, 7.0), s.cu.clone()
    for n, start in ((rows, 0), (b.T - 1, 0), (b.T, -1), (b.T, 1)):
        s.cu.copy_(cu + start)
        s.q, s.out = whole[:n], guard[:n]
        s.plan()
        s.attend()
        assert int(s.err.item()) == K.DEV_BOUNDS, (n, start)
        assert (guard == 7.0).all()
        s.err.zero_()
    s.cu.copy_(cu)
    s.q, s.out = whole, guard
    s.plan()
    for layer in (0, 1):
        s.attend(layer)
    s.check()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [40, 700]), ([1, 2, 0, 0, 0, 0], [40, 700, 1, 1, 1, 1]),
                                             ([70, 1], [300, 50])])
def test_rows_before_the_first_sequence_stay(q_lens, kv_lens, dt):
    b = Batch(q_lens, kv_lens, 2, dt, seed=3, pad_rows=2)
    s = Step(b)
    s.q = torch.cat([s.q[b.T:], s.q[:b.T]]).contiguous()
    s.cu += 2
    s.plan()
    s.attend()
    assert (s.out[:2] == 7.0).all()
    s.out = s.out[2:].contiguous()
    s.check()


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [40, 33, 300]), ([70, 1, 1], [300, 50, 900])])
def test_another_batch_s_plan_is_reported(q_lens, kv_lens):
    s = Step(Batch(q_lens, kv_lens, 2, BF, seed=4), max_seqs=4, max_tokens=100)
    S, T = s.S, s.T

    def attend(seqs=S, max_seqs=4, max_tokens=100):
        s.err.zero_()
        s.out.fill_(7.0)
        K.varlen_attention_q4(s.q, s.out, s.cache, s.b.layer, s.tables, s.cu, s.kv, seqs, max_seqs, max_tokens,
                              s.ws, err=s.err)
        return int(s.err.item())

    s.ws = torch.zeros(2 * s.ws.numel(), dtype=torch.uint8, device=dev)    # no size check stands in
    assert attend() == K.DEV_PLAN and (s.out == 7.0).all()                 # no plan yet
    s.plan()
    assert attend() == 0
    s.check()
    for kw in (dict(seqs=S - 1), dict(max_seqs=5), dict(max_tokens=200)):
        assert attend(**kw) == K.DEV_PLAN and (s.out == 7.0).all(), kw
    K.attention_plan(s.cu, s.kv, S, 1, 4, 100, s.ws, s.err)                # for one KV head
    assert attend() == K.DEV_PLAN and (s.out == 7.0).all()
    s.plan()
    assert attend() == 0
    s.check()


@pytest.mark.parametrize("q_lens,kv_lens", [
    ([1] * 5, [40, 700, 33, 2000, 64]), ([1, 1], [5003, 37]), ([130, 1, 1], [700, 40, 3000]),
    ([1, 3, 0, 0], [40, 50, 9, 9])])
def test_bf16_takes_the_sequences_from_the_plan(q_lens, kv_lens):
    """What the caller's arrays hold by the time of a call does not matter: its counts of key blocks
    and the sequences they belong to are of one plan."""
    s = Step(Batch(q_lens, kv_lens, 2, BF, seed=5))
    s.plan()
    keep = s.kv.clone(), s.cu.clone()
    for kv, cu in ((s.kv * 0 + 1, s.cu), (s.kv * 3, s.cu), (s.kv * 0 - 9, s.cu * 0), (s.kv, s.cu * 0 + 1000)):
        s.kv.copy_(kv)
        s.cu.copy_(cu)
        s.out.fill_(7.0)
        s.attend()
        s.check()
        s.kv.copy_(keep[0])
        s.cu.copy_(keep[1])


@pytest.mark.parametrize("dt", [F32, BF])
def test_no_tokens(dt):
    s = Step(Batch([1, 3], [40, 50], 2, dt, seed=6))
    s.q = s.out = torch.zeros(0, 8, 128, dtype=dt, device=dev)
    s.attend()
    assert int(s.err.item()) == 0


def test_each_refusal_of_a_workspace_says_why():
    s = Step(Batch([1, 3], [30, 40], 2, BF, seed=7))
    need = K.attention_workspace_size(2, 4, 2)
    room = torch.zeros(need + 512, dtype=torch.uint8, device=dev)
    assert room.data_ptr() % 256 == 0

    def call(ws, seqs=2, max_seqs=2, max_tokens=4):
        K.varlen_attention_q4(s.q, s.out, s.cache, 0, s.tables, s.cu, s.kv, seqs, max_seqs, max_tokens, ws, err=s.err)

    s.ws = room[256:]                                    # a slice of its own is as good as any
    s.plan()
    call(s.ws)
    assert int(s.err.item()) == 0
    for ws, kw, why in ((None, {}, "planned, 256-byte aligned"), (room[16:], {}, "planned, 256-byte aligned"),
                        (room[:need - 1], {}, "too small"), (room, dict(max_seqs=1), "above the workspace's"),
                        (room, dict(max_tokens=3), "above the workspace's")):
        with pytest.raises(HayateError, match=why):
            call(ws, **kw)
