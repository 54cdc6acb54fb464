"""The bf16 cache's attention on sequences whose query rows q does not have (run on a B200)."""
import pytest
import torch

from helpers import random_paged_batch, reference_attention
from hayate_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_lens,kv_lens,rows", [
    ([1, 1, 1], [300, 40, 900], 2),                      # a CTA per pair
    ([1] * 40, [700 + i for i in range(40)], 30),        # decode items split over all warps
    ([70, 130], [300, 900], 100), ([512], [4000], 511),  # prefill, also in pieces
    ([1, 40, 1, 17], [300, 40, 2049, 100], 58),          # both
])
def test_rows_that_q_does_not_have_are_reported(q_lens, kv_lens, rows):
    """Nothing is written, behind out least of all, also by a call that began its loads early; the
    plan serves a whole q afterwards."""
    b = random_paged_batch(q_lens, kv_lens, kv_heads=2, seed=rows)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.zeros(K.attention_workspace_size(b["S"], b["T"], 2), dtype=torch.uint8, device="cuda")
    guard = torch.full_like(b["q"], 7.0)

    def attend(n, early):
        K.varlen_attention(b["q"][:n], guard[:n], b["cache"], b["layer"], b["bt"], b["cu"], b["kv"], b["S"],
                           b["S"], b["T"], ws, err=err, early=early)
        return int(err.item())

    for n, start in ((rows, 0), (b["T"] - 1, 0), (b["T"], -1), (b["T"], 1)):
        b["cu"] += start
        K.attention_plan(b["cu"], b["kv"], b["S"], 2, b["S"], b["T"], ws, err)
        for early in (False, True):
            assert attend(n, early) == K.DEV_BOUNDS, (n, start)
            assert (guard == 7.0).all()
            err.zero_()
        b["cu"] -= start
    K.attention_plan(b["cu"], b["kv"], b["S"], 2, b["S"], b["T"], ws, err)
    want = reference_attention(b)
    torch.cuda.synchronize()
    for n, early in ((b["T"], False), (rows, True), (b["T"], True)):
        if n == rows:
            before = guard.clone()
            assert attend(n, early) == K.DEV_BOUNDS and torch.equal(guard, before)
            err.zero_()
            guard.fill_(7.0)
        else:
            assert attend(n, early) == 0
            # weights and output rounded to bf16 (2^-8 each) of values of a few units
            assert (guard.float() - want).abs().max().item() <= 2e-2
