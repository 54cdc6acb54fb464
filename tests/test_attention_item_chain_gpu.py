"""Prefill steps in which a CTA runs several items in a row, loading the next item's Q and first key
tiles while the last one ends (run on a B200)."""
import pytest
import torch

from helpers import random_paged_batch
from hayate_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_lens,kv_lens,reps", [
    ([512] * 16, [512 + 224 * i for i in range(16)], 400),
    ([64 + 7 * i for i in range(40)], [64 + 7 * i + 31 * (i % 5) for i in range(40)], 1500),
])
def test_no_wait_runs_out_between_items(q_lens, kv_lens, reps):
    b = random_paged_batch(q_lens, kv_lens, kv_heads=8, seed=3)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.zeros(K.attention_workspace_size(b["S"], b["T"], 8), dtype=torch.uint8, device="cuda")
    K.attention_plan(b["cu"], b["kv"], b["S"], 8, b["S"], b["T"], ws, err)
    first, out, differ = None, torch.empty_like(b["q"]), torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(reps):
        K.varlen_attention(b["q"], out, b["cache"], b["layer"], b["bt"], b["cu"], b["kv"], b["S"],
                           b["S"], b["T"], ws, err=err)
        first = out.clone() if first is None else first
        differ += (out != first).any()
    assert int(err.item()) == 0, K.describe_error(int(err.item()))
    assert int(differ.item()) == 0
