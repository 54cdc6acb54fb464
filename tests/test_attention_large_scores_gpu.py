"""Prefill attention on rows of large scores, whose running maximum grows over many key tiles, so
that the output is rescaled while products are in flight (run on a B200)."""
import pytest
import torch

from helpers import random_paged_batch
from hayate_b200 import kernels as K

pytestmark = pytest.mark.gpu


def exact(b):
    """float64 attention and the sum of p |v| of every output."""
    out, mag = [], []
    for i in range(b["S"]):
        q = b["q"][b["cu_list"][i]:b["cu_list"][i + 1]].double().transpose(0, 1)     # (Hq, T, 128)
        k, v = (x[i].double().permute(1, 0, 2).repeat_interleave(4, 0) for x in (b["ctx_k"], b["ctx_v"]))
        s = q @ k.transpose(1, 2) / 128 ** 0.5
        hidden = torch.ones(s.shape[1:], dtype=torch.bool, device=s.device).triu(s.shape[2] - s.shape[1] + 1)
        p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
        out.append((p @ v).transpose(0, 1))
        mag.append((p @ v.abs()).transpose(0, 1))
    return torch.cat(out), torch.cat(mag)


@pytest.mark.parametrize("q_lens,kv_lens,heads", [([130, 512], [700, 1111], 2), ([512] * 4, [1000] * 4, 8)])
@pytest.mark.parametrize("qscale", [8.0, 20.0])
def test_prefill_of_large_scores(q_lens, kv_lens, heads, qscale):
    b = random_paged_batch(q_lens, kv_lens, kv_heads=heads, seed=11)
    b["q"] = b["q"] * qscale
    want, mag = exact(b)
    # weights and output are each rounded once to bf16 (2^-8); scores of a few hundred are
    # off by their fp32 sums' roundings (2^-24 of each of 128 terms of up to 20 x 4 x 4)
    tol = 2.0 ** -8 * (want.abs() + mag) + mag * 1e-3
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    first = None
    for _ in range(10):
        out = torch.empty_like(b["q"])
        ws = torch.zeros(K.attention_workspace_size(b["S"], b["T"], heads), dtype=torch.uint8,
                         device="cuda")
        K.attention_plan(b["cu"], b["kv"], b["S"], heads, b["S"], b["T"], ws, err)
        K.varlen_attention(b["q"], out, b["cache"], b["layer"], b["bt"], b["cu"], b["kv"], b["S"],
                           b["S"], b["T"], ws, err=err)
        first = out if first is None else first
        assert torch.equal(out, first)                 # no result depends on timing
        worst = ((out.double() - want).abs() - tol).max().item()
        assert worst <= 0, worst
    assert int(err.item()) == 0
