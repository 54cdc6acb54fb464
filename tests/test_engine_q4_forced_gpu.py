"""The engine on a 4-bit KV cache, fed the reference's tokens, so that every step is compared and not
only those before the first near-tie (run on a B200)."""
import pytest
import torch

from hayate_b200 import weights as W
from hayate_b200.config import EngineConfig, TINY
from hayate_b200.engine import Engine
from test_engine_q4_gpu import STD, prompts, reference_tokens

pytestmark = pytest.mark.gpu


class Forced(Engine):
    """Commits the tokens of `script` and keeps what it would have chosen."""

    def sample(self, logits):
        assert logits.shape[0] == 1
        self.chosen.append(int(super().sample(logits)))
        return torch.full((1, 1), self.script[len(self.chosen) - 1], dtype=torch.int64, device=logits.device)


@pytest.mark.parametrize("chunk", [48, 256])
def test_every_clear_step_chooses_the_reference_s_token(monkeypatch, chunk):
    ps = prompts([5, 16, 17, 130, 200])
    ps += [ps[4][:160] + p for p in prompts([3, 30], seed=1)]
    want = reference_tokens(monkeypatch, ps, 12)
    eng = Forced("tiny", model_config=TINY, dtype=torch.float32, weights=W.exact_seeded(TINY, 0, std=STD),
                 engine_config=EngineConfig(max_num_seqs=4, max_batched_tokens=256, prefill_chunk=chunk,
                                            num_kv_blocks=64, max_model_len=1024, kv_cache_dtype="int4"))
    compared = 0
    for p, (tokens, margins) in zip(ps, want):
        eng.script, eng.chosen = tokens, []
        assert eng.generate_text(p, max_tokens=12).tokens == tokens
        for got, token, margin in zip(eng.chosen, tokens, margins):
            # a key within an fp32 rounding of a code's border may take the neighbouring code,
            # which moves the logits a little
            if margin > 0.15:
                assert got == token
                compared += 1
    assert compared == sum(m > 0.15 for _, margins in want for m in margins) >= 60      # of 84
    assert eng.check_device_errors() == 0
