"""The engine on a 4-bit KV cache: a step writes, attends and samples over it (run on a B200)."""
import numpy as np
import pytest
import torch

from hayate_b200 import kernels as K
from hayate_b200 import weights as W
from hayate_b200.config import EngineConfig, TINY
from hayate_b200.engine import Engine
from oracle import q4
from oracle import reference as R

pytestmark = pytest.mark.gpu
STD = 0.15


def engine(dtype=torch.float32, graphs=True, **kw):
    kw = dict(max_num_seqs=16, max_batched_tokens=256, prefill_chunk=48, num_kv_blocks=512,
              max_model_len=1024, cuda_graphs=graphs, kv_cache_dtype="int4") | kw
    return Engine("tiny", model_config=TINY, engine_config=EngineConfig(**kw), dtype=dtype,
                  weights=W.exact_seeded(TINY, 0, std=STD))


def prompts(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(1, TINY.vocab_size, (n,), generator=g).tolist() for n in lens]


def reference_tokens(monkeypatch, ps, n):
    """The reference's step loop with every key and value rounded to what the cache holds:
    (tokens, top-two margins) of each request."""
    plain = R.sdpa_gqa

    def rounded(x):
        return torch.from_numpy(q4.values(*q4.quantise(x.numpy())).astype(np.float32))

    monkeypatch.setattr(R, "sdpa_gqa", lambda q, k, v, mask: plain(q, rounded(k), rounded(v), mask))
    ref = R.RefEngine(R.RefWeights.from_host(W.exact_seeded(TINY, 0, std=STD), torch.float32),
                      record_margins=True)
    return [(r.tokens, r.margins) for r in ref.run(ps, n)]


def assert_same_while_clear(got, want, margin=0.15):
    """Tokens agree up to the first step whose two best logits nearly tie: a key within an fp32
    rounding of a code's border may take the neighbouring code, which moves the logits a little."""
    compared = 0
    for r, (tokens, margins) in zip(got, want):
        for a, b, m in zip(r.tokens, tokens, margins):
            if m <= margin:
                break
            assert a == b
            compared += 1
    return compared


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("caching", [False, True])
def test_tokens_follow_the_reference_on_a_rounded_cache(monkeypatch, graphs, caching):
    ps = prompts([5, 16, 17, 130, 200])
    ps += [ps[4][:160] + p for p in prompts([3, 30], seed=1)]       # a shared prefix of 10 blocks
    want = reference_tokens(monkeypatch, ps, 12)
    eng = engine(graphs=graphs, prefix_caching=caching)
    got = eng.generate_text(ps[:5], max_tokens=12) + eng.generate_text(ps[5:], max_tokens=12)
    assert all(len(r.tokens) == 12 for r in got)
    # how many tokens that compares is set by the reference's margins alone
    assert assert_same_while_clear(got, want) >= 10
    assert eng.check_device_errors() == 0
    assert (eng.graph_steps > 0) == graphs
    if caching:
        assert eng.prompt_tokens_computed < sum(map(len, ps))


def test_bf16_graph_steps_give_the_eager_tokens():
    ps = prompts([3, 40, 333, 90, 64, 7], seed=2)
    runs = []
    for graphs in (True, False):
        eng = engine(torch.bfloat16, graphs)
        runs.append([r.tokens for r in eng.generate_text(ps, max_tokens=24)])
        assert eng.check_device_errors() == 0
    assert runs[0] == runs[1]


def test_blocks_are_reused():
    """A pool that holds a few requests at a time: rows of earlier owners are overwritten."""
    ps = prompts([100, 120, 90, 60, 110, 80, 100, 75], seed=3)
    eng = engine(torch.bfloat16, num_kv_blocks=24)
    assert [len(r.tokens) for r in eng.generate_text(ps, max_tokens=8)] == [8] * 8
    again = eng.generate_text(ps[0], max_tokens=8).tokens
    assert again == engine(torch.bfloat16).generate_text(ps[0], max_tokens=8).tokens
    assert eng.check_device_errors() == 0


def test_the_pool_holds_more_blocks():
    """Sized from device memory, the 4-bit pool holds 32 / 9 as many blocks as the bf16 one."""
    counts = []
    for kind in ("auto", "int4"):
        e = engine(torch.bfloat16, kv_cache_dtype=kind)
        counts.append(e.runner._blocks_from_memory())
        assert e.runner.kv_cache.dtype == (torch.uint8 if kind == "int4" else torch.bfloat16)
        del e
        torch.cuda.empty_cache()
    assert 3.4 < counts[1] / counts[0] < 3.7


def test_kernel_count_of_a_decode_step():
    eng = engine(torch.bfloat16)
    eng.generate_text(prompts([20]), max_tokens=2)
    per = eng.runner.launches_per_step()
    before = eng.runner.kernel_launches
    eng._write_sched([(eng.scheduler.pad_slot, 0, 1, 1)])
    eng.runner.launch_step(1, 1, 1)
    torch.cuda.synchronize()
    assert eng.runner.kernel_launches - before == per
    assert tuple(eng.runner.kv_cache.shape[-2:]) == (2, K.Q4_TILE_BYTES)
