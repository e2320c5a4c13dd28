"""The engine harness on the 4-bit KV pool: the store, the prefill tables built on the GPU, extend
and decode run together as a serving step uses them.

fp32 greedy tokens are compared with a float64 full recomputation whose keys and values pass
through the pool's format (oracle.fp4.roundtrip).
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _oracle(model):
    from oracle import fp4 as F
    from oracle.engine import OracleQwen3

    class Fp4Qwen3(OracleQwen3):
        def cached(self, k, v):
            return F.roundtrip(k), F.roundtrip(v)

    return Fp4Qwen3(model)


@pytest.mark.parametrize("page_size,overlap,graphs,device_meta", [(16, True, True, True), (1, True, True, True),
                                                                  (4, False, False, True), (16, True, False, False)])
def test_engine_fp32_tokens_match_the_quantised_oracle(page_size, overlap, graphs, device_meta):
    from minisgl_b200 import FP4KVCache
    from minisgl_b200.core import SamplingParams
    from minisgl_b200.engine import LLM, EngineConfig, tiny_spec

    rng = np.random.default_rng(4)
    a = rng.integers(0, 500, 120).astype(np.int32)
    prompts = [a, np.concatenate([a[:96], rng.integers(0, 500, 30).astype(np.int32)]),
               rng.integers(0, 500, 300).astype(np.int32),  # chunked over several prefill steps
               rng.integers(0, 500, 1).astype(np.int32)]
    max_tokens = [9, 12, 8, 10]
    cfg = EngineConfig(spec=tiny_spec(num_layers=2, vocab_size=500), dtype="float32", max_running_req=4,
                       page_size=page_size, num_tokens=4096, max_extend_tokens=128, overlap_scheduling=overlap,
                       cuda_graph_max_bs=4 if graphs else 0, device_metadata=device_meta, kv_cache_dtype="fp4")
    llm = LLM(cfg)
    assert isinstance(llm.engine.kv_cache, FP4KVCache)
    outs = llm.generate(prompts, [SamplingParams(max_tokens=n, ignore_eos=True) for n in max_tokens])
    got = [o["token_ids"] for o in outs]
    assert got == _oracle(llm.engine.model).generate(prompts, max_tokens)
    llm.cache.check_integrity()
    llm.engine.shutdown()


def test_engine_bf16_runs_clean_and_repeats():
    """bf16 over the 4-bit pool: every request gets its tokens, twice the same ones, in fewer pool bytes."""
    from minisgl_b200.core import SamplingParams
    from minisgl_b200.engine import LLM, EngineConfig, tiny_spec

    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, 500, int(n)).astype(np.int32) for n in rng.integers(1, 700, 24)]
    sp = SamplingParams(max_tokens=20, ignore_eos=True)
    runs, nbytes = [], {}
    for kind in ("fp4", "fp4", "auto"):
        llm = LLM(EngineConfig(spec=tiny_spec(num_layers=2, vocab_size=500), max_running_req=16, num_tokens=16384,
                               max_extend_tokens=1024, kv_cache_dtype=kind))
        outs = [o["token_ids"] for o in llm.generate(prompts, sp)]
        assert all(len(o) == 20 for o in outs)
        runs.append(outs)
        nbytes[kind] = llm.engine.kv_cache.nbytes
        llm.cache.check_integrity()
        llm.engine.shutdown()
    assert runs[0] == runs[1]
    assert nbytes["fp4"] * 3.5 <= nbytes["auto"]


def test_unknown_pool_is_refused():
    from minisgl_b200.engine import LLM, EngineConfig, tiny_spec

    with pytest.raises(ValueError, match="kv_cache_dtype"):
        LLM(EngineConfig(spec=tiny_spec(num_layers=1, vocab_size=100), num_tokens=256, kv_cache_dtype="int3"))
