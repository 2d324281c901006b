"""Arguments that the runner refuses before it allocates anything."""
import importlib
from types import SimpleNamespace

import pytest


@pytest.mark.parametrize("kw", [
    dict(kv_cache_dtype="fp8_block", kv_group=48),
    dict(kv_cache_dtype="fp8_block", kv_group=16),
    dict(kv_cache_dtype="fp8_block", kv_group=64, block_size=96),
    dict(kv_cache_dtype="fp8_block", k_scale=0.5),
    dict(kv_cache_dtype="fp8_block", v_scale=0.5),
    dict(logprobs=33), dict(logprobs=-1),
])
def test_refused(kw):
    sr = importlib.import_module("hilda-vllm_amd.engine.spec_runner")
    model = SimpleNamespace(g=SimpleNamespace(vocab=1000))
    with pytest.raises(ValueError):
        sr.SpecRunner(model, model, batch=1, gamma=2, **kw)
