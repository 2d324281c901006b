"""A quantised model's state on the GPU."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_state_of_a_quantised_model(cuda):
    """The state of a quantised model, LM head included, makes another model the same one,
    also by way of the host; a model that shares the weights has them too."""
    q3 = importlib.import_module("hilda-vllm_amd.engine.qwen3_host")
    print("state of a quantised model", flush=True)
    g = q3.Qwen3Geometry(num_layers=2, hidden=256, num_heads=2, num_kv_heads=1, ffn=384, vocab=301,
                         max_position=64)
    a = q3.Qwen3Host(g, device=cuda, seed=1).quantize_int4(64, lm_head=True)
    b = q3.Qwen3Host(g, device=cuda, seed=2).quantize_int4(64, lm_head=True)
    h = torch.randn(5, 256, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    want = a.compute_logits(h)
    assert not torch.equal(b.compute_logits(h), want)
    b.load_state_dict({k: v.cpu() for k, v in a.state_dict().items()})
    assert torch.equal(b.compute_logits(h), want)
    for n, p in a.named_parameters():
        assert torch.equal(p, b.get_parameter(n)), n
    moved = b.to("cpu").to(cuda)
    assert torch.equal(moved.compute_logits(h), want)
    shared = q3.Qwen3Host(g, device=cuda, share_from=a, num_layers=1)
    assert torch.equal(shared.compute_logits(h), want)
    assert shared.layers[0].qkv is a.layers[0].qkv


def test_packed_weights_set_by_the_caller(hv, cuda):
    """Codes that come from elsewhere, as plain Int4Weights in the model's places."""
    q3 = importlib.import_module("hilda-vllm_amd.engine.qwen3_host")
    print("packed weights set by the caller", flush=True)
    g = q3.Qwen3Geometry(num_layers=1, hidden=256, num_heads=2, num_kv_heads=1, ffn=384, vocab=301,
                         max_position=64)
    a = q3.Qwen3Host(g, device=cuda, seed=1)
    w = hv.ops.quantize_int4(a.lm_head, 64)
    h = torch.randn(5, 256, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    want = hv.ops.linear_int4(h, w)
    del a.lm_head
    a.lm_head = w
    assert torch.equal(a.compute_logits(h), want)
    a.quantize_int4(128, lm_head=True)  # leaves it as it is
    assert a.lm_head is w
