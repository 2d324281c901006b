"""4-bit weights as parts of a model (on the host)."""
import copy
import importlib

import pytest
import torch


def _layer(seed, ffn=384):
    q3 = importlib.import_module("hilda-vllm_amd.engine.qwen3_host")
    g = q3.Qwen3Geometry(num_layers=1, hidden=256, num_heads=2, num_kv_heads=1, ffn=ffn, vocab=64,
                         max_position=64)
    torch.manual_seed(seed)
    return q3.Qwen3Layer(g, "cpu", torch.bfloat16, q3.Rope(128, 64, 1e6, "cpu"))


def test_parameters_and_state(hv):
    """The quantised projections are among the layer's parameters and in its state, and a
    state goes into another layer of the same form."""
    a, b = _layer(1), _layer(2)
    plain = dict(a.named_parameters())
    a.quantize_int4(64)
    b.quantize_int4(64)
    names = {f"{n}.{part}" for n in ("qkv", "o", "gate_up", "down") for part in ("packed", "scales")}
    kept = {"q_norm", "k_norm", "ln1", "ln2"}
    assert set(dict(a.named_parameters())) == names | kept
    assert not any(p.requires_grad for p in a.parameters())
    state = a.state_dict()
    assert names | kept <= set(state)
    for n in ("qkv", "o", "gate_up", "down"):
        want = hv.ops.quantize_int4(plain[n], 64)
        w = getattr(a, n)
        assert torch.equal(w.packed, want.packed) and torch.equal(w.scales, want.scales)
        assert (w.out_features, w.in_features, w.group) == want[2:]
        assert not torch.equal(w.packed, getattr(b, n).packed)
    b.load_state_dict(state)
    for n, p in a.named_parameters():
        assert torch.equal(p, b.get_parameter(n))


def test_moved_with_the_layer():
    a = _layer(3)
    a.quantize_int4(128)
    a.to("meta")
    assert all(p.device.type == "meta" for p in a.parameters())
    assert a.qkv.packed.device.type == "meta" and a.down.scales.device.type == "meta"


def test_a_layer_that_shares_weights_keeps_its_own():
    """Shallow copies, as models that share weights make them."""
    a = _layer(4)
    before = a.qkv
    b = copy.copy(a)
    b._parameters, b._modules = dict(a._parameters), dict(a._modules)
    a.quantize_int4(128)
    assert b.qkv is before and not isinstance(a.qkv, torch.Tensor)
    c = copy.copy(a)
    c._parameters, c._modules = dict(a._parameters), dict(a._modules)
    assert c.qkv is a.qkv
    first = a.qkv
    a.quantize_int4(64)  # a second call leaves what is quantised
    assert a.qkv is first


def test_the_restatement_refuses_4_bit_weights():
    a = _layer(5)
    a.quantize_int4(128)
    with pytest.raises(TypeError):
        a.forward_reference(torch.zeros(1, dtype=torch.int64),
                            torch.zeros(1, 256, dtype=torch.bfloat16), None)


def test_a_refused_group_changes_nothing():
    """Inputs of the down projection that the group does not divide: the other three stay
    as they are too."""
    a = _layer(6, ffn=192)
    before = dict(a.named_parameters())
    with pytest.raises(ValueError):
        a.quantize_int4(128)
    after = dict(a.named_parameters())
    assert set(before) == set(after) and all(before[n] is after[n] for n in before)
    a.quantize_int4(64)
    assert a.down.in_features == 192
