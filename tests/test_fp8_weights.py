"""e4m3 weights as parts of a model (on the host)."""
import copy
import importlib

import pytest
import torch

from test_int4_weights import _layer

_NAMES = ("qkv", "o", "gate_up", "down")


def test_parameters_and_state(hv):
    """The quantised projections are among the layer's parameters and in its state, and a
    state goes into another layer of the same form."""
    a, b = _layer(1), _layer(2)
    plain = dict(a.named_parameters())
    a.quantize_fp8()
    b.quantize_fp8()
    names = {f"{n}.{part}" for n in _NAMES for part in ("packed", "scales")}
    kept = {"q_norm", "k_norm", "ln1", "ln2"}
    assert set(dict(a.named_parameters())) == names | kept
    assert not any(p.requires_grad for p in a.parameters())
    for n in _NAMES:
        want, w = hv.ops.quantize_fp8(plain[n]), getattr(a, n)
        assert torch.equal(w.packed, want.packed) and torch.equal(w.scales, want.scales)
        assert (w.out_features, w.in_features) == want[2:]
        assert not torch.equal(w.packed, getattr(b, n).packed)
    b.load_state_dict(a.state_dict())
    for n, p in a.named_parameters():
        assert torch.equal(p, b.get_parameter(n))
    a.to("meta")
    assert all(p.device.type == "meta" for p in a.parameters())


def test_what_is_quantised_stays():
    """A second call, or one for the other kind of weights, leaves what is quantised; a layer
    that shares weights keeps its own."""
    a = _layer(4)
    before = a.qkv
    b = copy.copy(a)
    b._parameters, b._modules = dict(a._parameters), dict(a._modules)
    a.quantize_fp8()
    assert b.qkv is before and not isinstance(a.qkv, torch.Tensor)
    first = [getattr(a, n) for n in _NAMES]
    a.quantize_fp8()
    a.quantize_int4(64)
    assert all(getattr(a, n) is w for n, w in zip(_NAMES, first))
    b.quantize_int4(64)
    first = b.qkv
    b.quantize_fp8()
    assert b.qkv is first


def test_refusals():
    a = _layer(5)
    a.quantize_fp8()
    with pytest.raises(TypeError):  # the restatement is of bf16 weights
        a.forward_reference(torch.zeros(1, dtype=torch.int64),
                            torch.zeros(1, 256, dtype=torch.bfloat16), None)
    # inputs of the down projection that are no multiple of 16: all four stay as they are
    a = _layer(6, ffn=200)
    before = dict(a.named_parameters())
    with pytest.raises(ValueError):
        a.quantize_fp8()
    after = dict(a.named_parameters())
    assert set(before) == set(after) and all(before[n] is after[n] for n in before)
    q3 = importlib.import_module("hilda-vllm_amd.engine.qwen3_host")
    assert not isinstance(a.qkv, q3.Fp8Projection)
