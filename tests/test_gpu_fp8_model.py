"""The 8-bit floating-point path run together, as the decoder layers and the runner run it."""
import importlib

import numpy as np
import pytest
import torch

import fp8_ref as ref
from test_gpu_fp8_linear import _reference, _same
from test_gpu_fp8_rows import _norm

pytestmark = pytest.mark.gpu


def _mods():
    return (importlib.import_module("hilda-vllm_amd.engine.qwen3_host"),
            importlib.import_module("hilda-vllm_amd.engine.spec_runner"),
            importlib.import_module("hilda-vllm_amd.utils.context"))


def _unpack(w):
    """codes [N, K] and block scales of a packed weight (lane 16 g + f of a step: feature f,
    inputs 64 h + 16 g .. + 15)."""
    p = w.packed.cpu()
    tiles, steps = p.shape[:2]
    p = p.view(tiles, steps, 2, 4, 16, 16).permute(0, 4, 1, 2, 3, 5).reshape(tiles * 16, -1)
    codes = p[:w.out_features, :w.in_features].contiguous().view(torch.float8_e4m3fn)
    return codes, w.scales.cpu()[::8]


def _near_linear(got, x, w, epilogue="plain"):
    """got: the projection of x (rows in 8 bits, or bf16) by w, against the same in 64 bits."""
    codes, scales = _unpack(w)
    if isinstance(x, torch.Tensor):
        x = ref.values(*ref.rows(x.cpu()))
    else:
        x = ref.values(x.codes.cpu(), x.scales.cpu())
    n = w.out_features // (1 if epilogue == "plain" else 2)
    y, tol = _reference(x, codes, scales, epilogue, n)
    if epilogue == "eight":
        ref.check_rows(got.codes, got.scales, y, tol)
    else:
        err = (got.double().cpu() - y).abs()
        assert bool((err <= tol + 2.0 ** -8 * (y.abs() + tol)).all())


def _near_norm(got, h, res, w, eps):
    sum_, y, tol = _norm(h.cpu(), res.cpu(), w.cpu(), eps)
    ref.check_rows(got.codes, got.scales, y, tol)
    return sum_.float().to(torch.bfloat16)


def test_layer_in_steps(hv, cuda):
    """Ragged prompts, verify rows of which one sequence is left out, single tokens: every
    operator's result within its bound of the 64-bit one on the same inputs, and the layer's
    output that of the operators one by one."""
    q3, _, ctx = _mods()
    print("layer in steps, 8 bits", flush=True)
    ops, bs = hv.ops, 32
    g = q3.Qwen3Geometry(num_layers=1, hidden=512, num_heads=8, num_kv_heads=2, ffn=656,
                         vocab=300, max_position=512)
    host = q3.Qwen3Host(g, device=cuda, seed=5).quantize_fp8(lm_head=True)
    layer = host.layers[0]
    attn = layer.attn
    cache = torch.zeros((2, 16, bs, 2, 128), dtype=torch.bfloat16, device=cuda)
    attn.k_cache, attn.v_cache = cache
    tables = torch.arange(18, dtype=torch.int32).view(3, 6).remainder(16)
    lens = [0, 0, 0]
    gen = torch.Generator().manual_seed(bs)
    for new in ([70, 1, 33], [4, 0, 4], [1, 1, 1], [6, 3, 8]):
        ends = [a + b for a, b in zip(lens, new)]
        slots = [int(tables[b, i // bs]) * bs + i % bs for b in range(3)
                 for i in range(lens[b], ends[b])]
        pos = torch.tensor([i for b in range(3) for i in range(lens[b], ends[b])], device=cuda)
        cq = torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32, device=cuda)
        ck = torch.tensor([0] + np.cumsum(ends).tolist(), dtype=torch.int32, device=cuda)
        sm = torch.tensor(slots, dtype=torch.int32, device=cuda)
        h = torch.randn(len(slots), 512, generator=gen).to(torch.bfloat16).to(cuda)
        res = torch.randn(len(slots), 512, generator=gen).to(torch.bfloat16).to(cuda)
        own = cache.clone()
        ctx.set_context(True, cq, ck, max(new), max(ends), sm, None, tables.to(cuda))
        out, out_res = layer(pos, h.clone(), res.clone())

        r = res.clone()
        x = ops.rmsnorm_fp8(h, layer.ln1, g.rms_eps, residual=r)
        assert torch.equal(r.cpu(), _near_norm(x, h, res, layer.ln1, g.rms_eps))
        qkv = ops.linear_fp8(x, layer.qkv)
        _near_linear(qkv, x, layer.qkv)
        attn.k_cache, attn.v_cache = own
        o = attn.attend_qkv(qkv, layer.q_norm, layer.k_norm, layer.rope.cos_sin, pos, g.rms_eps)
        attn.k_cache, attn.v_cache = cache
        ctx.reset_context()
        o = o.reshape(len(slots), -1)
        h2 = ops.linear_fp8(o, layer.o)
        _near_linear(h2, o, layer.o)
        before = r.clone()
        x2 = ops.rmsnorm_fp8(h2, layer.ln2, g.rms_eps, residual=r)
        assert torch.equal(r.cpu(), _near_norm(x2, h2, before, layer.ln2, g.rms_eps))
        eight = len(slots) > 16
        act = ops.linear_fp8(x2, layer.gate_up, swiglu=True, quantize=eight)
        _near_linear(act, x2, layer.gate_up, "eight" if eight else "swiglu")
        y2 = ops.linear_fp8(act, layer.down)
        _near_linear(y2, act, layer.down)
        assert torch.equal(out, y2) and torch.equal(out_res, r)
        _near_linear(host.compute_logits(h2), h2, host.lm_head)
        lens = ends


def test_layer_is_near_the_bf16_one(cuda):
    """A whole model's hidden states against those of its bf16 weights: 8 bits have a relative
    error of at most 2^-4 a value, 2^-4 / sqrt(3) if it is spread evenly; over the two operands
    of four projections a layer's own output is off by less than their sum, sqrt(8) of it."""
    q3, _, ctx = _mods()
    print("model near bf16", flush=True)
    g = q3.Qwen3Geometry(num_layers=1, hidden=512, num_heads=4, num_kv_heads=2, ffn=1024, vocab=64,
                         max_position=128)
    host = q3.Qwen3Host(g, device=cuda, seed=3)
    n = 90
    cu = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    pos = torch.arange(n, device=cuda)
    slots = torch.arange(n, dtype=torch.int32, device=cuda)
    h = torch.randn(n, 512, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda)
    layer, outs = host.layers[0], []
    for quantise in (False, True):
        if quantise:
            host.quantize_fp8()
        cache = torch.zeros((2, 4, 32, 2, 128), dtype=torch.bfloat16, device=cuda)
        layer.attn.k_cache, layer.attn.v_cache = cache
        ctx.set_context(True, cu, cu, n, n, slots, None,
                        torch.arange(4, dtype=torch.int32, device=cuda)[None])
        outs.append(layer(pos, h.clone(), None)[0].double())
        ctx.reset_context()
    off = float((outs[1] - outs[0]).norm() / outs[0].norm())
    assert 0 < off < 2.0 ** -4 / 3 ** 0.5 * 8 ** 0.5


def test_state_of_a_quantised_model(hv, cuda):
    """The state of a quantised model, LM head included, makes another model the same one,
    also by way of the host; weights that a caller sets in the model's places run; a model that
    shares the weights has them too."""
    q3, _, _ = _mods()
    print("state of a model in 8 bits", flush=True)
    g = q3.Qwen3Geometry(num_layers=2, hidden=256, num_heads=2, num_kv_heads=1, ffn=384, vocab=301,
                         max_position=64)
    a = q3.Qwen3Host(g, device=cuda, seed=1)
    plain = hv.ops.quantize_fp8(a.lm_head)
    a.quantize_fp8(lm_head=True)
    b = q3.Qwen3Host(g, device=cuda, seed=2).quantize_fp8(lm_head=True)
    h = torch.randn(5, 256, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    want = a.compute_logits(h)
    assert torch.equal(want, hv.ops.linear_fp8(h, plain))
    assert not torch.equal(b.compute_logits(h), want)
    b.load_state_dict({k: v.cpu() for k, v in a.state_dict().items()})
    assert torch.equal(b.to("cpu").to(cuda).compute_logits(h), want)
    shared = q3.Qwen3Host(g, device=cuda, share_from=a, num_layers=1)
    assert torch.equal(shared.compute_logits(h), want)
    assert shared.layers[0].qkv is a.layers[0].qkv
    del b.lm_head
    b.lm_head = plain
    assert torch.equal(b.compute_logits(h), want)
    b.quantize_fp8(lm_head=True)  # leaves it as it is
    assert b.lm_head is plain


@pytest.mark.parametrize("batch,kv", [(1, "bf16"), (3, "fp8_block"), (7, "fp8")])
def test_runner_graph_replay_matches_eager(cuda, batch, kv):
    """e4m3 target weights in the runner: eager steps and replayed graphs emit the same tokens
    (4 rows to a sequence: 4, 12 and 28)."""
    q3, sr, _ = _mods()
    print("runner, 8-bit weights", batch, kv, flush=True)
    gt = q3.Qwen3Geometry(num_layers=2, hidden=512, num_heads=4, num_kv_heads=2, ffn=1024,
                          vocab=3001, max_position=1024)
    gd = q3.Qwen3Geometry(num_layers=1, hidden=512, num_heads=4, num_kv_heads=2, ffn=1024,
                          vocab=3001, max_position=1024)

    def make():
        target = q3.Qwen3Host(gt, device=cuda, seed=21).quantize_fp8(lm_head=batch == 3)
        draft = q3.Qwen3Host(gd, device=cuda, seed=22).quantize_fp8()
        r = sr.SpecRunner(target, draft, batch=batch, gamma=3, max_model_len=400, block_size=64,
                          kv_cache_dtype=kv, temperature=0.7, mode="reference", device=cuda)
        r.load_prompts([[3, 4, 5, 6], list(range(200, 240)), [9] * 130, [1] * 17, [7, 8],
                        list(range(50, 99)), [5]][:batch])
        torch.manual_seed(5)
        r.prefill()
        return r

    eager, graph = make(), make()
    torch.manual_seed(77)
    for _ in range(7):
        eager.step()
    torch.manual_seed(77)
    graph.step()
    graph.capture()
    for _ in range(6):
        graph.replay()
    graph.check()
    assert graph.lengths() == eager.lengths()
    for b in range(batch):
        assert graph.tokens(b) == eager.tokens(b)
