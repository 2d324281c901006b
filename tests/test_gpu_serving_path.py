"""The 8-bit cache with group scales, the 4-bit projections and the log-probabilities run
together as the decoder layers and the runner run them."""
import importlib

import numpy as np
import pytest
import torch

import scaled_ref as ref
from test_gpu_int4_linear import _reference, _tolerance

pytestmark = pytest.mark.gpu


def _mods():
    return (importlib.import_module("hilda-vllm_amd.engine.qwen3_host"),
            importlib.import_module("hilda-vllm_amd.engine.spec_runner"),
            importlib.import_module("hilda-vllm_amd.utils.context"))


def _unpack(w):
    """codes [N, K] and scales [N, K / group] of a packed weight (dword i of lane 16 g + f of a
    step: feature f, inputs 32 i + 8 g .. + 7, two codes every 4 bits, 16 apart)."""
    p, s = w.packed.cpu(), w.scales.cpu()
    tiles, steps = p.shape[:2]
    p = p.view(tiles, steps, 4, 16, 4, 1) >> torch.tensor([4 * (e // 2) + 16 * (e % 2)
                                                           for e in range(8)], dtype=torch.int32)
    codes = (p & 15).permute(0, 3, 1, 4, 2, 5).reshape(tiles * 16, steps * 128)
    scales = s.permute(0, 2, 1).reshape(tiles * 16, -1)
    return (codes[:w.out_features, :w.in_features].to(torch.uint8),
            scales[:w.out_features, :w.in_features // w.group])


def _near_linear(got, x, w, swiglu=False):
    codes, scales = _unpack(w)
    y, size = _reference(x.cpu(), codes, scales, w.group)
    tol = _tolerance(size, w.in_features, w.group)
    if swiglu:
        n = w.out_features // 2
        g, u = y[:, :n], y[:, n:]
        y = torch.nn.functional.silu(g) * u
        # silu's slope is below 1.1; its exponential and quotient are good to 2^-18 here
        tol = 1.1 * tol[:, :n] * (u.abs() + tol[:, n:]) + \
            torch.nn.functional.silu(g).abs() * tol[:, n:] + 2.0 ** -18 * y.abs()
    tol = tol + 2.0 ** -8 * y.abs()
    assert bool(((got.double().cpu() - y).abs() <= tol).all())


@pytest.mark.parametrize("bs,kv_group,group", [(32, 32, 128), (256, 64, 64)])
def test_layer_in_steps(hv, cuda, bs, kv_group, group):
    """Ragged prompts, verify rows of which one sequence is left out, single tokens: every
    operator's result within its bound of the 64-bit one on the same inputs, the cache bit for
    bit, and the layer's output that of the operators one by one."""
    q3, _, ctx = _mods()
    print("layer in steps", bs, kv_group, group, flush=True)
    g = q3.Qwen3Geometry(num_layers=1, hidden=512, num_heads=8, num_kv_heads=2, ffn=640,
                         vocab=300, max_position=512)
    host = q3.Qwen3Host(g, device=cuda, seed=5).quantize_int4(group, lm_head=True)
    layer, attn = host.layers[0], host.layers[0].attn
    nb = 16
    cache = torch.full((2, nb, bs, 2, 128), float("nan"), device=cuda).to(torch.float8_e4m3fn)
    scales = torch.zeros((2, nb, bs // kv_group, 2), device=cuda)
    attn.k_cache, attn.v_cache, attn.k_scales, attn.v_scales = *cache, *scales
    attn.kv_cache_dtype = "fp8_block"
    want = [t.double().cpu().numpy().copy() for t in (*cache, *scales)]
    W = 6 if bs == 32 else 1
    tables = torch.full((3, W), -1, dtype=torch.int32)
    free = iter([7, 2, 11, 0, 15, 4, 9, 1, 13, 6, 3, 10, 5, 8])
    lens = [0, 0, 0]
    gen = torch.Generator().manual_seed(bs + group)
    for new in ([70, 1, 33], [4, 0, 4], [1, 1, 1], [1, 3, 1]):
        ends = [a + b for a, b in zip(lens, new)]
        for b in range(3):
            for i in range(-(-ends[b] // bs)):
                if tables[b, i] < 0:
                    tables[b, i] = next(free)
        slots = [int(tables[b, i // bs]) * bs + i % bs for b in range(3)
                 for i in range(lens[b], ends[b])]
        pos = torch.tensor([i for b in range(3) for i in range(lens[b], ends[b])], device=cuda)
        cq = torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32, device=cuda)
        ck = torch.tensor([0] + np.cumsum(ends).tolist(), dtype=torch.int32, device=cuda)
        sm = torch.tensor(slots, dtype=torch.int32, device=cuda)
        h = torch.randn(len(slots), 512, generator=gen).to(torch.bfloat16).to(cuda)
        res = torch.randn(len(slots), 512, generator=gen).to(torch.bfloat16).to(cuda)
        start = [t.clone() for t in (attn.k_cache, attn.v_cache, attn.k_scales, attn.v_scales)]
        ctx.set_context(True, cq, ck, max(new), max(ends), sm, None, tables.to(cuda))
        out, out_res = layer(pos, h.clone(), res.clone())
        ctx.reset_context()

        r = res.clone()
        x = hv.ops.rmsnorm(h, layer.ln1, g.rms_eps, residual=r)
        qkv = hv.ops.linear_int4(x, layer.qkv)
        _near_linear(qkv, x, layer.qkv)
        q, k = hv.ops.qk_norm_rope(qkv, 8, 2, layer.q_norm, layer.k_norm, layer.rope.cos_sin,
                                   pos, g.rms_eps)
        v = qkv[:, 10 * 128:].unflatten(1, (2, 128))
        hv.ops.store_kvcache_scaled(k, v, *start, sm)
        ref.store(k.double().cpu().numpy(), want[0], want[2], slots)
        ref.store(v.double().cpu().numpy(), want[1], want[3], slots)
        for mine, layers_own, w in zip(start, (attn.k_cache, attn.v_cache, attn.k_scales,
                                               attn.v_scales), want):
            assert np.array_equal(mine.double().cpu().numpy(), w, equal_nan=True)
            assert np.array_equal(layers_own.double().cpu().numpy(), w, equal_nan=True)
        o = hv.ops.verify_attention_scaled(q, *start, tables.to(cuda), cq, ck, max(new),
                                           max(ends), attn.scale)
        at = 0
        for b in range(3):
            where = [(int(tables[b, i // bs]), i % bs) for i in range(ends[b])]
            kk, vv = (np.stack([c[t] * s[t[0], t[1] // kv_group][:, None] for t in where])
                      for c, s in ((want[0], want[2]), (want[1], want[3])))
            rows = slice(at, at + new[b])
            at += new[b]
            y, most, size = ref.attention(q[rows].double().cpu().numpy(), kk, vv, new[b], ends[b],
                                          attn.scale)
            err = np.abs(o[rows].double().cpu().numpy() - y)
            assert (err <= ref.tolerance(y, most, size)).all()
        h2 = hv.ops.linear_int4(o.view(len(slots), -1), layer.o)
        _near_linear(h2, o.view(len(slots), -1), layer.o)
        x2 = hv.ops.rmsnorm(h2, layer.ln2, g.rms_eps, residual=r)
        act = hv.ops.linear_int4(x2, layer.gate_up, swiglu=True)
        _near_linear(act, x2, layer.gate_up, swiglu=True)
        y2 = hv.ops.linear_int4(act, layer.down)
        _near_linear(y2, act, layer.down)
        assert torch.equal(out, y2) and torch.equal(out_res, r)
        head = host.compute_logits(x2)
        _near_linear(head, x2, host.lm_head)
        lens = ends


def test_attention_module(hv, cuda):
    """The layer's own forward: a prompt without block tables stores its rows and attends over
    them as they are; single tokens with context lengths attend over the cache."""
    _, _, ctx = _mods()
    print("attention module, group scales", flush=True)
    A = importlib.import_module("hilda-vllm_amd.layers.attention").Attention
    attn = A(4, 128, 0.09, 2)
    attn.kv_cache_dtype = "fp8_block"
    cache = torch.zeros((2, 5, 64, 2, 128), device=cuda).to(torch.float8_e4m3fn)
    scales = torch.zeros((2, 5, 2, 2), device=cuda)
    attn.k_cache, attn.v_cache, attn.k_scales, attn.v_scales = *cache, *scales
    other = [t.clone() for t in (*cache, *scales)]
    gen = torch.Generator().manual_seed(3)
    table = torch.tensor([[3, 1]], dtype=torch.int32, device=cuda)

    def rows(n, heads):
        return torch.randn(n, heads * 128, generator=gen).to(torch.bfloat16).to(cuda)

    n = 75
    q, k, v = rows(n, 4), rows(n, 2), rows(n, 2)
    cu = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    slots = torch.tensor([int(table[0, i // 64]) * 64 + i % 64 for i in range(n + 1)],
                         dtype=torch.int32, device=cuda)
    ctx.set_context(True, cu, cu, n, n, slots[:n], None, None)
    got = attn(q, k, v)
    k3, v3 = k.view(n, 2, 128), v.view(n, 2, 128)
    assert torch.equal(got, hv.ops.verify_attention(q.view(n, 4, 128), k3, v3, None, cu, cu, n, n,
                                                    0.09))
    hv.ops.store_kvcache_scaled(k3, v3, *other, slots[:n])
    q, k, v = rows(1, 4), rows(1, 2), rows(1, 2)
    ctx.set_context(False, None, None, 0, 0, slots[n:],
                    torch.tensor([n + 1], dtype=torch.int32, device=cuda), table)
    got = attn(q, k, v)
    ctx.reset_context()
    hv.ops.store_kvcache_scaled(k.view(1, 2, 128), v.view(1, 2, 128), *other, slots[n:])
    one = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    assert torch.equal(got, hv.ops.verify_attention_scaled(
        q.view(1, 4, 128), *other, table, one, one * (n + 1), 1, 128, 0.09))
    for a, b in zip((attn.k_cache, attn.v_cache), other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(attn.k_scales, other[2]) and torch.equal(attn.v_scales, other[3])


def _check_logprobs(lp, logits, tokens, olen, top):
    """Against log softmax in 64 bits: chunk maxima m and sums in 32 bits move a row's
    logarithm by 2^-21 (2 max |logit - m| + log V + 32) at most."""
    x = logits.double().cpu()
    want = torch.log_softmax(x, -1)
    m = (x - x.amax(-1, keepdim=True)).abs().amax()
    tol = 2.0 ** -21 * (2 * float(m) + np.log(x.shape[-1]) + 32)
    for b in range(len(olen)):
        for j in range(int(olen[b])):
            assert abs(float(lp["logprobs"][b, j]) - float(want[b, j, int(tokens[b, j])])) <= tol
            order = torch.argsort(x[b, j], descending=True, stable=True)[:top]
            assert torch.equal(lp["top_ids"][b, j].cpu(), order)
            assert float((lp["top_logprobs"][b, j].cpu().double() - want[b, j][order]).abs().max()) \
                <= tol


@pytest.mark.parametrize("batch,mode", [(1, "reference"), (3, "reference"), (2, "greedy")])
def test_runner_graph_replay_matches_eager(cuda, batch, mode):
    """4-bit target weights, a cache with group scales and log-probabilities in the runner:
    eager steps and replayed graphs emit the same tokens, and every step's log-probabilities
    are those of the rows its tokens were accepted or drawn from."""
    q3, sr, _ = _mods()
    print("runner, group scales + 4 bits + logprobs", batch, mode, flush=True)
    gt = q3.Qwen3Geometry(num_layers=2, hidden=512, num_heads=4, num_kv_heads=2, ffn=1024,
                          vocab=3001, max_position=1024)
    gd = q3.Qwen3Geometry(num_layers=1, hidden=512, num_heads=4, num_kv_heads=2, ffn=1024,
                          vocab=3001, max_position=1024)

    def make():
        target = q3.Qwen3Host(gt, device=cuda, seed=21).quantize_int4(128, lm_head=batch == 3)
        draft = q3.Qwen3Host(gd, device=cuda, seed=22)
        r = sr.SpecRunner(target, draft, batch=batch, gamma=3, max_model_len=400, block_size=64,
                          kv_cache_dtype="fp8_block", kv_group=32, logprobs=5,
                          temperature=0.0 if mode == "greedy" else 0.7, mode=mode, device=cuda)
        r.load_prompts([[3, 4, 5, 6], list(range(200, 240)), [9] * 130][:batch])
        torch.manual_seed(5)
        r.prefill()
        assert r.first_logprobs["logprobs"].shape == (batch,)
        assert bool((r.first_logprobs["logprobs"] <= 0).all())
        return r

    def check(r):
        _, out, olen = r.last
        _check_logprobs(r.logprobs, r._g().logits, out.cpu(), olen.cpu(), 5)

    eager, graph = make(), make()
    torch.manual_seed(77)
    history = []
    for _ in range(7):
        eager.step()
        check(eager)
        history.append([t.clone() for t in eager.logprobs.values()])
    torch.manual_seed(77)
    graph.step()
    graph.capture()
    check(graph)
    for i in range(6):
        graph.replay()
        check(graph)
        olen = graph.last[2].cpu()
        for a, b in zip(graph.logprobs.values(), history[i + 1]):
            for s in range(batch):
                assert torch.equal(a[s, :olen[s]], b[s, :olen[s]])
    graph.check()
    assert graph.lengths() == eager.lengths()
    for b in range(batch):
        assert graph.tokens(b) == eager.tokens(b)
    assert graph.kv_saturation() == 0.0
