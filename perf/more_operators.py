"""Performance cases of the 8-bit floating-point path's operators.

Each case is one call as an engine built on this package makes it:
  linear    a projection of e4m3 rows by e4m3 weights (ops.linear_fp8): the rows have a
            power of two for every 128 inputs, the weights an f32 scale for every block of
            128 x 128; plain, with the SwiGLU product, or with that product in 8 bits
  norm      RMSNorm, with or without the residual's addition, to e4m3 rows with scales
            (ops.rmsnorm_fp8)
  quantize  bf16 rows to e4m3 rows with scales (ops.quantize_rows_fp8)
Sizes follow the framework's benchmark configurations: hidden 4096 with a feed-forward of
12288 and 32/8 heads of 128, hidden 1024 with 16/8 heads, vocabulary 151936.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

VOCAB = 151936
DEV = "cuda"
GROUP = 128  # inputs of a scale, and the side of a weight's blocks
E4M3_MAX = 448.0
MIN_EXP = -126  # smallest exponent of a row's scale
EPS = 1e-6


def listed():
    return [
        # the output projection of one decoded token, from the attention's bf16 row: the
        # smallest call, one in every layer of an interactive user's every step
        dict(name="linear-o-1", kind="linear", rows=1, k=4096, n=4096, x="bf16", out="bf16"),
        # the fused q, k and v projection of a batch-1 verify step (4 rows) behind its norm
        dict(name="linear-qkv-4", kind="linear", rows=4, k=4096, n=6144, x="fp8", out="bf16"),
        # gate and up projections of 16 decoding sequences with the SwiGLU product
        dict(name="linear-gate-up-16", kind="linear", rows=16, k=4096, n=12288, x="fp8",
             out="swiglu"),
        # the LM head over the rows of four verify steps
        dict(name="linear-head-16", kind="linear", rows=16, k=4096, n=VOCAB, x="bf16",
             out="bf16"),
        # the down projection of a batch-16 verify step (64 rows)
        dict(name="linear-down-64", kind="linear", rows=64, k=12288, n=4096, x="fp8",
             out="bf16"),
        # a ragged prompt of one user
        dict(name="linear-qkv-531", kind="linear", rows=531, k=4096, n=6144, x="fp8",
             out="bf16"),
        # admission of prompts: the layer's largest projection, its product handed to the
        # down projection in 8 bits
        dict(name="linear-gate-up-4096", kind="linear", rows=4096, k=4096, n=12288, x="fp8",
             out="swiglu-fp8"),
        # the norm before a projection of a batch-1 verify step
        dict(name="norm-4", kind="norm", rows=4, hidden=4096, residual=True),
        # the first norm of the small model over a ragged prompt (no residual yet)
        dict(name="norm-first-1021", kind="norm", rows=1021, hidden=1024, residual=False),
        # the norm over admitted prompts
        dict(name="norm-4096", kind="norm", rows=4096, hidden=4096, residual=True),
        # the attention's rows of a batch-16 verify step
        dict(name="quantize-64", kind="quantize", rows=64, width=4096, slack=0),
        # the attention's rows of prompts, heads of a wider buffer
        dict(name="quantize-2003", kind="quantize", rows=2003, width=4096, slack=2048),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "norm", "quantize"])
    if kind == "linear":
        k, n, gate = rng.choice([(4096, 4096, False), (4096, 6144, False), (4096, 12288, True),
                                 (12288, 4096, False), (1024, 4096, False), (2048, 1024, False),
                                 (1024, 2048, True), (4096, VOCAB, False), (352, 200, False),
                                 (1056, 1001, False), (4000, 2512, True)])
        rows = _log_int(rng, 1, 64) if rng.random() < 0.6 else _log_int(rng, 65, 4000)
        if n == VOCAB:
            rows = min(rows, 24)
        return dict(kind=kind, rows=rows, k=k, n=n, x=rng.choice(["bf16", "fp8", "fp8"]),
                    out=rng.choice(["swiglu", "swiglu-fp8"]) if gate else "bf16")
    rows = _log_int(rng, 1, 4000)
    width = rng.choice([4096, 4096, 1024, 2048, 5120, 8192, 1056, 272])
    if kind == "norm":
        return dict(kind=kind, rows=rows, hidden=width, residual=rng.random() < 0.7)
    return dict(kind=kind, rows=rows, width=width, slack=rng.choice([0, 0, 64, 2048]))


# ---------------------------------------------------------------- prepare

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def prepare(case, seed):
    with torch.inference_mode():
        return _PREPARE[case["kind"]](case, _gen(seed))


def _hidden(gen, rows, width, spread=0.7):
    """Hidden states: rows of different size, and a few channels far larger than the
    others, as trained models have."""
    x = torch.randn(rows, width, generator=gen, device=DEV)
    x *= torch.exp(spread * torch.randn(width, generator=gen, device=DEV))
    return x * (torch.rand(rows, 1, generator=gen, device=DEV) * 2 + 0.2)


def _weights(case, gen):
    """Codes [N, K] and f32 scales [N / 128, K / 128] of weights that spread as a trained
    projection's: the scale of a block is its largest value over 448, any f32 number."""
    n = case["n"] * (2 if case["out"] != "bf16" else 1)
    k = case["k"]
    nb, kb = -(-n // GROUP), -(-k // GROUP)
    codes = torch.empty(n, k, device=DEV, dtype=torch.float8_e4m3fn)
    scales = torch.rand(nb, kb, generator=gen, device=DEV) * 2e-4 + 1e-4
    for i in range(0, n, 16384):
        w = torch.randn(min(16384, n - i), k, generator=gen, device=DEV).mul_(105)
        codes[i:i + 16384] = w.clamp_(-E4M3_MAX, E4M3_MAX).to(codes.dtype)
    return codes, scales


def _pack(codes, scales):
    """The layout the projections are kept in: 16-feature tiles by 128-input steps. Lane l
    of a step holds two times 16 codes of feature l % 16: inputs 64 h + 16 (l // 16) .. + 15,
    h = 0 and 1, the halves one after the other. Features and inputs are padded with zeros.
    Scales lie by tile and step."""
    n, k = codes.shape
    tiles, steps = -(-n // 16), -(-k // GROUP)
    c = torch.zeros(tiles * 16, steps * GROUP, dtype=torch.uint8, device=codes.device)
    c[:n, :k] = codes.view(torch.uint8)
    c = c.view(tiles, 16, steps, 2, 4, 16).permute(0, 2, 3, 4, 1, 5).contiguous()
    s = scales.repeat_interleave(GROUP // 16, 0)[:tiles].contiguous()
    return c.view(tiles, steps, 2, 64, 16), s


def _prepare_linear(case, gen):
    packed, scales = _pack(*_weights(case, gen))
    x = _hidden(gen, case["rows"], case["k"]).to(torch.bfloat16)
    s = dict(case=case, packed=packed, scales=scales)
    if case["x"] == "bf16":
        return dict(s, x=x)
    codes, xs = _plain_rows(x.float())
    return dict(s, x=codes, x_scales=xs)


def _prepare_norm(case, gen):
    rows, hidden = case["rows"], case["hidden"]
    x = _hidden(gen, rows, hidden).to(torch.bfloat16)
    weight = torch.rand(hidden, generator=gen, device=DEV) + 0.5
    res = None
    if case["residual"]:
        res = (_hidden(gen, rows, hidden, 1.2) * 4).to(torch.bfloat16)
    return dict(case=case, x=x, weight=weight.to(torch.bfloat16), residual=res)


def _prepare_quantize(case, gen):
    x = _hidden(gen, case["rows"], case["width"] + case["slack"]).to(torch.bfloat16)
    return dict(case=case, x=x[:, case["slack"]:])


_PREPARE = dict(linear=_prepare_linear, norm=_prepare_norm, quantize=_prepare_quantize)


# ---------------------------------------------------------------- run

def run(state):
    with torch.inference_mode():
        return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


def _ops():
    return importlib.import_module("hilda-vllm_amd").ops


def _own_linear(s):
    ops, c = _ops(), s["case"]
    gate = c["out"] != "bf16"
    w = ops.Fp8Weight(s["packed"], s["scales"], c["n"] * (2 if gate else 1), c["k"])
    x = s["x"] if c["x"] == "bf16" else ops.Fp8Rows(s["x"], s["x_scales"])
    y = ops.linear_fp8(x, w, swiglu=gate, quantize=c["out"] == "swiglu-fp8")
    return [y.codes, y.scales] if c["out"] == "swiglu-fp8" else y


def _own_norm(s):
    y = _ops().rmsnorm_fp8(s["x"], s["weight"], EPS, residual=s["residual"])
    return [y.codes, y.scales] + ([] if s["residual"] is None else [s["residual"]])


def _own_quantize(s):
    y = _ops().quantize_rows_fp8(s["x"])
    return [y.codes, y.scales]


def _plain_rows(x):
    """f32 rows to e4m3 codes and e8m0 scales: for every 128 inputs the smallest power of
    two s with |x| <= 448 s."""
    rows, width = x.shape
    groups = -(-width // GROUP)
    g = torch.nn.functional.pad(x, (0, groups * GROUP - width)).view(rows, groups, GROUP)
    m, e = torch.frexp(g.abs().amax(-1))  # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(m > 0, e, MIN_EXP).clamp(min=MIN_EXP)
    inverse = ((127 - e.int()) << 23).view(torch.float32)  # 2^-e, exactly
    codes = (g * inverse[..., None]).to(torch.float8_e4m3fn).view(rows, -1)[:, :width]
    return codes.contiguous(), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _plain_linear(s):
    c, p = s["case"], s["packed"]
    n = c["n"] * (2 if c["out"] != "bf16" else 1)
    tiles, steps = p.shape[:2]
    w = p.view(tiles, steps, 2, 4, 16, 16).permute(0, 4, 1, 2, 3, 5)
    w = w.contiguous().view(torch.float8_e4m3fn).float().view(tiles, 16, steps, GROUP)
    w = (w * s["scales"][:, None, :, None]).view(tiles * 16, -1)[:n, :c["k"]]
    codes, xs = (s["x"], s["x_scales"]) if c["x"] == "fp8" else _plain_rows(s["x"].float())
    x = codes.float() * xs.float().repeat_interleave(GROUP, 1)[:, :c["k"]]
    y = torch.nn.functional.linear(x, w)
    if c["out"] == "bf16":
        return y.to(torch.bfloat16)
    gate, up = y[:, :c["n"]], y[:, c["n"]:]
    y = gate / (1 + torch.exp(-gate)) * up
    return list(_plain_rows(y)) if c["out"] == "swiglu-fp8" else y.to(torch.bfloat16)


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
        s["residual"].copy_(h)
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
    return list(_plain_rows(y)) + ([] if s["residual"] is None else [s["residual"]])


def _plain_quantize(s):
    return list(_plain_rows(s["x"].float()))


_OWN = dict(linear=_own_linear, norm=_own_norm, quantize=_own_quantize)
_PLAIN = dict(linear=_plain_linear, norm=_plain_norm, quantize=_plain_quantize)


# ---------------------------------------------------------------- work

def work(case):
    """Bytes that have to be read and written and operations of one pass."""
    rows = case["rows"]

    def fp8(width):  # codes and scales of the rows
        return rows * (width + -(-width // GROUP))

    if case["kind"] == "norm":
        h = case["hidden"]
        return dict(bytes=rows * h * (6 if case["residual"] else 2) + fp8(h) + 2 * h,
                    flops=rows * h * 8)
    if case["kind"] == "quantize":
        return dict(bytes=2 * rows * case["width"] + fp8(case["width"]),
                    flops=rows * case["width"] * 3)
    n, k = case["n"] * (2 if case["out"] != "bf16" else 1), case["k"]
    x = fp8(k) if case["x"] == "fp8" else 2 * rows * k
    y = fp8(case["n"]) if case["out"] == "swiglu-fp8" else 2 * rows * case["n"]
    return dict(bytes=n * k + 4 * -(-n // GROUP) * -(-k // GROUP) + x + y,
                flops=2 * rows * n * k)


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    with torch.inference_mode():
        return _EXACT[case["kind"]](case, prepare(case, seed), seed)


def _pow2(e):
    """2^e as doubles, of exponents of normal ones."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3(x):
    """The e4m3 value nearest to x (a double): three bits behind the leading one, steps of
    2^-9 below 2^-6, ties to the even one."""
    _, e = torch.frexp(x)
    step = _pow2((e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _exact_rows(y):
    codes, scales = torch.empty_like(y), []
    for i in range(0, y.shape[1], GROUP):
        g = y[:, i:i + GROUP]
        e = torch.ceil(torch.log2(g.abs().amax(1) / E4M3_MAX)).clamp(min=MIN_EXP)
        scales.append(_pow2(e))
        codes[:, i:i + GROUP] = _e4m3(g / scales[-1][:, None])
    return [codes, torch.stack(scales, 1)]


def _exact_linear(case, s, seed):
    codes, scales = _weights(case, _gen(seed))
    k = case["k"]
    if case["x"] == "fp8":
        x, xs = s["x"].double(), s["x_scales"].double()
    else:
        x, xs = _exact_rows(s["x"].double())
    x = torch.cat([x[:, b * GROUP:(b + 1) * GROUP] * xs[:, b:b + 1] for b in range(xs.shape[1])], 1)
    y = []
    for i in range(0, codes.shape[0], 16384):
        w = codes[i:i + 16384].double()
        w *= scales.double().repeat_interleave(GROUP, 0)[i:i + 16384].repeat_interleave(
            GROUP, 1)[:w.shape[0], :k]
        y.append(x @ w.t().contiguous())
    y = torch.cat(y, 1)
    if case["out"] == "bf16":
        return y
    y = torch.nn.functional.silu(y[:, :case["n"]]) * y[:, case["n"]:]
    return _exact_rows(y) if case["out"] == "swiglu-fp8" else y


def _exact_norm(case, s, seed):
    h = s["x"].double()
    if case["residual"]:
        h = h + s["residual"].double()
    norm = torch.linalg.vector_norm(h, dim=1, keepdim=True) / math.sqrt(case["hidden"])
    y = h / torch.sqrt(norm ** 2 + EPS) * s["weight"].double()
    return _exact_rows(y) + ([h] if case["residual"] else [])


def _exact_quantize(case, s, seed):
    return _exact_rows(s["x"].double())


_EXACT = dict(linear=_exact_linear, norm=_exact_norm, quantize=_exact_quantize)
