"""Performance cases of the quantised verify step's operators.

Each case is one call as an engine built on this package makes it:
  store    the step's K/V rows into an 8-bit paged cache that holds a scale for
           every group of tokens and kv head (ops.store_kvcache_scaled)
  attend   decode, verify and prompt attention over that cache
           (ops.verify_attention_scaled)
  linear   a projection with 4-bit weights and group scales (ops.linear_int4)
  logprobs log-probabilities of the emitted tokens with the rows' entropy and
           their most likely alternatives (ops.token_logprobs)
Sizes follow the framework's benchmark configurations: 32/8 and 16/8 heads of
128, hidden 4096 with a feed-forward of 12288, vocabulary 151936, contexts up
to 40960 tokens, blocks of 256 tokens.
"""
from __future__ import annotations

import importlib
import math
import random

import torch
import torch.nn.functional as F

own = False

VOCAB = 151936
BLOCK = 256  # tokens per KV block, the framework's default
D = 128
DEV = "cuda"
HEADS = {"8b": (32, 8), "0.6b": (16, 8)}  # query and kv heads
E4M3_MAX = 448.0
MIN_EXP = -96  # smallest exponent of a stored scale


def listed():
    return [
        # one new token of each of 64 running sequences, mid-way through their groups:
        # the store of a decode step, once a layer
        dict(name="store-decode-b64", kind="store", model="8b", batch=64, q_min=1, q_max=1,
             k_min=64, k_max=700, group=32),
        # admission of ragged prompts, some behind a cached prefix that ends inside a group
        dict(name="store-prompts", kind="store", model="8b", batch=4, q_min=61, q_max=1021,
             k_min=1021, k_max=1200, group=32),
        # the batch-1 verify step, 4 query rows on a 320-token context: the smallest
        # call, one in every layer of every step of an interactive user
        dict(name="attend-verify-b1", kind="attend", model="8b", batch=1, q_min=4, q_max=4,
             k_min=320, k_max=320, bound=4096, group=32),
        # a serving batch of draft / small-model verify rows with ragged contexts
        dict(name="attend-verify-b64", kind="attend", model="0.6b", batch=64, q_min=4, q_max=4,
             k_min=64, k_max=2048, bound=2048, group=64),
        # long generations, one token each, 8B heads: the largest read of a cache
        dict(name="attend-decode-b32", kind="attend", model="8b", batch=32, q_min=1, q_max=1,
             k_min=2048, k_max=8192, bound=8192, group=32),
        # one user at the longest context the model takes
        dict(name="attend-verify-long", kind="attend", model="8b", batch=1, q_min=4, q_max=4,
             k_min=40001, k_max=40001, bound=40960, group=128),
        # prompt chunks behind cached prefixes
        dict(name="attend-prompts", kind="attend", model="8b", batch=2, q_min=509, q_max=2043,
             k_min=2043, k_max=3100, bound=4096, group=32),
        # the output projection of a batch-1 verify step (4 rows)
        dict(name="linear-o-4", kind="linear", rows=4, k=4096, n=4096, group=128, swiglu=False),
        # gate and up projections of the same step with the SwiGLU product
        dict(name="linear-gate-up-4", kind="linear", rows=4, k=4096, n=12288, group=128,
             swiglu=True),
        # the down projection of a batch-16 verify step (64 rows)
        dict(name="linear-down-64", kind="linear", rows=64, k=12288, n=4096, group=64,
             swiglu=False),
        # the four rows of a batch-1 verify step, five alternatives for the client
        dict(name="logprobs-verify-b1", kind="logprobs", rows=4, vocab=VOCAB, logits="bf16",
             top=5, tempered=False),
        # a serving batch that asks for the most alternatives the API allows
        dict(name="logprobs-256", kind="logprobs", rows=256, vocab=VOCAB, logits="bf16", top=20,
             tempered=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "linear", "linear", "logprobs"])
    if kind == "store":
        model, group = rng.choice(["8b", "0.6b"]), rng.choice([32, 64, 128, 256])
        if rng.random() < 0.5:  # decode or verify rows
            q = rng.choice([1, 2, 4, 6])
            hi = _log_int(rng, 16, 700)
            return dict(kind=kind, model=model, batch=_log_int(rng, 1, 64), q_min=q, q_max=q,
                        k_min=max(q, hi // 4), k_max=max(q, hi), group=group)
        batch = _log_int(rng, 1, 8)
        hi = _log_int(rng, 17, 4000 // batch)
        return dict(kind=kind, model=model, batch=batch, q_min=max(1, hi // 3), q_max=hi,
                    k_min=hi, k_max=hi + rng.choice([0, 45, 300]), group=group)
    if kind == "attend":
        model, group = rng.choice(["8b", "0.6b"]), rng.choice([32, 64, 128, 256])
        if rng.random() < 0.7:  # decode and verify rows
            batch = _log_int(rng, 1, 64)
            q = rng.choice([1, 1, 2, 3, 4, 5, 6, 9])
            hi = max(q, _log_int(rng, 33, min(40000, 150000 // batch)))
            lo = max(q, int(hi * rng.choice([0.05, 0.3, 1.0])))
            bound = next(b for b in (2048, 4096, 8192, 40960) if hi <= b)
            return dict(kind=kind, model=model, batch=batch, q_min=q, q_max=q, k_min=lo,
                        k_max=hi, bound=bound, group=group)
        batch = _log_int(rng, 1, 8)
        hi = _log_int(rng, 17, 2000 // batch)
        lo = max(1, int(hi * rng.choice([0.1, 0.5, 1.0])))
        k = hi + rng.choice([0, 0, 77, 900])
        return dict(kind=kind, model=model, batch=batch, q_min=lo, q_max=hi, k_min=hi, k_max=k,
                    bound=4096 if k <= 4096 else 8192, group=group)
    if kind == "linear":
        k, n, swiglu = rng.choice([(4096, 4096, False), (4096, 6144, False), (4096, 12288, True),
                                   (12288, 4096, False), (1024, 4096, False), (2048, 1024, False),
                                   (1024, 2048, True), (4096, VOCAB, False), (352, 200, False),
                                   (1056, 1001, False), (4000, 2512, True)])
        group = 32 if k % 128 else rng.choice([32, 64, 128])
        rows = _log_int(rng, 1, 64) if rng.random() < 0.8 else _log_int(rng, 65, 600)
        if n == VOCAB:
            rows = min(rows, 24)
        return dict(kind=kind, rows=rows, k=k, n=n, group=group, swiglu=swiglu)
    return dict(kind=kind, rows=_log_int(rng, 1, 250), vocab=rng.choice([VOCAB, VOCAB, 32003, 1001]),
                logits=rng.choice(["bf16", "f32"]), top=rng.choice([0, 1, 5, 20]),
                tempered=rng.random() < 0.5)


# ---------------------------------------------------------------- shapes of a case

def _lens(case):
    """(new tokens, tokens in all) of every sequence: from the case alone, so that
    inputs of another seed are of the same shapes."""
    rng = random.Random(f"{case['batch']}-{case['q_min']}-{case['q_max']}-{case['k_max']}")
    out = []
    for i in range(case["batch"]):
        q = case["q_max"] if i == 0 else rng.randint(case["q_min"], case["q_max"])
        k = case["k_max"] if i == 0 else rng.randint(case["k_min"], case["k_max"])
        out.append((q, max(q, k)))
    return out


def _cu(values):
    c = [0]
    for v in values:
        c.append(c[-1] + v)
    return c


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(gen, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _tables(lens, gen, bound):
    """Block tables of a running batch over a pool whose blocks are in no order."""
    nblk = [-(-k // BLOCK) for _, k in lens]
    pool = sum(nblk) + 2
    perm = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    tables = torch.full((len(lens), -(-(bound + 10) // BLOCK)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(nblk):
        tables[b, :n] = perm[at:at + n]
        at += n
    return tables, pool


def _cache(gen, pool, heads, group):
    """A cache whose groups were written by the store: codes, and scales that are the
    power of two above the group's largest value over 448."""
    codes = torch.empty(pool, BLOCK, heads, D, device=DEV, dtype=torch.float8_e4m3fn)
    scales = torch.empty(pool, BLOCK // group, heads, device=DEV, dtype=torch.float32)
    for i in range(0, pool, 64):
        n = min(64, pool - i)
        x = torch.randn(n, BLOCK // group, group, heads, D, generator=gen, device=DEV)
        x *= torch.rand(n, BLOCK // group, 1, heads, 1, generator=gen, device=DEV) * 2 + 0.1
        s = _pow2_over(x.abs().amax((2, 4)))
        codes[i:i + n] = (x / s[:, :, None, :, None]).reshape(n, BLOCK, heads, D).to(codes.dtype)
        scales[i:i + n] = s
    return codes, scales


# ---------------------------------------------------------------- prepare

def prepare(case, seed):
    with torch.inference_mode():
        return _PREPARE[case["kind"]](case, seed)


def _prepare_store(case, seed):
    gen, lens, (_, heads) = _gen(seed), _lens(case), HEADS[case["model"]]
    tables, pool = _tables(lens, gen, max(k for _, k in lens))
    pos = torch.cat([torch.arange(k - q, k, device=DEV) for q, k in lens])
    seq = torch.cat([torch.full((q,), b, device=DEV) for b, (q, _) in enumerate(lens)])
    slots = (tables[seq, pos // BLOCK].long() * BLOCK + pos % BLOCK).to(torch.int32)
    kc, ks = _cache(gen, pool, heads, case["group"])
    vc, vs = _cache(gen, pool, heads, case["group"])
    # k and v as slices of a fused projection's rows, each token with its own amplitude
    n = pos.numel()
    kv = _normal(gen, n, 2 * heads, D, dtype=torch.float32)
    kv = (kv * (torch.rand(n, 1, 1, generator=gen, device=DEV) * 2 + 0.2)).to(torch.bfloat16)
    return dict(case=case, k=kv[:, :heads], v=kv[:, heads:], kc=kc, vc=vc, ks=ks, vs=vs,
                slots=slots)


def _prepare_attend(case, seed):
    gen, lens, (hq, heads) = _gen(seed), _lens(case), HEADS[case["model"]]
    tables, pool = _tables(lens, gen, case["bound"])
    kc, ks = _cache(gen, pool, heads, case["group"])
    vc, vs = _cache(gen, pool, heads, case["group"])
    n = sum(q for q, _ in lens)
    return dict(case=case, q=_normal(gen, n, hq, D), kc=kc, vc=vc, ks=ks, vs=vs, tables=tables,
                cu_q=_ints(_cu([q for q, _ in lens])), cu_k=_ints(_cu([k for _, k in lens])),
                max_q=max(q for q, _ in lens), max_k=max(k for _, k in lens))


def _weights(case, gen):
    """Codes 0..15 [N, K] (the value is code - 8) and bf16 scales [N, K / group] of
    weights that spread as a trained projection's."""
    n = case["n"] * (2 if case["swiglu"] else 1)
    codes = torch.randn(n, case["k"], generator=gen, device=DEV, dtype=torch.float16)
    codes = (codes * 3 + 8).round_().clamp_(0, 15).to(torch.uint8)
    scales = torch.rand(n, case["k"] // case["group"], generator=gen, device=DEV) * 0.008 + 0.003
    return codes, scales.to(torch.bfloat16)


def _pack(codes, scales, group):
    """The layout the projections are kept in: 16-feature tiles by 128-wide steps. Dword i
    of lane l of a step holds the codes of feature l % 16, inputs 32 i + 8 (l // 16) .. + 7:
    input 2 p at bits 4 p, input 2 p + 1 at bits 16 + 4 p. Scales lie by tile, group,
    feature. Features and inputs are padded with code 8 (zero) and scale 0."""
    n, k = codes.shape
    tiles, steps, per = -(-n // 16), -(-k // 128), 128 // group
    c = torch.full((tiles * 16, steps * 128), 8, dtype=torch.uint8, device=codes.device)
    c[:n, :k] = codes
    c = c.view(tiles, 16, steps, 4, 4, 8).permute(0, 2, 4, 1, 3, 5).int()
    word = torch.zeros(c.shape[:-1], dtype=torch.int32, device=codes.device)
    for e in range(8):
        word |= c[..., e] << (4 * (e // 2) + 16 * (e % 2))
    s = torch.zeros(tiles * 16, steps * per, dtype=scales.dtype, device=scales.device)
    s[:n, :scales.shape[1]] = scales
    return (word.view(tiles, steps, 64, 4),
            s.view(tiles, 16, steps * per).permute(0, 2, 1).contiguous())


def _prepare_linear(case, seed):
    gen = _gen(seed)
    codes, scales = _weights(case, gen)
    packed, ps = _pack(codes, scales, case["group"])
    # hidden states: a few channels far larger than the others, as trained models have
    x = torch.randn(case["rows"], case["k"], generator=gen, device=DEV)
    x *= torch.exp(0.7 * torch.randn(case["k"], generator=gen, device=DEV))
    return dict(case=case, x=x.to(torch.bfloat16), packed=packed, scales=ps)


def _prepare_logprobs(case, seed):
    gen, rows, vocab = _gen(seed), case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=gen, device=DEV) * 3
    # rows from flat to certain: a likely token stands out by its own margin
    top = torch.randint(vocab, (rows,), generator=gen, device=DEV)
    margin = torch.rand(rows, generator=gen, device=DEV) * 14
    x[torch.arange(rows, device=DEV), top] += margin
    tokens = torch.where(torch.rand(rows, generator=gen, device=DEV) < 0.7, top,
                         torch.randint(vocab, (rows,), generator=gen, device=DEV))
    t = torch.rand(rows, generator=gen, device=DEV) * 0.9 + 0.5 if case["tempered"] else None
    return dict(case=case, logits=x.to(torch.bfloat16 if case["logits"] == "bf16" else
                                       torch.float32), tokens=tokens, temperatures=t)


_PREPARE = dict(store=_prepare_store, attend=_prepare_attend, linear=_prepare_linear,
                logprobs=_prepare_logprobs)


# ---------------------------------------------------------------- run

def run(state):
    with torch.inference_mode():
        return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


def _ops():
    return importlib.import_module("hilda-vllm_amd").ops


def _own_store(s):
    _ops().store_kvcache_scaled(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"])
    return [s["kc"], s["vc"], s["ks"], s["vs"]]


def _own_attend(s):
    return _ops().verify_attention_scaled(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["tables"],
                                          s["cu_q"], s["cu_k"], s["max_q"], s["case"]["bound"],
                                          D ** -0.5)


def _own_linear(s):
    ops, c = _ops(), s["case"]
    w = ops.Int4Weight(s["packed"], s["scales"], c["n"] * (2 if c["swiglu"] else 1), c["k"],
                       c["group"])
    return ops.linear_int4(s["x"], w, swiglu=c["swiglu"])


def _own_logprobs(s):
    r = _ops().token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"],
                              temperatures=s["temperatures"])
    return [r["logprobs"], r["entropy"]] + ([r["top_ids"], r["top_logprobs"]]
                                            if s["case"]["top"] else [])


def _pow2_over(a):
    """The smallest power of two s with a <= 448 s, not below 2^MIN_EXP."""
    m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(a > 0, e, MIN_EXP).clamp(min=MIN_EXP)
    return ((e.int() + 127) << 23).view(torch.float32)


def _values(codes, *at):
    """Entries of a cache's codes as floats."""
    return codes.view(torch.uint8)[at].view(codes.dtype).float()


def _plain_store(s):
    group = s["case"]["group"]
    slots = s["slots"].long()
    gid, off = slots // group, slots % group
    for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = x.float()
        c, sc = codes.view(-1, group, *codes.shape[2:]), scales.view(-1, scales.shape[2])
        # of every group of the cache: the largest value of its new tokens, and whether
        # one of them is the group's first
        need = _pow2_over(torch.zeros_like(sc).index_reduce_(0, gid, x.abs().amax(-1), "amax"))
        first = torch.zeros(len(sc), device=DEV).index_add_(0, gid, (off == 0).float()) > 0
        new = torch.where(first[:, None], need, torch.maximum(sc, need))
        # the other values of the groups, as they stand under the new scale: of the
        # tokens' groups, or of all where there are fewer
        at = gid if len(gid) < len(sc) else torch.arange(len(sc), device=DEV)
        factor = torch.where(first[:, None], 1.0, sc / new)[at, None, :, None]
        moved = (_values(c, at) * factor).clamp(-E4M3_MAX, E4M3_MAX).to(c.dtype)
        c.view(torch.uint8)[at] = moved.view(torch.uint8)
        sc.copy_(new)
        x = (x / new[gid, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(c.dtype)
        c.view(torch.uint8)[gid, off] = x.view(torch.uint8)
    return [s["kc"], s["vc"], s["ks"], s["vs"]]


def _plain_attend(s):
    case, (hq, heads) = s["case"], HEADS[s["case"]["model"]]
    cq, ck, mq, mk = s["cu_q"].long(), s["cu_k"].long(), s["max_q"], s["max_k"]
    lq, lk = cq[1:] - cq[:-1], ck[1:] - ck[:-1]
    i, j = torch.arange(mq, device=DEV), torch.arange(mk, device=DEV)
    live = j[None] < lk[:, None]
    blk = s["tables"].long()[:, j // BLOCK].clamp(min=0)
    row = torch.where(i[None] < lq[:, None], cq[:-1, None] + i, 0)
    q = s["q"].float()[row].view(len(lq), mq, heads, hq // heads, D)

    def values(codes, scales):  # [B, heads, keys, D], zero behind the sequences' ends
        x = _values(codes, blk, j % BLOCK)
        x = x * scales[blk, (j % BLOCK) // case["group"]][..., None]
        return torch.where(live[..., None, None], x, 0).transpose(1, 2).contiguous()

    q = q.permute(0, 2, 3, 1, 4).reshape(len(lq), heads, -1, D)  # rows (head of the group, token)
    w = torch.matmul(q, values(s["kc"], s["ks"]).transpose(2, 3).contiguous())
    w = w.view(len(lq), heads, -1, mq, mk)
    w *= D ** -0.5
    seen = live[:, None] & (j <= (lk - lq)[:, None, None] + i[:, None])
    w.masked_fill_(~seen[:, None, None], -math.inf)
    m = w.amax(-1, keepdim=True)
    w -= torch.where(m == -math.inf, 0, m)
    w.exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(len(lq), heads, -1, mk), values(s["vc"], s["vs"]))
    o = o.view(len(lq), heads, -1, mq, D) / torch.where(total == 0, 1, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(len(lq), mq, hq, D)
    # the sequences' rows one after the other
    b = torch.searchsorted(cq, torch.arange(s["q"].shape[0], device=DEV), right=True) - 1
    return o[b, torch.arange(s["q"].shape[0], device=DEV) - cq[b]].to(torch.bfloat16)


def _plain_linear(s):
    c, p = s["case"], s["packed"]
    n = c["n"] * (2 if c["swiglu"] else 1)
    shifts = _ints([0, 16, 4, 20, 8, 24, 12, 28])
    w = ((p[..., None] >> shifts) & 15).float() - 8  # [tiles, steps, lane, dword, code]
    tiles, steps = p.shape[:2]
    w = w.view(tiles, steps, 4, 16, 4, 8).permute(0, 3, 1, 4, 2, 5).reshape(tiles * 16, -1)
    sc = s["scales"].float().permute(0, 2, 1).reshape(tiles * 16, -1)
    w = (w.view(tiles * 16, -1, c["group"]) * sc[..., None]).view(tiles * 16, -1)[:n, :c["k"]]
    y = F.linear(s["x"].float(), w)
    if c["swiglu"]:
        gate, up = y[:, :c["n"]], y[:, c["n"]:]
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(torch.bfloat16)


def _plain_logprobs(s):
    x = s["logits"].float()
    if s["temperatures"] is not None:
        x = x / s["temperatures"][:, None]
    rows, vocab = x.shape
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    entropy = log_total - (e * d).sum(1) / total
    chosen = d.gather(1, s["tokens"][:, None])[:, 0] - log_total
    if not s["case"]["top"]:
        return [chosen, entropy]
    # whole numbers that order the values, the lower index first among equal ones
    bits = (s["logits"].float() + 0.0).view(torch.int32)  # -0.0 as 0.0
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() * (1 << 32)
    order += vocab - 1 - torch.arange(vocab, device=DEV)
    ids = vocab - 1 - (torch.topk(order, s["case"]["top"], dim=1).values & 0xffffffff)
    return [chosen, entropy, ids, d.gather(1, ids) - log_total[:, None]]


_OWN = dict(store=_own_store, attend=_own_attend, linear=_own_linear, logprobs=_own_logprobs)
_PLAIN = dict(store=_plain_store, attend=_plain_attend, linear=_plain_linear,
              logprobs=_plain_logprobs)


# ---------------------------------------------------------------- work

def work(case):
    """Bytes that have to be read and written and operations of one pass."""
    kind = case["kind"]
    if kind in ("store", "attend"):
        lens, (hq, heads) = _lens(case), HEADS[case["model"]]
        n, keys = sum(q for q, _ in lens), sum(k for _, k in lens)
    if kind == "store":
        groups = sum(-(-k // case["group"]) - (k - q) // case["group"] for q, k in lens)
        return dict(bytes=2 * n * heads * D * 3 + groups * heads * 8 + 4 * n,
                    flops=2 * n * heads * D * 2)
    if kind == "attend":
        pairs = sum(sum(k - q + i + 1 for i in range(q)) for q, k in lens)
        groups = sum(-(-k // case["group"]) for _, k in lens)
        return dict(bytes=2 * keys * heads * D + groups * heads * 8 + 4 * n * hq * D,
                    flops=4 * pairs * hq * D)
    if kind == "linear":
        n = case["n"] * (2 if case["swiglu"] else 1)
        return dict(bytes=n * case["k"] // 2 + 2 * n * case["k"] // case["group"]
                    + 2 * case["rows"] * (case["k"] + case["n"]),
                    flops=2 * case["rows"] * n * case["k"])
    esz = 2 if case["logits"] == "bf16" else 4
    return dict(bytes=case["rows"] * (case["vocab"] * esz + 16 + 12 * case["top"]),
                flops=4 * case["rows"] * case["vocab"])


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.inference_mode():
        return _EXACT[case["kind"]](case, s, seed)


def _e4m3(x):
    """The e4m3 value nearest to x (a double): three bits behind the leading one, steps of
    2^-9 below 2^-6, ties to the even one, at most 448."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_store(case, s, seed):
    group, out, new_scales = case["group"], [], []
    slots = s["slots"].tolist()
    touched = {}
    for t, slot in enumerate(slots):
        touched.setdefault(slot // group, []).append((slot % group, t))
    for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = x.double()
        c = codes.double().view(-1, group, *codes.shape[2:])
        sc = scales.double().view(-1, scales.shape[2])
        for g, members in touched.items():
            at, ts = _ints([o for o, _ in members], torch.int64), _ints([t for _, t in members],
                                                                        torch.int64)
            most = x[ts].abs().amax((0, 2))
            need = torch.exp2(torch.ceil(torch.log2(most / E4M3_MAX)).clamp(min=MIN_EXP))
            if members[0][0] == 0:
                new = need
            else:
                new = torch.maximum(sc[g], need)
                c[g] = _e4m3(c[g] * (sc[g] / new)[:, None])
            sc[g] = new
            c[g, at] = _e4m3(x[ts] / new[:, None])
        out.append(c.view(codes.shape))
        new_scales.append(sc.view(scales.shape))
    return out + new_scales


def _exact_attend(case, s, seed):
    hq, heads = HEADS[case["model"]]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    first = 0
    for b, (nq, nk) in enumerate(_lens(case)):
        blocks = s["tables"][b, :-(-nk // BLOCK)].long()
        k, v = (c[blocks].double().view(-1, BLOCK // case["group"], case["group"], heads, D)
                * sc[blocks].double()[:, :, None, :, None]
                for c, sc in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
        k, v = (t.reshape(-1, heads, D)[:nk] for t in (k, v))
        hidden = torch.ones(nq, nk, dtype=torch.bool, device=DEV).triu(nk - nq + 1)
        for h in range(hq):
            kvh = h // (hq // heads)
            a = s["q"][first:first + nq, h].double() @ k[:, kvh].t().contiguous() / math.sqrt(D)
            a = torch.softmax(a.masked_fill(hidden, -math.inf), 1)
            out[first:first + nq, h] = a @ v[:, kvh].contiguous()
        first += nq
    return out


def _exact_linear(case, s, seed):
    codes, scales = _weights(case, _gen(seed))
    y = []
    for i in range(0, codes.shape[0], 16384):
        w = codes[i:i + 16384].double() - 8
        w *= scales[i:i + 16384].double().repeat_interleave(case["group"], 1)
        y.append(s["x"].double() @ w.t().contiguous())
    y = torch.cat(y, 1)
    if case["swiglu"]:
        y = F.silu(y[:, :case["n"]]) * y[:, case["n"]:]
    return y


def _exact_logprobs(case, s, seed):
    out = [[], [], [], []]
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        if s["temperatures"] is not None:
            x = x / s["temperatures"][r].double()
        lp = torch.log_softmax(x, 0)
        out[0].append(lp[s["tokens"][r]])
        out[1].append(-(lp.exp() * lp).sum())
        if case["top"]:
            _, at = torch.sort(s["logits"][r].double(), descending=True, stable=True)
            out[2].append(at[:case["top"]])
            out[3].append(lp[at[:case["top"]]])
    return [torch.stack(o) for o in out if o]


_EXACT = dict(store=_exact_store, attend=_exact_attend, linear=_exact_linear,
              logprobs=_exact_logprobs)
