"""Attention over the cache with group scales: the size of its error, and values that are
not finite."""
import math

import pytest
import torch

import test_gpu_scaled_kv as kv

pytestmark = pytest.mark.gpu

# decode and verify rows in one and in many splits, and prompts of one tile a wave
_CASES = [
    ("error-decode", 32, 8, 256, 32, [1] * 8, [2000, 1900, 1500, 700, 1100, 1024, 300, 1999], 2048),
    ("error-verify", 16, 8, 256, 64, [4] * 6, [500, 480, 333, 400, 290, 512], 512),
    ("error-long", 32, 8, 256, 128, [4], [9001], 10240),
    ("error-prompts-1", 32, 8, 256, 32, [130, 61], [333, 261], 512),
]


# prompts of two and three tiles a wave
_LONG = [c for c in kv._ATTEND if c[0] in ("prompts-2", "prompts-3")]


def _exact(case, host):
    """The results in 64 bits, and sum_j p_j^2 (v_j - o)^2: the square of how far errors of
    the probabilities that are independent and of relative size 1 would move them."""
    name, Hq, Hkv, bs, group, lq, lk, _ = case
    out, moves, at = [], [], 0
    for b, (nq, nk) in enumerate(zip(lq, lk)):
        blocks = host["bt"][b, :-(-nk // bs)].long()
        k, v = ((c[blocks].double().view(-1, bs // group, group, Hkv, 128)
                 * s[blocks].double()[:, :, None, :, None]).reshape(-1, Hkv, 128)[:nk]
                for c, s in ((host["kc"], host["ks"]), (host["vc"], host["vs"])))
        hidden = torch.ones(nq, nk, dtype=torch.bool).triu(nk - nq + 1)
        o, w = torch.zeros(nq, Hq, 128).double(), torch.zeros(nq, Hq, 128).double()
        for h in range(Hq):
            kk, vv = k[:, h // (Hq // Hkv)], v[:, h // (Hq // Hkv)]
            p = (host["q"][at:at + nq, h].double() @ kk.t() * 128 ** -0.5).masked_fill(hidden, -math.inf)
            p = torch.softmax(p, 1).masked_fill(hidden, 0)  # a row may see no key
            o[:, h] = p @ vv
            w[:, h] = (p * p) @ (vv * vv) - 2 * o[:, h] * ((p * p) @ vv) \
                + o[:, h] ** 2 * (p * p).sum(1, keepdim=True)
        out.append(o)
        moves.append(w)
        at += nq
    return torch.cat(out), torch.cat(moves).clamp(min=0)


def _rms(t):
    return float(t.square().mean().sqrt())


@pytest.mark.parametrize("odd", [False, True], ids=["powers-of-two", "other-scales"])
@pytest.mark.parametrize("case", _CASES + _LONG, ids=[c[0] for c in _CASES + _LONG])
def test_error_is_one_rounding(hv, cuda, case, odd):
    """The error's root mean square. Everywhere: that of rounding the exact results to bf16;
    the scores' 32-bit sums move the probabilities by some 2^-20, the probabilities' two bf16
    parts leave 2^-17 of each, which together is 2^-15 of the outputs at most. Prompts of two
    and three tiles a wave round each probability to bf16 once, half a step of 2^-7, evenly
    spread (2^-8 / sqrt 3), in the sum above and in the sum below alike. 2 % above the root sum
    of squares is room for the sample's spread. (One rounding in the first cases is 4 % and
    more; a second rounding of the product's weights alone, up to 60 %.)"""
    print("scaled attention, error", case[0], odd, flush=True)
    host, x = kv._attend_inputs(cuda, case, seed=7)
    if odd:
        for k in ("ks", "vs"):
            host[k] *= 0.83
        host["vs"][::2] *= -1
        x = {k: v.to(cuda) for k, v in host.items()}
    got = kv._run(hv, case, x).double().cpu()
    want, moves = _exact(case, host)
    parts = [_rms(want.to(torch.bfloat16).double() - want), 2.0 ** -15 * _rms(want)]
    if case in _LONG:
        parts.append(2.0 ** -8 / math.sqrt(3) * float(moves.mean().sqrt()))
    err = _rms(got - want)
    assert err <= 1.02 * math.hypot(*parts), (err, parts)


@pytest.mark.parametrize("rows", [1, 64, 200, 600, 1600])
def test_value_scales_at_the_ends_of_the_range(hv, cuda, rows):
    """One key a sequence: the output is its value, infinite where the scale is, and finite
    where the scale is negative and next to the largest number. (From one split tile to three
    tiles a wave.)"""
    print("scaled attention, scales at the ends", rows, flush=True)
    vs = [float("inf"), -float("inf"), -3.0e38, 3.0e38, 1e-40, -2.0 ** -130]
    nb = len(vs)
    codes = torch.tensor([1.0, -1.0, 0.5, -0.25, 1.0, 0.75]).repeat(22)[:128]
    vc = codes.view(1, 1, 1, 128).expand(nb, 32, 8, 128).contiguous().to(torch.float8_e4m3fn)
    kc = torch.ones(nb, 32, 8, 128).to(torch.float8_e4m3fn)
    scales = torch.tensor(vs).view(nb, 1, 1).expand(nb, 1, 8).contiguous()
    q = torch.randn(nb * rows, 32, 128, generator=torch.Generator().manual_seed(rows))
    # one row a sequence sees its key, the others see none and get zeros
    cu_q = torch.arange(nb + 1, dtype=torch.int32) * rows
    got = hv.ops.verify_attention_scaled(
        q.to(torch.bfloat16).to(cuda), kc.to(cuda), vc.to(cuda), torch.ones_like(scales).to(cuda),
        scales.to(cuda), torch.arange(nb, dtype=torch.int32)[:, None].to(cuda), cu_q.to(cuda),
        torch.arange(nb + 1, dtype=torch.int32).to(cuda), rows, 32, 0.1).cpu()
    got = got.view(nb, rows, 32, 128)
    assert bool((got[:, :-1] == 0).all())
    for b, s in enumerate(vs):
        want = (codes.double() * torch.tensor(s).double()).float().to(torch.bfloat16)
        assert torch.equal(got[b, -1], want.expand(32, 128)), (s, got[b, -1, 0, :6])
