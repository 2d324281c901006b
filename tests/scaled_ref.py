"""Plain restatements, in 64 bits, of the 8-bit cache with group scales: its store and
the attention over it (numpy / torch on the host)."""
import math

import numpy as np
import torch

E4M3_MAX = 448.0


def e4m3(x):
    """The e4m3 value nearest to each double: steps of 2^(e - 3) from 2^e on, of 2^-9 below
    2^-6, ties to the even one, at most +-448; NaN stays."""
    x = np.asarray(x, np.float64)
    _, e = np.frexp(np.where(np.isfinite(x), x, 448.0))
    step = np.ldexp(1.0, np.maximum(e - 4, -9))
    with np.errstate(invalid="ignore"):
        return np.clip(np.rint(np.where(np.isinf(x), np.sign(x) * 1e9, x) / step) * step,
                       -E4M3_MAX, E4M3_MAX)


def codes_of(values):
    """float8_e4m3fn tensor of exactly representable doubles (or NaN)."""
    t = torch.from_numpy(np.ascontiguousarray(values)).float().to(torch.float8_e4m3fn)
    back = t.double().numpy()
    assert np.array_equal(back, values, equal_nan=True)
    return t


def need_of(a):
    """The smallest power of two >= a / 448, at least 2^-96."""
    if not a > 0:
        return 2.0 ** -96
    e = math.floor(math.log2(a / E4M3_MAX)) - 2
    while not a <= E4M3_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** max(e, -96)


def store(x, codes, scales, slots):
    """x [N, H, D] doubles into codes [nb, bs, H, D] / scales [nb, bs / group, H] (doubles,
    changed in place)."""
    nb, bs, H, _ = codes.shape
    group = bs // scales.shape[1]
    touched = {}
    for t, s in enumerate(slots):
        if s >= 0 and s // bs < nb:
            touched.setdefault((s // bs, s % bs // group), {}).setdefault(s % group, []).append(t)
    for (b, g), members in touched.items():
        for h in range(H):
            rows = [x[t, h] for ts in members.values() for t in ts]
            live = np.concatenate([x[ts[-1], h] for ts in members.values()])
            del rows
            live = np.abs(live[np.isfinite(live)])
            need = need_of(live.max() if live.size else 0.0)
            old = scales[b, g, h]
            fresh = 0 in members or not (old > 0 and np.isfinite(old))
            now = need if fresh else max(old, need)
            part = codes[b, g * group:(g + 1) * group, h]
            if not fresh and now > old:
                for o in range(group):
                    if o not in members:
                        part[o] = e4m3(part[o] * old / now)
            for o, ts in members.items():
                part[o] = e4m3(x[ts[-1], h] / now)
            scales[b, g, h] = now


def attention(q, k, v, Lq, Lk, scale):
    """One sequence: q [Lq, Hq, D], k / v [Lk, Hkv, D] doubles -> (out, sum p |v|, the largest
    sum |q k| of a row times the scale). NaN of a key or value reaches the rows that see it."""
    Hq, Hkv = q.shape[1], k.shape[1]
    out, most = np.zeros(q.shape), np.zeros(q.shape)
    size = np.zeros(q.shape[:2])
    if Lk == 0 or Lq == 0:
        return out, most, size
    seen = np.arange(Lk)[None] <= Lk - Lq + np.arange(Lq)[:, None]
    any_seen = seen.any(1)
    for h in range(Hq):
        kk, vv = k[:, h // (Hq // Hkv)], v[:, h // (Hq // Hkv)]
        s = np.where(seen, q[:, h] @ kk.T * scale, -np.inf)
        top = np.where(any_seen, s.max(1), 0.0)
        p = np.where(seen, np.exp(s - np.where(np.isnan(top), 0.0, top)[:, None]), 0.0)
        p /= np.where(any_seen, p.sum(1), 1.0)[:, None]
        clean = np.where(np.isnan(vv), 0.0, vv)
        out[:, h] = p @ clean
        hit = seen.astype(float) @ np.isnan(vv).astype(float) > 0
        out[:, h][hit] = np.nan
        most[:, h] = p @ np.abs(clean)
        size[:, h] = np.where(seen, np.abs(q[:, h]) @ np.abs(kk).T, 0.0).max(1) * abs(scale)
    return out, most, size


def tolerance(out, most, size):
    """Elementwise: each probability rounds to bf16 once, p_j (1 + d_j) with |d_j| <= 2^-8, in
    the sum above and in the sum below, which makes sum p v / sum p at most
    2^-8 (sum p |v| / sum p + |out|) / (1 - 2^-8) off (both sums move, by sum d p v and sum d p);
    a scale that is no power of two rounds the product's weights once more, and the output
    rounds once. Scores are sums of 128 exact products in 32 bits, so off by at most
    128 * 2^-24 of sum |q k|, which moves a probability (and the sum under it) by that
    share, with as much again for the products by the scale and the exponential; sums and
    rescalings in 32 bits: 2^-16."""
    return (2.0 ** -8 + 4 * 128 * 2.0 ** -24 * size[..., None] + 2.0 ** -16) * most * 1.01 \
        + 2 * 2.0 ** -8 * 1.01 * np.abs(out) + 1e-30
