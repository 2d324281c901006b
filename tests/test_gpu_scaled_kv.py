"""The 8-bit cache with group scales on the GPU: the store against its 64-bit restatement,
bit for bit, and decode / verify / prompt attention over it within derived tolerances."""
import numpy as np
import pytest
import torch

import scaled_ref as ref

pytestmark = pytest.mark.gpu
D = 128


def _rows(gen, n, h, spread=6.0):
    """bf16 rows whose tokens and heads differ widely in size."""
    x = torch.randn(n, h, D, generator=gen) * torch.exp2(torch.rand(n, h, 1, generator=gen)
                                                        * spread - spread / 2)
    return x.to(torch.bfloat16)


def _cache(gen, nb, bs, h, group):
    codes = torch.randn(nb, bs, h, D, generator=gen) * 60
    codes = codes.clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.exp2(torch.randint(-9, -4, (nb, bs // group, h), generator=gen).float())
    return codes, scales


# name, kv heads, blocks, block size, group, calls (each a list of slots)
_STORES = [
    ("one-token", 8, 3, 256, 32, [[300]]),
    ("appends", 2, 2, 64, 32, [[32], [33], [34, 35], [36], [37, 38, 39, 40, 41], [42]]),
    ("decode", 8, 40, 256, 64, [[(i * 256 + 37 * i) % 10240 for i in range(40)]]),
    ("prompt", 4, 6, 96, 32, [list(range(96, 96 + 250)), list(range(346, 500))]),
    ("ragged-prompts", 8, 12, 256, 128, [list(range(512, 1291)) + list(range(5, 70)) + [1500]
                                         + list(range(2000, 2600))]),
    ("scattered", 1, 4, 256, 256, [[(i * 389) % 1024 for i in range(700)]]),
    ("skipped", 8, 2, 256, 32, [[-1, 40, -1, 41, 512, 100000, 2147483647, -2147483648, 42]]),
    ("repeated", 2, 2, 64, 64, [[70, 71, 70, 72, 70], [64, 64], [90, 91, 90]]),
    ("last-slots", 3, 2, 32, 32, [[63, 31], list(range(64))]),
    ("many-chunks", 2, 20, 256, 32, [[(i * 1031) % 5120 for i in range(2500)]]),
]


@pytest.mark.parametrize("case", _STORES, ids=[c[0] for c in _STORES])
def test_store(hv, cuda, case):
    name, H, nb, bs, group, calls = case
    print(f"scaled store {name}", flush=True)
    gen = torch.Generator().manual_seed(len(name) * 7 + nb)
    # planes of a layered cache: strides larger than the shape's own
    kc, ks = _cache(gen, 2 * nb, bs, H, group)
    vc, vs = _cache(gen, 2 * nb, bs, H, group)
    if name == "appends":
        ks.zero_(), vs.zero_()  # a new cache
    dk, dv, dks, dvs = (t.view(nb, 2, *t.shape[1:]).to(cuda)[:, 1] for t in (kc, vc, ks, vs))
    want = [t.view(nb, 2, *t.shape[1:])[:, 1].double().numpy().copy() for t in (kc, vc, ks, vs)]
    before = [t._base.clone() if t._base is not None else None for t in (dk, dv)]
    for slots in calls:
        x = _rows(gen, len(slots), 2 * H)
        dx = x.to(cuda)
        hv.ops.store_kvcache_scaled(dx[:, :H], dx[:, H:], dk, dv, dks, dvs,
                                    torch.tensor(slots, dtype=torch.int32, device=cuda))
        ref.store(x[:, :H].double().numpy(), want[0], want[2], slots)
        ref.store(x[:, H:].double().numpy(), want[1], want[3], slots)
        for got, w in zip((dk, dv, dks, dvs), want):
            assert np.array_equal(got.double().cpu().numpy(), w, equal_nan=True)
    for t, b in zip((dk, dv), before):  # the other plane is as it was
        if b is not None:
            assert torch.equal(t._base[:, 0].view(torch.uint8), b[:, 0].view(torch.uint8))


def test_store_values_that_are_not_finite(hv, cuda):
    """NaN becomes the NaN code, infinities saturate at the scale of the finite values, and
    rows of zeros or tiny values take the smallest scale."""
    gen = torch.Generator().manual_seed(3)
    H, nb, bs, group = 2, 2, 64, 32
    x = _rows(gen, 6, H)
    x[0, 0, 5], x[1, 0, 7], x[2, 0, 9] = float("nan"), float("inf"), float("-inf")
    x[:, 1] = 0
    x[3, 1, 0] = 2.0 ** -125
    x[4, 1, 1] = -(2.0 ** -130)  # subnormal
    slots = [32, 33, 34, 3, 40, 41]
    kc, ks = _cache(gen, nb, bs, H, group)
    want = [kc.double().numpy().copy(), ks.double().numpy().copy()]
    dk, dks = kc.to(cuda), ks.to(cuda)
    dv, dvs = dk.clone(), dks.clone()
    dx = x.to(cuda)
    hv.ops.store_kvcache_scaled(dx, dx, dk, dv, dks, dvs,
                                torch.tensor(slots, dtype=torch.int32, device=cuda))
    ref.store(x.double().numpy(), want[0], want[1], slots)
    for c, s in ((dk, dks), (dv, dvs)):
        assert np.array_equal(c.double().cpu().numpy(), want[0], equal_nan=True)
        assert np.array_equal(s.double().cpu().numpy(), want[1])


def test_store_keeps_a_larger_scale_of_another_producer(hv, cuda):
    """A stored scale that is no power of two stays while it suffices, and its codes move
    to the next power of two once it does not."""
    H, nb, bs, group = 1, 1, 32, 32
    kc = torch.full((nb, bs, H, D), 3.0).to(torch.float8_e4m3fn)
    ks = torch.full((nb, 1, H), 0.37)
    want = [kc.double().numpy().copy(), ks.double().numpy().copy()]
    dk, dks = kc.to(cuda), ks.to(cuda)
    dv, dvs = dk.clone(), dks.clone()
    for slot, size in ((5, 100.0), (6, 165.0), (7, 166.0), (8, 1000.0)):
        x = torch.full((1, H, D), size, dtype=torch.bfloat16)
        x[0, 0, 1::2] = -0.11
        dx = x.to(cuda)
        hv.ops.store_kvcache_scaled(dx, dx, dk, dv, dks, dvs,
                                    torch.tensor([slot], dtype=torch.int32, device=cuda))
        want[1] = want[1].astype(np.float32).astype(np.float64)
        ref.store(x.double().numpy(), want[0], want[1], [slot])
        assert torch.equal(dk.view(torch.uint8), dv.view(torch.uint8))
        got = dk.double().cpu().numpy()
        assert np.array_equal(dks.double().cpu().numpy(), want[1])
        # x / 0.37 rounds in 32 bits before it rounds to a code: the nearest code or, within
        # 2^-22 of a middle between two, its neighbour (one step is 2^-3 at the most)
        assert np.all(np.abs(got - want[0]) <= 2.0 ** -3 * np.abs(want[0]) + 2.0 ** -9)
        assert np.mean(got != want[0]) == 0 or size < 165


# name, Hq, Hkv, block size, group, query lengths, key lengths, declared longest sequence
_ATTEND = [
    ("b1-verify", 32, 8, 256, 32, [4], [320], 4096),
    ("decode-edges", 32, 8, 256, 32, [1] * 12, [1, 2, 31, 32, 33, 63, 64, 255, 256, 257, 511, 513],
     2048),
    ("verify-ragged", 16, 8, 256, 64, [4, 1, 3, 2, 4, 4], [4, 700, 3, 65, 2047, 1300], 2048),
    ("splits", 16, 8, 256, 128, [2, 2], [3001, 2500], 3001),
    ("longer-than-declared", 16, 8, 64, 32, [2, 1], [1500, 90], 300),
    ("more-queries-than-keys", 32, 8, 256, 32, [6, 4, 5], [3, 4, 0], 256),
    ("no-queries", 32, 8, 256, 32, [0, 2, 0, 1], [40, 70, 0, 33], 256),
    ("group-1", 8, 8, 96, 32, [9, 5], [200, 95], 256),
    ("group-16", 32, 2, 32, 32, [3, 1], [77, 400], 512),
    ("group-5", 10, 2, 160, 32, [4, 7], [77, 400], 512),
    ("two-tiles", 32, 8, 256, 256, [9, 16], [300, 16], 512),
    ("prompts", 32, 8, 256, 32, [61, 130, 1], [61, 333, 500], 512),
    ("prompt-group-1", 4, 4, 256, 128, [300, 77], [300, 400], 512),
    # one, two and three tiles to a wave, and keys past the first 64 windows
    ("prompts-1", 32, 8, 256, 32, [130, 61], [333, 61], 512),
    ("prompts-2", 32, 8, 256, 64, [390, 7], [2500, 1000], 4096),
    ("prompts-3", 64, 64, 96, 32, [400, 391, 17, 250], [400, 1300, 64, 249], 2048),
    ("prompts-3-group-8", 128, 16, 256, 256, [300, 290, 1], [2300, 290, 31], 4096),
    ("prompt-odd-heads", 14, 2, 96, 32, [97, 30], [97, 30], 512),
]


def _attend_inputs(cuda, case, seed=0, plane=True):
    name, Hq, Hkv, bs, group, lq, lk, declared = case
    gen = torch.Generator().manual_seed(seed + len(name))
    nblk = [-(-n // bs) for n in lk]
    nb = sum(nblk) + 2
    perm = torch.randperm(nb, generator=gen)
    bt = torch.full((len(lk), max(nblk) + 2), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(nblk):
        bt[b, :n] = perm[at:at + n].int()
        at += n
    kc, ks = _cache(gen, nb, bs, Hkv, group)
    vc, vs = _cache(gen, nb, bs, Hkv, group)
    # slots behind the sequences' ends hold anything: NaN codes, and NaN scales where a
    # whole group lies there
    used = torch.zeros(nb, bs, dtype=torch.bool)
    for b, n in enumerate(lk):
        for i in range(n):
            used[int(bt[b, i // bs]), i % bs] = True
    for c, s in ((kc, ks), (vc, vs)):
        c.view(torch.uint8)[~used] = 0x7f
        s[~used.view(nb, -1, group).any(2)] = float("nan")
    q = torch.randn(sum(lq), Hq, D, generator=gen).to(torch.bfloat16)
    cu = [torch.tensor([0] + list(np.cumsum(x)), dtype=torch.int32) for x in (lq, lk)]
    host = dict(q=q, kc=kc, vc=vc, ks=ks, vs=vs, bt=bt, cu_q=cu[0], cu_k=cu[1])
    return host, {k: v.to(cuda) for k, v in host.items()}


def _run(hv, case, x, out=None):
    return hv.ops.verify_attention_scaled(x["q"], x["kc"], x["vc"], x["ks"], x["vs"], x["bt"],
                                          x["cu_q"], x["cu_k"], max(case[5]), case[7], D ** -0.5,
                                          out=out)


def _check(case, host, got):
    _, Hq, Hkv, bs, group, lq, lk, _ = case
    at = 0
    for b, (nq, nk) in enumerate(zip(lq, lk)):
        blocks = host["bt"][b, :-(-nk // bs)].long()
        k, v = ((c[blocks].double().view(-1, bs // group, group, Hkv, D)
                 * s[blocks].double()[:, :, None, :, None]).reshape(-1, Hkv, D)[:nk].numpy()
                for c, s in ((host["kc"], host["ks"]), (host["vc"], host["vs"])))
        out, most, size = ref.attention(host["q"][at:at + nq].double().numpy(), k, v, nq, nk,
                                        D ** -0.5)
        g = got[at:at + nq].double().cpu().numpy()
        assert np.array_equal(np.isnan(g), np.isnan(out)), (case[0], b)
        err, tol = np.abs(g - out), ref.tolerance(out, most, size)
        fine = ~np.isnan(out)
        assert np.all(err[fine] <= tol[fine]), (case[0], b, np.max((err / tol)[fine]))
        at += nq


@pytest.mark.parametrize("case", _ATTEND, ids=[c[0] for c in _ATTEND])
def test_attention(hv, cuda, case):
    print(f"scaled attention {case[0]}", flush=True)
    host, x = _attend_inputs(cuda, case)
    _check(case, host, _run(hv, case, x))


@pytest.mark.parametrize("case", [c for c in _ATTEND if c[0] in ("verify-ragged", "prompts-1", "prompts-2",
                                                                 "prompts-3")],
                         ids=["verify", "prompts-1", "prompts-2", "prompts-3"])
def test_nan_values_stay_with_the_rows_that_see_them(hv, cuda, case):
    """A NaN code of V or K in a key that only later query rows see leaves the earlier rows'
    results as they are."""
    host, x = _attend_inputs(cuda, case, seed=1)
    bs = case[3]
    for b, (nq, nk) in enumerate(zip(case[5], case[6])):
        last = nk - 1  # seen by the last row alone
        blk = int(host["bt"][b, last // bs])
        host["vc"].view(torch.uint8)[blk, last % bs, 0, 3] = 0x7f
        host["vc"].view(torch.uint8)[blk, last % bs, 1, 120] = 0xff
        if nq > 1:
            host["kc"].view(torch.uint8)[blk, last % bs, 2, 11] = 0xff
    x = {k: v.to(cuda) for k, v in host.items()}
    _check(case, host, _run(hv, case, x))


@pytest.mark.parametrize("case", [c for c in _ATTEND if c[0] in ("splits", "prompts-1", "prompts-3")],
                         ids=["splits", "prompts-1", "prompts-3"])
def test_views_and_rows_behind_the_last_sequence(hv, cuda, case):
    """q and out as slices of wider rows, caches as planes of a layered cache; rows of out
    behind the last sequence's stay as they were."""
    host, x = _attend_inputs(cuda, case, seed=2)
    N, Hq = host["q"].shape[:2]
    wide = torch.randn(N + 5, Hq + 3, D, device=cuda).to(torch.bfloat16)
    wide[:N, 1:1 + Hq] = x["q"]
    planes = {k: torch.stack([torch.zeros_like(x[k]), x[k]], 1)[:, 1] for k in ("kc", "vc", "ks", "vs")}
    out = torch.full((N + 5, Hq + 2, D), 7.0, dtype=torch.bfloat16, device=cuda)
    y = dict(x, q=wide[:, 1:1 + Hq], **planes)
    _run(hv, case, y, out=out[:, 2:])
    _check(case, host, out[:N, 2:])
    assert bool((out[N:] == 7).all()) and bool((out[:, :2] == 7).all())


def test_scales_that_are_no_powers_of_two(hv, cuda):
    """Scales of another producer: of any size, zero among them."""
    case = ("odd-scales", 16, 8, 64, 32, [4, 2, 150], [200, 130, 150], 512)
    host, _ = _attend_inputs(cuda, case, seed=5)
    for k in ("ks", "vs"):
        live = ~host[k].isnan()
        host[k][live] = (torch.rand(int(live.sum()), generator=torch.Generator().manual_seed(1))
                         * 0.03 + 1e-3)
        host[k][:, 0, 3] = torch.where(live[:, 0, 3], 0.0, host[k][:, 0, 3])
    host["vs"][:, 1, 2] *= -1
    x = {k: v.to(cuda) for k, v in host.items()}
    _check(case, host, _run(hv, case, x))
    big = ("odd-scales-prompt", 16, 8, 64, 32, [1100, 2], [1200, 130], 2048)
    host, _ = _attend_inputs(cuda, big, seed=6)
    host["vs"] *= 0.7
    x = {k: v.to(cuda) for k, v in host.items()}
    _check(big, host, _run(hv, big, x))


def test_blocks_that_the_table_does_not_have_are_left_out(hv, cuda):
    """Entries outside the pool, and positions past the table, give no keys."""
    case = ("bad-blocks", 16, 8, 64, 32, [2, 1, 1], [200, 130, 64], 512)
    host, x = _attend_inputs(cuda, case, seed=3)
    nb = host["kc"].shape[0]
    host["bt"][0, 1] = -1
    host["bt"][1, 0] = nb
    host["bt"][2, 0] = -5
    x["bt"] = host["bt"][:, :3].to(cuda)  # sequence 0's fourth block lies past the table
    got = _run(hv, case, x).double().cpu().numpy()
    Hkv, group, bs = 8, 32, 64
    live = {0: [0, 2], 1: [1, 2], 2: []}
    at = 0
    for b, (nq, nk) in enumerate(zip(case[5], case[6])):
        keep = [i for i in range(nk) if i // bs in live[b]]
        k, v = (np.stack([(c[int(host["bt"][b, i // bs]), i % bs].double()
                           * s[int(host["bt"][b, i // bs]), i % bs // group].double()[:, None]).numpy()
                          for i in keep]) if keep else np.zeros((0, Hkv, D))
                for c, s in ((host["kc"], host["ks"]), (host["vc"], host["vs"])))
        for r in range(nq):
            n = sum(i < nk - nq + r + 1 for i in keep)
            out, most, size = ref.attention(host["q"][at:at + 1].double().numpy(), k[:n], v[:n], 1,
                                            n, D ** -0.5)
            assert np.all(np.abs(got[at] - out[0]) <= ref.tolerance(out, most, size)[0])
            at += 1


def test_two_streams_and_a_replayed_graph(hv, cuda):
    """Calls in flight on two streams, and a captured one replayed between eager calls,
    give what each gives alone."""
    cases = [c for c in _ATTEND if c[0] in ("splits", "verify-ragged")]
    xs = [_attend_inputs(cuda, c, seed=4)[1] for c in cases]
    want = [_run(hv, c, x) for c, x in zip(cases, xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_run(hv, cases[i], xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g.view(torch.int16), want[i].view(torch.int16)) for g in got[i])
    graphs = []
    for i in range(2):
        g, s = torch.cuda.CUDAGraph(), streams[i]
        with torch.cuda.graph(g, stream=s):
            out = _run(hv, cases[i], xs[i])
        graphs.append((g, out))
    for _ in range(3):
        for i, (g, out) in enumerate(graphs):
            out.zero_()
            g.replay()
            eager = _run(hv, cases[1 - i], xs[1 - i])
            torch.cuda.synchronize()
            assert torch.equal(out.view(torch.int16), want[i].view(torch.int16))
            assert torch.equal(eager.view(torch.int16), want[1 - i].view(torch.int16))


def test_store_at_the_ends_of_the_range(hv, cuda):
    """Scales whose 448-fold is past the largest f32: an infinity still saturates, and the
    group's other codes still move to the raised scale."""
    print("scaled store, largest scales", flush=True)
    gen = torch.Generator().manual_seed(2)
    olds = [1.3e36, 0.0, 1e37, 2.0 ** -120, 3e38]  # of five blocks of one group each
    slots = [5, 32, 64 + 9, 96 + 1, 128 + 30]
    k = torch.randn(5, 1, D, generator=gen).to(torch.bfloat16)
    k[:, :, 0], k[:, :, 1], k[:, :, 2] = 3.3e38, float("inf"), float("-inf")
    v = (torch.randn(5, 1, D, generator=gen) * 1e30).to(torch.bfloat16)
    v[:, :, 7] = float("-inf")
    codes = (torch.randn(5, 32, 1, D, generator=gen) * 300).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.tensor(olds).view(5, 1, 1)
    dk, dv, dks, dvs = (t.clone().to(cuda) for t in (codes, codes, scales, scales))
    want = [t.double().numpy().copy() for t in (codes, codes, scales, scales)]
    hv.ops.store_kvcache_scaled(k.to(cuda), v.to(cuda), dk, dv, dks, dvs,
                                torch.tensor(slots, dtype=torch.int32, device=cuda))
    ref.store(k.double().numpy(), want[0], want[2], slots)
    ref.store(v.double().numpy(), want[1], want[3], slots)
    for got, w in zip((dk, dv, dks, dvs), want):
        assert np.array_equal(got.double().cpu().numpy(), w, equal_nan=True)


_FEW_SPLITS = [
    ("few-longer-than-declared", 16, 8, 64, 32, [2, 1], [1500, 90], 600),
    ("few-group-5", 10, 2, 160, 32, [4, 7], [77, 900], 900),
    ("few-no-queries", 32, 8, 256, 64, [0, 2, 0, 1], [40, 1024, 0, 33], 1024),
    ("one-split-at-its-limit", 32, 8, 256, 32, [4, 3], [512, 511], 512),
    ("one-split-of-1024", 32, 8, 256, 32, [1] * 16, [1024 - 61 * i for i in range(16)], 1024),
    ("many-of-1025", 32, 8, 256, 32, [1] * 16, [1025 - 61 * i for i in range(16)], 1025),
]


@pytest.mark.parametrize("case", _FEW_SPLITS, ids=[c[0] for c in _FEW_SPLITS])
def test_attention_with_few_splits(hv, cuda, case):
    """Where a call leaves its keys whole, and where two to nine workgroups share them."""
    test_attention(hv, cuda, case)
