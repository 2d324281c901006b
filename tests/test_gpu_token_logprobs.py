"""Log-probabilities, entropy and top alternatives on the GPU against 64-bit sums and a
stable sort."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# rows, vocabulary, top
_SIZES = [(1, 1, 1), (3, 7, 7), (2, 33, 32), (5, 1001, 0), (4, 2048, 20), (2, 2049, 5),
          (1, 8193, 32), (4, 151936, 5), (30, 151936, 20), (300, 32003, 1), (70, 100003, 20),
          (2, 1 << 21, 32)]


def _reference(x, tokens, top, temps):
    y = x.double() if temps is None else x.double() / temps.double()[:, None]
    lp = torch.log_softmax(y, 1)
    p = lp.exp()
    ent = -torch.where(p == 0, 0, p * lp).sum(1)
    V = x.shape[1]
    chosen = torch.where((tokens >= 0) & (tokens < V), lp.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0],
                         -float("inf"))
    # NaN first, then by value, ties (and -0 against 0) by index
    key = torch.where(x.isnan(), float("inf"), x.double() + 0.0)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    if x.isnan().any():
        order = order.gather(1, torch.sort(x.isnan().gather(1, order).to(torch.uint8), dim=1,
                                           descending=True, stable=True).indices)
    ids = order[:, :top]
    return chosen, ent, ids, lp.gather(1, ids), y, lp


def _check(got, x, tokens, top, temps):
    chosen, ent, ids, tlp, y, lp = _reference(x, tokens, top, temps)
    m = y.abs().nan_to_num(0, 0, 0).amax(1)
    log_s = (y.amax(1) - (lp + 0).amax(1)).nan_to_num(0, 0, 0).abs()  # about 0, at least finite
    spread = (lp.exp() * lp.abs().nan_to_num(0, 0, 0)).nan_to_num(0).sum(1)
    # y is a product rounded twice, m and ln S are subtracted in 32 bits, S has fewer
    # than 64 roundings on the way to any term, and a term's exponent is off by 2^-22
    # (|m| + |d|), where terms with |d| > 32 weigh nothing: 2^-21 of all that together
    tol = 2.0 ** -21 * (2 * m + log_s + 32)

    def near(a, b, t):
        a = a.double().cpu()
        assert torch.equal(a.isnan(), b.isnan())
        fine = b.isfinite()
        assert torch.equal(a[~fine].nan_to_num(1.5, 2, 3), b[~fine].nan_to_num(1.5, 2, 3))
        err = ((a - b).abs() - t - 2.0 ** -22 * b.abs())[fine]
        assert not err.numel() or float(err.max()) <= 0, float(err.max())

    near(got["logprobs"], chosen, tol)
    near(got["entropy"], ent, tol + 2.0 ** -17 * spread)
    if top:
        assert torch.equal(got["top_ids"].cpu(), ids)
        near(got["top_logprobs"], tlp, tol[:, None])
    else:
        assert got["top_ids"] is None and got["top_logprobs"] is None


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("size", _SIZES, ids=["x".join(map(str, s)) for s in _SIZES])
def test_token_logprobs(hv, cuda, size, dtype):
    rows, V, top = size
    print("token logprobs", size, dtype, flush=True)
    gen = torch.Generator().manual_seed(rows + V)
    x = torch.randn(rows, V, generator=gen) * 4
    x = x.to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    tokens = torch.randint(V, (rows,), generator=gen)
    temps = torch.rand(rows, generator=gen) + 0.4 if rows != 4 else None
    got = hv.ops.token_logprobs(x.to(cuda), tokens.to(cuda), top=top,
                                temperatures=None if temps is None else temps.to(cuda))
    _check(got, x, tokens, top, temps)
    # rows of a wider tensor, off the 16-byte alignment
    wide = torch.zeros(rows, V + 3, dtype=x.dtype, device=cuda)
    wide[:, 1:1 + V] = x.to(cuda)
    again = hv.ops.token_logprobs(wide[:, 1:1 + V], tokens.to(cuda), top=top,
                                  temperatures=None if temps is None else temps.to(cuda))
    for k, v in got.items():
        assert v is None or torch.equal(v, again[k])


@pytest.mark.parametrize("rows", [6, 300])
def test_rows_at_the_edges(hv, cuda, rows):
    """Ties over the whole row and across chunks, sorted rows, masked tokens, rows that are
    certain, and rows whose values are not finite."""
    V, top = 20001, 20
    inf, nan = float("inf"), float("nan")
    x = torch.randn(rows, V, generator=torch.Generator().manual_seed(1)) * 3
    x[0] = 1.25  # every value the same
    x[1] = torch.arange(V) * 0.001  # ascending
    x[2] = torch.arange(V, 0, -1) * 0.001
    x[3] = -inf  # all but three masked, two of them equal
    x[3, [19999, 5, 8200]] = torch.tensor([2.0, 2.0, -1.0])
    x[4, :] = -50
    x[4, 12345] = 40  # certain
    x[5, ::2] = 0.0
    x[5, 1::2] = -0.0
    if rows > 6:
        x[6] = -inf
        x[7, 77] = nan
        x[8, [3, 900]] = inf
        x[9, [15000, 2]] = nan
        x[10, 100:] = -inf
        x[11] = torch.round(x[11])
        x[12] = -3.0e38
    tokens = torch.randint(V, (rows,), generator=torch.Generator().manual_seed(2))
    tokens[3], tokens[4] = 8200, 12345
    tokens[rows - 1], tokens[rows - 2] = -1, V
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        got = hv.ops.token_logprobs(y.to(cuda), tokens.to(cuda), top=top)
        _check(got, y, tokens, top, None)


@pytest.mark.parametrize("rows", [3, 300])
def test_alternatives_do_not_go_by_the_temperature(hv, cuda, rows):
    """The order is that of the logits, also where a temperature outside its domain leaves
    no log-probabilities."""
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(rows, 9001, generator=gen)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :20]
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-30):
        got = hv.ops.token_logprobs(x.to(cuda), top=20,
                                    temperatures=torch.full((rows,), t, device=cuda))
        assert torch.equal(got["top_ids"].cpu(), ids)


def test_arguments_left_out(hv, cuda):
    x = torch.randn(3, 500, device=cuda)
    r = hv.ops.token_logprobs(x)
    assert r["logprobs"] is None and r["top_ids"] is None
    t = hv.ops.token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=cuda), top=2)
    assert torch.equal(t["entropy"], r["entropy"])
    e = hv.ops.token_logprobs(x[:0], torch.zeros(0, dtype=torch.int64, device=cuda), top=2)
    assert e["logprobs"].shape == (0,) and e["top_ids"].shape == (0, 2)


def test_replayed_graphs_and_streams(hv, cuda):
    gen = torch.Generator().manual_seed(4)
    xs = [torch.randn(r, 151936, generator=gen).to(torch.bfloat16).to(cuda) for r in (4, 40)]
    toks = [torch.randint(151936, (x.shape[0],), generator=gen).to(cuda) for x in xs]
    want = [hv.ops.token_logprobs(x, t, top=5) for x, t in zip(xs, toks)]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x, t, s in zip(xs, toks, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            r = hv.ops.token_logprobs(x, t, top=5)
        graphs.append((g, r))
    for _ in range(3):
        for s, (g, r) in zip(streams, graphs):
            with torch.cuda.stream(s):
                for v in r.values():
                    v.zero_()
                g.replay()
        eager = [hv.ops.token_logprobs(x, t, top=5) for x, t in zip(xs, toks)]
        torch.cuda.synchronize()
        for i in range(2):
            for k in want[i]:
                assert torch.equal(graphs[i][1][k], want[i][k])
                assert torch.equal(eager[i][k], want[i][k])
