"""Projections of rows in 8 bits by e4m3 weights on the GPU against the same sums in 64
bits."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu

# inputs, features, rows, epilogue
_CASES = [
    (16, 1, 1, "plain"), (128, 16, 2, "plain"), (96, 17, 5, "plain"), (352, 200, 16, "plain"),
    (1056, 1001, 3, "plain"), (1024, 4096, 7, "plain"), (4096, 6144, 4, "plain"),
    (4096, 20000, 1, "plain"), (12288, 4096, 16, "plain"), (256, 60000, 9, "plain"),
    (1024, 1001, 17, "plain"), (96, 40, 33, "plain"), (4096, 4096, 63, "plain"),
    (12288, 1024, 64, "plain"), (384, 777, 65, "plain"), (2048, 512, 300, "plain"),
    (128, 16, 130, "plain"), (160, 130000, 20, "plain"), (4096, 1024, 129, "plain"),
    (4096, 6144, 531, "plain"), (1040, 2600, 1000, "plain"), (640, 528, 257, "plain"),
    (16, 16, 1, "swiglu"), (1024, 2048, 4, "swiglu"), (4000, 2512, 9, "swiglu"),
    (512, 208, 64, "swiglu"), (4096, 1040, 100, "swiglu"), (1024, 1152, 600, "swiglu"),
    (4096, 12288, 17, "swiglu"),
    (16, 16, 1, "eight"), (1024, 2048, 4, "eight"), (4000, 2512, 9, "eight"),
    (512, 208, 64, "eight"), (4096, 1040, 100, "eight"), (1024, 1152, 600, "eight"),
    (2048, 4096, 300, "eight"), (400, 16, 700, "eight"),
]


def _weights(gen, n, k):
    codes = torch.randn(n, k, generator=gen).mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.rand(-(-n // 128), -(-k // 128), generator=gen) * 2e-3 + 1e-5
    scales[0, 0] = 0  # a block of zeros' scale may be anything
    return codes, scales


def _rows(gen, m, k):
    x = torch.randn(m, k, generator=gen) * torch.exp(torch.randn(k, generator=gen))
    return (x * torch.exp(2 * torch.randn(m, 1, generator=gen)) * 0.1).to(torch.bfloat16)


def _reference(x, codes, scales, epilogue, n):
    """The outputs in 64 bits of rows x (64 bits), and how far the kernels' sums may be off.
    The matrix unit adds the products of 8 neighbouring inputs as multiples of 2^(e - 13), e
    the largest sum of two exponents among them: each of the 8 loses less than 2^-13 of the
    largest product. Over the K / 8 groups these largest products come to at most
    sqrt(K / 8 sum p^2) (Cauchy and Schwarz). Beyond that, 16 groups a block are added in 32
    bits and the blocks' sums scaled and added (each taken as truncating, 2^-23), some more
    for the parts that are joined."""
    w = ref.weight(codes, scales)
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    square = x.square() @ w.square().t()
    tol = size * (128 + 2 * (codes.shape[1] // 128) + 32) * 2.0 ** -23 \
        + 2.0 ** -10 * torch.sqrt(square * (codes.shape[1] / 8))
    if epilogue != "plain":
        g, u = y[:, :n], y[:, n:]
        act = torch.nn.functional.silu(g)
        y = act * u
        # silu's slope is below 1.1; its exponential and quotient are good to 2^-18 here
        tol = 1.1 * tol[:, :n] * (u.abs() + tol[:, n:]) + act.abs() * tol[:, n:] \
            + 2.0 ** -18 * y.abs()
    return y, tol


def _same(a, b):
    if isinstance(a, torch.Tensor):
        return torch.equal(a.view(torch.int16), b.view(torch.int16))
    return torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and \
        torch.equal(a.scales.view(torch.uint8), b.scales.view(torch.uint8))


@pytest.mark.parametrize("case", _CASES, ids=lambda c: "-".join(map(str, c)))
def test_linear_fp8(hv, cuda, case):
    k, n, rows, epilogue = case
    print("fp8 linear", case, flush=True)
    ops, gate = hv.ops, epilogue != "plain"
    gen = torch.Generator().manual_seed(k + n + rows)
    codes, scales = _weights(gen, 2 * n if gate else n, k)
    w = ops.pack_fp8(codes.to(cuda), scales.to(cuda))
    x = _rows(gen, rows, k)
    xc, xs = ref.rows(x)
    y, tol = _reference(ref.values(xc, xs), codes, scales, epilogue, n)
    how = dict(swiglu=gate, quantize=epilogue == "eight")
    f8 = xc.float().to(torch.float8_e4m3fn).to(cuda)
    e8 = xs.float().to(torch.float8_e8m0fnu).to(cuda)
    got = [ops.linear_fp8(ops.Fp8Rows(f8, e8), w, **how), ops.linear_fp8(x.to(cuda), w, **how)]
    # codes and scales as slices of wider ones whose other bytes are NaN, aligned and not
    for at, st in ((16, 4), (5, 3)):
        cw = torch.full((rows, k + 32), 0x7f, dtype=torch.uint8, device=cuda)
        sw = torch.full((rows, -(-xs.shape[1] // 4) * 4 + 8), 255, dtype=torch.uint8, device=cuda)
        cw[:, at:at + k] = f8.view(torch.uint8)
        sw[:, st:st + xs.shape[1]] = e8.view(torch.uint8)
        got.append(ops.linear_fp8(ops.Fp8Rows(
            cw.view(torch.float8_e4m3fn)[:, at:at + k],
            sw.view(torch.float8_e8m0fnu)[:, st:st + xs.shape[1]]), w, **how))
    for at in (8, 3):  # bf16 rows
        xw = torch.full((rows, k + 24), float("nan"), dtype=torch.bfloat16, device=cuda)
        xw[:, at:at + k] = x.to(cuda)
        got.append(ops.linear_fp8(xw[:, at:at + k], w, **how))
    if epilogue != "eight":
        yw = torch.full((rows + 1, n + 5), 7.0, dtype=torch.bfloat16, device=cuda)
        ops.linear_fp8(ops.Fp8Rows(f8, e8), w, out=yw[:rows, 3:3 + n], **how)
        got.append(yw[:rows, 3:3 + n])
        assert bool((yw[rows] == 7).all() and (yw[:, :3] == 7).all())
        assert bool((yw[:, 3 + n:] == 7).all())
    for t in got:
        assert _same(t, got[0])
    if epilogue == "eight":
        ref.check_rows(got[0].codes, got[0].scales, y, tol)
    else:
        err, tol = (got[0].double().cpu() - y).abs(), tol + 2.0 ** -8 * (y.abs() + tol)
        assert bool((err <= tol).all()), float((err / tol).max())
        # by norm: bf16's rounding, evenly spread over half a step of 2^-8 at most, and the
        # products' cuts, independent of each other, with 8 to a group: together below 2^-8
        assert float(err.norm()) <= 2.0 ** -8 * float(y.norm())


@pytest.mark.parametrize("rows", [2, 16, 40, 300])
def test_rows_do_not_meet(hv, cuda, rows):
    """A row that holds a NaN or an infinity gives NaN, and leaves the others as they are."""
    gen = torch.Generator().manual_seed(rows)
    codes, scales = _weights(gen, 100, 512)
    w = hv.ops.pack_fp8(codes.to(cuda), scales.abs().clamp(min=1e-3).to(cuda))
    x = torch.randn(rows, 512, generator=gen).to(torch.bfloat16).to(cuda)
    want = hv.ops.linear_fp8(x, w)
    bad = x.clone()
    bad[1, 77] = float("nan")
    bad[rows - 1, 500] = float("inf")
    got = hv.ops.linear_fp8(bad, w)
    rest = [r for r in range(rows) if r not in (1, rows - 1)]
    assert torch.equal(got[rest], want[rest])
    assert bool(got[[1, rows - 1]].isnan().all())


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_rows_of_any_size(hv, cuda, rows):
    """Scales from 2^-100 to 2^100 in one row: the blocks' sums keep their own size."""
    gen = torch.Generator().manual_seed(rows)
    codes, scales = _weights(gen, 64, 640)
    w = hv.ops.pack_fp8(codes.to(cuda), scales.to(cuda))
    xc = torch.randn(rows, 640, generator=gen).mul(100).clamp(-448, 448).to(torch.float8_e4m3fn)
    e = torch.tensor([-100, -50, 0, 50, 100])[torch.rand(rows, 5, generator=gen).argsort(1)]
    xs = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    y, tol = _reference(ref.values(xc, xs), codes, scales, "plain", 64)
    got = hv.ops.linear_fp8(hv.ops.Fp8Rows(xc.to(cuda), xs.to(cuda)), w).double().cpu()
    assert bool(((got - y).abs() <= tol + 2.0 ** -8 * (y.abs() + tol)).all())


@pytest.mark.parametrize("rows", [3, 40, 200, 1100])
def test_scales_at_their_ends(hv, cuda, rows):
    """A scale that is NaN (byte 255) makes its row NaN and no other; the least ones (bytes 0
    and 1) stand for less than 2^-100 here; bytes behind a row's last scale are not read as
    scales. (640 inputs are five scales, kept in eight bytes.)"""
    gen = torch.Generator().manual_seed(rows)
    codes, scales = _weights(gen, 200, 640)
    w = hv.ops.pack_fp8(codes.to(cuda), scales.to(cuda))
    xc = torch.randn(rows, 640, generator=gen).mul(100).clamp(-448, 448).to(torch.float8_e4m3fn)
    e = torch.full((rows, 8), 255, dtype=torch.uint8)
    e[:, :5] = 120 + torch.randint(0, 9, (rows, 5), generator=gen).to(torch.uint8)

    def run():
        es = e.to(cuda).view(torch.float8_e8m0fnu)[:, :5]
        return hv.ops.linear_fp8(hv.ops.Fp8Rows(xc.to(cuda), es), w)

    want = run()
    assert bool(torch.isfinite(want).all())
    e[1, 4] = 255
    e[rows - 1, 0] = 255
    e[0, :5] = torch.tensor([0, 1, 0, 1, 0], dtype=torch.uint8)
    got = run()
    assert bool(got[[1, rows - 1]].isnan().all())
    assert bool((got[0].abs() < 2.0 ** -100).all())
    rest = [r for r in range(2, rows - 1)]
    assert torch.equal(got[rest], want[rest])


def test_one_row_of_many_sizes(hv, cuda):
    """A row's result is the same in every batch that one kernel serves, and near itself in all
    (the sums' order differs): the first rows of batches around the kernels' limits."""
    gen = torch.Generator().manual_seed(77)
    codes, scales = _weights(gen, 528, 1040)
    w = hv.ops.pack_fp8(codes.to(cuda), scales.to(cuda))
    x = _rows(gen, 2100, 1040)
    rows = hv.ops.quantize_rows_fp8(x.to(cuda))
    y, tol = _reference(ref.values(*ref.rows(x[:1])), codes, scales, "plain", 528)
    for m in (1, 8, 9, 16, 17, 32, 33, 64, 65, 127, 129, 256, 300, 512, 513, 1024, 2100):
        part = hv.ops.Fp8Rows(rows.codes[:m], rows.scales[:m])
        got = hv.ops.linear_fp8(part, w)
        assert bool(((got[:1].double().cpu() - y).abs() <= tol + 2.0 ** -8 * (y.abs() + tol)).all())
        assert bool(torch.isfinite(got).all()), m


def test_quantize_fp8(hv, cuda):
    """The product is that of the weight the codes stand for, at most half a step off."""
    gen = torch.Generator().manual_seed(5)
    weight = torch.randn(300, 256, generator=gen)
    w = hv.ops.quantize_fp8(weight.to(cuda))
    eye = torch.eye(256, dtype=torch.bfloat16, device=cuda)
    back = hv.ops.linear_fp8(eye, w).t().double().cpu()  # one product each: exact to bf16
    s = hv.ops.quantize_fp8(weight).scales.double().repeat_interleave(16, 0)[:300]
    half = torch.maximum(weight.abs().double() * 2.0 ** -4, s.repeat_interleave(128, 1) * 2.0 ** -10)
    assert bool(((back - weight.double()).abs() <= half * 1.001 + back.abs() * 2.0 ** -8).all())


def test_captured_calls_share_nothing(hv, cuda):
    """Graphs of projections replayed in turn, with eager calls between, on two streams."""
    gen = torch.Generator().manual_seed(9)
    codes, scales = _weights(gen, 512, 2048)
    w = hv.ops.pack_fp8(codes.to(cuda), scales.to(cuda))
    calls = [(_rows(gen, r, 2048).to(cuda), dict(swiglu=g, quantize=q))
             for r, g, q in ((3, True, True), (40, False, False), (64, True, True),
                             (300, False, False))]
    want = [hv.ops.linear_fp8(x, w, **how) for x, how in calls]
    graphs = []
    for x, how in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = hv.ops.linear_fp8(x, w, **how)
        graphs.append((g, y))
    side = torch.cuda.Stream()
    for _ in range(3):
        for g, y in graphs:
            (y if isinstance(y, torch.Tensor) else y.codes.view(torch.uint8)).zero_()
        side.wait_stream(torch.cuda.current_stream())
        for g, _ in graphs[:2]:
            g.replay()
        with torch.cuda.stream(side):
            for g, _ in graphs[2:]:
                g.replay()
            beside = [hv.ops.linear_fp8(x, w, **how) for x, how in calls]
        eager = [hv.ops.linear_fp8(x, w, **how) for x, how in calls]
        torch.cuda.synchronize()
        for i in range(len(calls)):
            assert _same(graphs[i][1], want[i]) and _same(eager[i], want[i])
            assert _same(beside[i], want[i])


@pytest.mark.parametrize("rows,features", [(3, 256), (40, 256), (300, 4096), (1100, 2048),
                                           (2048, 4096)])
def test_swiglu_leaves_nonfinite_values_to_themselves(hv, cuda, rows, features):
    """silu(gate) * up = 2^57 * 2^57 but for one feature whose product overflows and one with
    a negative gate (silu(-2^57) is 0): the overflow is NaN and takes no part in the scale. A
    row with a NaN is NaN, with the least scale."""
    ops = hv.ops
    codes = torch.ones(2 * features, 128)
    codes[5] = codes[features + 5] = 448.0
    codes[7] = -1
    w = ops.pack_fp8(codes.to(torch.float8_e4m3fn).to(cuda),
                     torch.ones(features // 64, 1, device=cuda))
    xc = torch.ones(rows, 128)
    xc[1, 99] = float("nan")
    e = torch.full((rows, 4), 127 + 50, dtype=torch.uint8, device=cuda)
    x = ops.Fp8Rows(xc.to(torch.float8_e4m3fn).to(cuda), e.view(torch.float8_e8m0fnu)[:, :1])
    got = ops.linear_fp8(x, w, swiglu=True, quantize=True)
    c, s = got.codes.float().cpu(), got.scales.float().cpu()
    rest = [r for r in range(rows) if r != 1]
    assert bool(c[1].isnan().all()) and bool((s[1] == 2.0 ** -126).all())
    assert bool((s[rest] == 2.0 ** 106).all())  # 2^114 <= 448 * 2^106
    assert bool(c[rest, 5].isnan().all()) and bool((c[rest, 7] == 0).all())
    assert bool((c[rest][:, [j for j in range(features) if j not in (5, 7)]] == 256).all())


def _units(gen, n, k, cuda):
    """-1, 0 and 1, whose products are summed without rounding."""
    return torch.randint(-1, 2, (n, k), generator=gen).to(torch.float8_e4m3fn).to(cuda)


def _rows_of_one(codes):
    steps = -(-codes.shape[1] // 128)
    e = torch.full((codes.shape[0], -(-steps // 4) * 4), 127, dtype=torch.uint8,
                   device=codes.device)
    return e.view(torch.float8_e8m0fnu)[:, :steps]


def _exact(x, w):
    return (x.cpu().double() @ w.cpu().double().t()).to(torch.bfloat16)


@pytest.mark.parametrize("k,n", [(4352, 16), (16, 2064)])
def test_offsets_past_32_bits_of_rows(hv, cuda, k, n):
    """2^20 rows: codes or outputs of more than 2^32 bytes."""
    ops, gen, rows = hv.ops, torch.Generator().manual_seed(k), 1 << 20
    codes = _units(gen, n, k, cuda)
    w = ops.pack_fp8(codes, torch.ones(-(-n // 128), -(-k // 128), device=cuda))
    last = _units(gen, 40, k, cuda)
    x = torch.zeros(rows, k, dtype=torch.float8_e4m3fn, device=cuda)
    x[-40:] = last
    got = ops.linear_fp8(ops.Fp8Rows(x, _rows_of_one(x)), w)
    assert torch.equal(got[-40:].cpu(), _exact(last, codes))
    assert not bool(got[:-40].any())


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_offsets_past_32_bits_of_weights(hv, cuda, rows):
    ops, gen, k, n = hv.ops, torch.Generator().manual_seed(rows), 4352, 1 << 20
    codes = _units(gen, 48, k, cuda)
    tail = ops.pack_fp8(codes, torch.ones(1, 34, device=cuda))
    packed = torch.zeros(n // 16, 34, 2, 64, 16, dtype=torch.uint8, device=cuda)
    packed[-3:] = tail.packed
    w = ops.Fp8Weight(packed, torch.ones(n // 16, 34, device=cuda), n, k)
    x = _units(gen, rows, k, cuda)
    got = ops.linear_fp8(ops.Fp8Rows(x, _rows_of_one(x)), w)
    assert torch.equal(got[:, -48:].cpu(), _exact(x, codes))
    assert not bool(got[:, :-48].any())


def test_linear_refusals(hv, cuda):
    ops = hv.ops
    w = ops.quantize_fp8(torch.ones(40, 160, device=cuda))
    x = torch.zeros(3, 160, dtype=torch.bfloat16, device=cuda)
    rows = ops.quantize_rows_fp8(x)
    out = torch.zeros(3, 40, dtype=torch.bfloat16, device=cuda)
    for a, more in ((x.float(), {}), (x[0], {}), (x[:, :144], {}), (x, dict(quantize=True)),
                    (x, dict(swiglu=True)), (x, dict(out=out[:2])), (x, dict(out=out.float())),
                    (x.cpu(), {}), (ops.Fp8Rows(rows.codes, rows.scales[:, :1]), {}),
                    (ops.Fp8Rows(rows.codes[:, :144], rows.scales), {}),
                    (x, dict(swiglu=True, quantize=True, out=out))):
        with pytest.raises(ValueError):
            ops.linear_fp8(a, w, **more)
    with pytest.raises(ValueError):
        ops.linear_fp8(x, ops.Fp8Weight(w.packed, w.scales, 48 + 16, 160))
    for bad in (ops.Fp8Rows(rows.codes.float(), rows.scales),
                ops.Fp8Rows(rows.codes, rows.scales.float())):
        with pytest.raises(TypeError):
            ops.linear_fp8(bad, w)
    assert ops.linear_fp8(x[:0], w).shape == (0, 40)
