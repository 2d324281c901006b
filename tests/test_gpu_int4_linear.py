"""Projections with 4-bit weights on the GPU against the same sums in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# inputs, features, group, rows, swiglu
_CASES = [
    (32, 1, 32, 1, False), (128, 16, 128, 2, False), (96, 17, 32, 5, False),
    (352, 200, 32, 16, False), (1056, 1001, 32, 3, False), (1024, 4096, 64, 7, False),
    (4096, 6144, 128, 4, False), (4096, 20000, 128, 1, False), (12288, 4096, 64, 16, False),
    (1024, 1001, 64, 17, False), (96, 40, 32, 33, False), (4096, 4096, 128, 63, False),
    (12288, 1024, 64, 64, False), (384, 777, 128, 65, False), (2048, 512, 32, 300, False),
    (128, 16, 128, 130, False), (160, 130000, 32, 20, False),
    (32, 16, 32, 1, True), (1024, 2048, 128, 4, True), (4000, 2512, 32, 9, True),
    (512, 208, 64, 64, True), (4096, 1040, 64, 100, True),
]


def _weights(gen, n, k, group):
    codes = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.uint8)
    scales = (torch.rand(n, k // group, generator=gen) * 0.02 + 0.001).to(torch.bfloat16)
    return codes, scales


def _reference(x, codes, scales, group):
    """Sums in 64 bits, and sum |x| s: the size that the sums' roundings go by."""
    s = scales.double().repeat_interleave(group, 1)
    return x.double() @ ((codes.double() - 8) * s).t(), x.double().abs() @ s.t()


def _tolerance(size, k, group):
    """Every group's sum starts at -24 sum x and adds x (16 + c), c <= 15: its partial sums
    stay below 55 sum |x|, over at most 2 group additions of 32 bits (taken as truncating,
    2^-23 each); then the groups' results, each below 55 sum |x| s again, are scaled and
    added."""
    return size * 55 * (2 * group + k // group + 16) * 2.0 ** -23


@pytest.mark.parametrize("case", _CASES, ids=["-".join(map(str, c)) for c in _CASES])
def test_linear_int4(hv, cuda, case):
    k, n, group, rows, swiglu = case
    print("int4 linear", case, flush=True)
    gen = torch.Generator().manual_seed(k + n + rows)
    codes, scales = _weights(gen, 2 * n if swiglu else n, k, group)
    x = (torch.randn(rows, k, generator=gen) * torch.exp(torch.randn(k, generator=gen))
         ).to(torch.bfloat16)
    w = hv.ops.pack_int4(codes.to(cuda), scales.to(cuda))
    y, size = _reference(x, codes, scales, group)
    tol = _tolerance(size, k, group)
    if swiglu:
        g, u = y[:, :n], y[:, n:]
        y = torch.nn.functional.silu(g) * u
        # silu's slope is below 1.1; its exponential and quotient are good to 2^-18 here
        act = torch.nn.functional.silu(g).abs()
        tol = 1.1 * tol[:, :n] * (u.abs() + tol[:, n:]) + act * tol[:, n:] + 2.0 ** -18 * y.abs()
    tol = tol + 2.0 ** -8 * y.abs()
    # rows and outputs as slices of wider ones, and a row of x off the 16-byte alignment
    xw = torch.full((rows, k + 24), float("nan"), dtype=torch.bfloat16, device=cuda)
    xw[:, 8:8 + k] = x.to(cuda)
    yw = torch.full((rows + 1, n + 5), 7.0, dtype=torch.bfloat16, device=cuda)
    got = [hv.ops.linear_int4(x.to(cuda), w, swiglu=swiglu)]
    hv.ops.linear_int4(xw[:, 8:8 + k], w, swiglu=swiglu, out=yw[:rows, 3:3 + n])
    got.append(yw[:rows, 3:3 + n])
    xw[:, 5:5 + k] = x.to(cuda)
    got.append(hv.ops.linear_int4(xw[:, 5:5 + k], w, swiglu=swiglu))
    for t in got:
        err = (t.double().cpu() - y).abs()
        assert bool((err <= tol).all()), float((err / tol).max())
        assert torch.equal(t, got[0])
    assert bool((yw[rows] == 7).all() and (yw[:, :3] == 7).all() and (yw[:, 3 + n:] == 7).all())


@pytest.mark.parametrize("rows", [2, 16, 40])
def test_rows_do_not_meet(hv, cuda, rows):
    """A row that holds a NaN or an infinity gives NaN, and leaves the others as they are."""
    gen = torch.Generator().manual_seed(rows)
    codes, scales = _weights(gen, 100, 512, 128)
    w = hv.ops.pack_int4(codes.to(cuda), scales.to(cuda))
    x = torch.randn(rows, 512, generator=gen).to(torch.bfloat16).to(cuda)
    want = hv.ops.linear_int4(x, w)
    bad = x.clone()
    bad[1, 77] = float("nan")
    bad[rows - 1, 500] = float("inf")
    got = hv.ops.linear_int4(bad, w)
    rest = [r for r in range(rows) if r not in (1, rows - 1)]
    assert torch.equal(got[rest], want[rest])
    assert bool(got[[1, rows - 1]].isnan().all())


def test_quantize_int4(hv, cuda):
    """Codes are the nearest ones: the weight is at most half a scale off, and the product
    is that of the weight the codes stand for."""
    gen = torch.Generator().manual_seed(5)
    weight = torch.randn(48, 256, generator=gen)
    weight[3, :64] = 0
    w = hv.ops.quantize_int4(weight.to(cuda), 64)
    assert (w.out_features, w.in_features, w.group) == (48, 256, 64)
    eye = torch.eye(256, dtype=torch.bfloat16, device=cuda)
    back = hv.ops.linear_int4(eye, w).t().double().cpu()  # one product each: exact to bf16
    s = (weight.view(48, 4, 64).abs().amax(-1) / 7).to(torch.bfloat16).double()
    off = (back - weight.double()).abs()
    # 7 s is below the largest value by up to half a bf16 step of it
    most = 0.5 * s + 7 * s * 2.0 ** -8
    assert bool((off <= most.repeat_interleave(64, 1) + back.abs() * 2.0 ** -8).all())
    assert bool((back[3, :64] == 0).all())


def test_captured_calls_share_nothing(hv, cuda):
    """Graphs of split projections replayed in turn, with eager calls between."""
    gen = torch.Generator().manual_seed(9)
    codes, scales = _weights(gen, 512, 2048, 64)
    w = hv.ops.pack_int4(codes.to(cuda), scales.to(cuda))
    xs = [torch.randn(r, 2048, generator=gen).to(torch.bfloat16).to(cuda) for r in (40, 64)]
    want = [hv.ops.linear_int4(x, w) for x in xs]
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = hv.ops.linear_int4(x, w)
        graphs.append((g, y))
    for _ in range(3):
        for g, y in graphs:
            y.zero_()
            g.replay()
        eager = [hv.ops.linear_int4(x, w) for x in xs]
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(graphs[i][1], want[i]) and torch.equal(eager[i], want[i])


@pytest.mark.parametrize("case", [(12288, 4100, 64, 40, False), (4000, 5200, 32, 33, True),
                                  (1056, 30000, 32, 20, False), (4096, 8208, 128, 64, True)],
                         ids=lambda c: "-".join(map(str, c)))
def test_linear_int4_many_steps(hv, cuda, case):
    """Enough steps that a workgroup's two sets of waves share them: split and not, odd
    numbers of steps."""
    test_linear_int4(hv, cuda, case)
