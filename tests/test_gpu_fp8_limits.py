"""Projections of rows in 8 bits at the ends of the number range, in every kernel that serves
them (the sizes reach them in turn), against the same sums in 64 bits."""
import pytest
import torch

import fp8_ref as ref
from test_gpu_fp8_linear import _reference

pytestmark = pytest.mark.gpu

# inputs, features, rows, epilogue
_SIZES = [
    (1040, 200, 9, "plain"), (1040, 200, 300, "plain"), (2048, 512, 300, "plain"),
    (1040, 1040, 300, "plain"), (1040, 4096, 300, "plain"), (1040, 4096, 600, "plain"),
    (1040, 4096, 1100, "plain"), (1040, 6144, 2048, "plain"), (12288, 4096, 64, "plain"),
    (1040, 208, 9, "swiglu"), (1040, 1040, 300, "swiglu"), (1040, 4096, 300, "swiglu"),
    (1040, 4096, 600, "swiglu"), (1040, 4096, 1100, "swiglu"), (4096, 1024, 128, "swiglu"),
    (12288, 1024, 128, "swiglu"),
    (1040, 208, 9, "eight"), (1040, 1040, 300, "eight"), (1040, 4096, 300, "eight"),
    (1040, 4096, 1100, "eight"), (4096, 1040, 100, "eight"),
]
_ids = lambda c: "-".join(map(str, c))  # noqa: E731


def _codes(x):
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _near(got, y, tol, epilogue):
    if epilogue == "eight":
        ref.check_rows(got.codes, got.scales, y.cpu(), tol.cpu())
        return
    err, tol = (got.double() - y).abs(), tol + 2.0 ** -8 * (y.abs() + tol)
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("case", _SIZES, ids=_ids)
def test_inputs_up_to_the_largest(hv, cuda, case):
    """Inputs of bf16's largest values (and, in 8 bits, up to 448 * 2^120) with weights that
    bring their sums back into range: no sum on the way becomes an infinity, nor two of
    opposite signs NaN."""
    k, n, rows, epilogue = case
    print("largest inputs", case, flush=True)
    ops, gate = hv.ops, epilogue != "plain"
    gen = torch.Generator().manual_seed(k + n + rows)
    features = 2 * n if gate else n
    codes = torch.randn(features, k, generator=gen) * 100
    codes[0] = 448
    codes[1] = 448 * (1 - 2 * (torch.arange(k) % 2))
    scales = torch.rand(-(-features // 128), -(-k // 128), generator=gen) * 1e-8 + 1e-12
    if gate:
        codes[2:n:2] *= 2.0 ** -11  # gates of a few units, and of some thousands
        scales *= 1e-16
        scales[:-(-n // 128)] = scales[:-(-n // 128)] * 1e-14 + 2.0 ** -126
    codes = _codes(codes)
    w = ops.pack_fp8(codes.to(cuda), scales.to(cuda))
    most = torch.finfo(torch.bfloat16).max
    x = (torch.randn(rows, k, generator=gen).clamp(-1.9, 1.9).double() * 2.0 ** 127)
    x = x.float().to(torch.bfloat16)
    x[-1] = most
    xc, xs = ref.rows(x)
    y, tol = _reference(ref.values(xc, xs).to(cuda), codes.to(cuda), scales.to(cuda), epilogue, n)
    assert bool((y.abs() < 2.0 ** 127).all())
    how = dict(swiglu=gate, quantize=epilogue == "eight")
    _near(ops.linear_fp8(x.to(cuda), w, **how), y, tol, epilogue)
    xc, xs = xc.float(), torch.full_like(xs, 2.0 ** 120)
    xc[0] = 448
    y, tol = _reference(ref.values(xc, xs).to(cuda), codes.to(cuda), scales.to(cuda), epilogue, n)
    assert bool((y.abs() < 2.0 ** 127).all())
    f8 = ops.Fp8Rows(_codes(xc).to(cuda), xs.float().to(torch.float8_e8m0fnu).to(cuda))
    _near(ops.linear_fp8(f8, w, **how), y, tol, epilogue)


@pytest.mark.parametrize("case", [c for c in _SIZES if c[3] == "plain"], ids=_ids)
def test_inputs_down_to_the_least(hv, cuda, case):
    """Rows of the least scales with weights that bring their sums up: the 32 bits of a
    block's sum are multiples of 2^-132 there, taken as lost at each of the 128 additions."""
    k, n, rows, epilogue = case
    print("least inputs", case, flush=True)
    gen = torch.Generator().manual_seed(k + n + rows)
    codes = _codes(torch.randn(n, k, generator=gen) * 100)
    scales = torch.rand(-(-n // 128), -(-k // 128), generator=gen) * 2.0 ** 20
    w = hv.ops.pack_fp8(codes.to(cuda), scales.to(cuda))
    xc = torch.randn(rows, k, generator=gen)
    xc = _codes(xc * torch.exp2(torch.rand(rows, 1, generator=gen) * -12))
    xs = torch.randint(1, 12, (rows, -(-k // 128)), generator=gen).to(torch.uint8)
    xs = xs.view(torch.float8_e8m0fnu)
    y, tol = _reference(ref.values(xc, xs).to(cuda), codes.to(cuda), scales.to(cuda), epilogue, n)
    tol += (scales.double().sum(1) * 2.0 ** -125).repeat_interleave(128)[:n].to(cuda)
    got = hv.ops.linear_fp8(hv.ops.Fp8Rows(xc.to(cuda), xs.to(cuda)), w)
    _near(got, y, tol, epilogue)
    some = xc.float().abs().amax(1) > 0  # (the smallest rows' codes may all be zeros)
    assert bool((got.abs().amax(1) > 0).cpu()[some].all()) and int(some.sum()) > rows // 4


@pytest.mark.parametrize("rows,features,quantize", [
    (3, 256, False), (300, 4096, False), (1100, 4096, False), (2100, 4096, False),
    (3, 256, True), (300, 1024, True), (300, 4096, True), (1100, 4096, True)])
def test_silu_of_far_gates(hv, cuda, rows, features, quantize):
    """Gates from -80 to -88.7, whose exponential is near f32's largest value, times 2^120.
    The exponent's argument is rounded to 2^-17 there (128 by 2^-24), its quotient to 2^-22."""
    ops = hv.ops
    j = torch.arange(features)
    gate = torch.zeros(features, 128)
    gate[:, 0], gate[:, 1], gate[:, 2] = -80, -(j % 9), -(j // 9 % 6) / 8
    gate[:, 2] = torch.where(j % 9 == 8, gate[:, 2], gate[:, 2] * 1.5)
    up = torch.zeros(features, 128)
    up[:, 0] = 1
    scales = torch.ones(features // 64, 1)
    scales[features // 128:] = 2.0 ** 120
    w = ops.pack_fp8(_codes(torch.cat([gate, up])).to(cuda), scales.to(cuda))
    x = torch.zeros(rows, 128, dtype=torch.bfloat16, device=cuda)
    x[:, :3] = 1
    got = ops.linear_fp8(x, w, swiglu=True, quantize=quantize)
    g = gate.double().sum(1)
    y = (g * torch.sigmoid(g) * 2.0 ** 120)[None].expand(rows, features)
    assert float(g.min()) < -88.5
    epilogue = "eight" if quantize else "swiglu"
    _near(got if quantize else got.cpu(), y, y.abs() * 2.0 ** -16, epilogue)


def test_a_single_row_of_any_stride(hv, cuda):
    """One row's stride says nothing: an output whose rows would overlap if there were more."""
    gen = torch.Generator().manual_seed(1)
    w = hv.ops.quantize_fp8(torch.randn(200, 256, generator=gen).to(cuda))
    x = torch.randn(1, 256, generator=gen).to(torch.bfloat16).to(cuda)
    want = hv.ops.linear_fp8(x, w)
    for out in (torch.empty(200, dtype=torch.bfloat16, device=cuda)[:, None].t(),
                torch.empty(200, dtype=torch.bfloat16, device=cuda).as_strided((1, 200), (0, 1))):
        assert hv.ops.linear_fp8(x, w, out=out) is out and torch.equal(out, want)
    two = torch.empty(400, dtype=torch.bfloat16, device=cuda).as_strided((2, 200), (100, 1))
    with pytest.raises(RuntimeError):  # rows that do overlap
        hv.ops.linear_fp8(x.expand(2, 256), w, out=two)
