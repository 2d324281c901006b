"""Rows in 8 bits on the GPU against their definition in 64 bits."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu

_SIZES = [(1, 16), (3, 128), (2, 144), (5, 272), (1, 4096), (64, 4096), (333, 1056), (1021, 1024),
          (7, 5120), (4, 8192), (2, 16384), (130, 2048), (3, 40960)]
_ids = lambda c: "-".join(map(str, c))  # noqa: E731


def _x(gen, m, k):
    """Rows and channels of very different size, with groups of zeros."""
    x = torch.randn(m, k, generator=gen) * torch.exp(3 * torch.randn(k, generator=gen))
    x *= torch.exp(5 * torch.randn(m, 1, generator=gen))
    x[:, k // 2:k // 2 + 9] = 0
    if k >= 384:
        x[:, 128:256] = 0
    return x.to(torch.bfloat16)


def _views(x, device, fill=float("nan")):
    """x as it is, as a slice of wider rows, and off the 16-byte alignment."""
    m, k = x.shape
    out = [x.to(device)]
    for at in (8, 5):
        wide = torch.full((m, k + 24), fill, dtype=x.dtype, device=device)
        wide[:, at:at + k] = x.to(device)
        out.append(wide[:, at:at + k])
    return out


def _same(rows, codes, scales):
    got = rows.codes.double().cpu()
    assert torch.equal(got.isnan(), codes.isnan())
    assert torch.equal(got.nan_to_num(nan=1e9), codes.nan_to_num(nan=1e9))
    assert torch.equal(rows.scales.double().cpu(), scales)


@pytest.mark.parametrize("size", _SIZES, ids=_ids)
def test_quantize_rows(hv, cuda, size):
    print("quantize rows", size, flush=True)
    x = _x(torch.Generator().manual_seed(size[1]), *size)
    codes, scales = ref.rows(x)
    for view in _views(x, cuda) + [x.t().contiguous().to(cuda).t()]:
        got = hv.ops.quantize_rows_fp8(view)
        assert got.codes.dtype == torch.float8_e4m3fn and got.codes.shape == size
        assert got.scales.dtype == torch.float8_e8m0fnu
        _same(got, codes, scales)


def test_quantize_every_bf16_value(hv, cuda):
    """Every bf16 number, in groups of neighbours (subnormals, NaN and infinities among
    them), and the amax on both sides of a scale's border."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = x.view(-1, 256)
    _same(hv.ops.quantize_rows_fp8(x.to(cuda)), *ref.rows(x))
    x = torch.zeros(6, 128, dtype=torch.bfloat16)
    x[:, 3] = torch.tensor([448.0, 450.0, -448.0, 446.0, -450.0, 1.75])
    x[:, 4] = 0.3
    _same(hv.ops.quantize_rows_fp8(x.to(cuda)), *ref.rows(x))


@pytest.mark.parametrize("rows", [1, 70])
def test_quantize_leaves_nonfinite_values_to_themselves(hv, cuda, rows):
    x = torch.randn(rows, 400, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    for at, v in ((0, "nan"), (130, "inf"), (131, "-inf"), (399, "nan")):
        x[rows // 2, at] = float(v)
    x[0, 256:384] = float("inf")  # nothing finite: the least scale
    _same(hv.ops.quantize_rows_fp8(x.to(cuda)), *ref.rows(x))


def _norm(x, res, w, eps):
    """The rows in 64 bits and how far fp32 may be off: the sum h (2^-24), its squares (2^-24
    each) and their sum (below 64 + H / 64 additions one after the other, 2^-24 each), half of
    that behind the root, the root, its quotient and two products (2^-22 together)."""
    h = x.double() + (0 if res is None else res.double())
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * w.double()
    return h, y, y.abs() * ((64 + x.shape[1] / 64) * 2.0 ** -25 + 2.0 ** -21)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("size", _SIZES, ids=_ids)
def test_rmsnorm_fp8(hv, cuda, size, residual):
    print("norm", size, residual, flush=True)
    m, k = size
    gen = torch.Generator().manual_seed(k + 7)
    x = (torch.randn(m, k, generator=gen) * torch.exp(torch.randn(m, 1, generator=gen) * 2)
         ).to(torch.bfloat16)
    r = torch.randn(m, k, generator=gen).mul(20).to(torch.bfloat16) if residual else None
    w = (torch.rand(k, generator=gen) * 3 - 1).to(torch.bfloat16)
    h, y, tol = _norm(x, r, w, 1e-6)
    first = None
    for view, weight in zip(_views(x, cuda), _views(w[None], cuda)):
        for res in _views(r, cuda, 7.0) if residual else [None]:
            got = hv.ops.rmsnorm_fp8(view, weight[0], 1e-6, residual=res)
            ref.check_rows(got.codes, got.scales, y, tol)
            first = first or got
            assert torch.equal(got.codes.view(torch.uint8), first.codes.view(torch.uint8))
            assert torch.equal(got.scales.view(torch.uint8), first.scales.view(torch.uint8))
            if residual:
                assert torch.equal(res.cpu(), h.float().to(torch.bfloat16))
                if res._base is not None:
                    wide, at = res._base, res.storage_offset()
                    assert bool((wide[:, :at] == 7).all() and (wide[:, at + k:] == 7).all())


def test_rmsnorm_fp8_of_its_own_residual(hv, cuda):
    """x and the residual the same rows: h = 2 x, in place."""
    x = torch.randn(9, 1040, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16)
    w = torch.ones(1040, dtype=torch.bfloat16)
    h, y, tol = _norm(x, x, w, 1e-6)
    both = x.to(cuda)
    got = hv.ops.rmsnorm_fp8(both, w.to(cuda), 1e-6, residual=both)
    ref.check_rows(got.codes, got.scales, y, tol)
    assert torch.equal(both.cpu(), (2 * x.float()).to(torch.bfloat16))


def test_rmsnorm_fp8_limits(hv, cuda):
    """Rows of zeros, one that holds a NaN and one with an infinity: the others stay."""
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(5, 512, generator=gen).to(torch.bfloat16)
    w = torch.ones(512, dtype=torch.bfloat16, device=cuda)
    want = hv.ops.rmsnorm_fp8(x.to(cuda), w, 1e-6)
    bad = x.clone()
    bad[1] = 0
    bad[2, 77] = float("nan")
    bad[3, 500] = float("inf")
    got = hv.ops.rmsnorm_fp8(bad.to(cuda), w, 1e-6)
    for i in (0, 4):
        assert torch.equal(got.codes[i].view(torch.uint8), want.codes[i].view(torch.uint8))
    assert bool((got.codes[1].float() == 0).all())
    assert bool((got.scales[1].float() == 2.0 ** -126).all())
    assert bool(got.codes[2].float().isnan().all())
    assert bool(got.codes[3, 500].float().isnan())


def test_offsets_past_32_bits(hv, cuda):
    """2^20 rows of 4112: more than 2^32 codes, and 2^33 bytes of bf16."""
    gen = torch.Generator().manual_seed(6)
    x = torch.zeros(1 << 20, 4112, dtype=torch.bfloat16, device=cuda)
    last = torch.randn(30, 4112, generator=gen).to(torch.bfloat16).to(cuda)
    x[-30:] = last
    w = torch.ones(4112, dtype=torch.bfloat16, device=cuda)
    res = x.clone()
    for got, want in ((hv.ops.quantize_rows_fp8(x), hv.ops.quantize_rows_fp8(last)),
                      (hv.ops.rmsnorm_fp8(x, w, 1e-6, residual=res),
                       hv.ops.rmsnorm_fp8(last, w, 1e-6, residual=last.clone()))):
        for a, b in zip(got, want):
            assert torch.equal(a[-30:].view(torch.uint8), b.view(torch.uint8))
        assert not bool(got.codes[:-30].view(torch.uint8).any())
        assert bool((got.scales[:-30].view(torch.uint8) == 1).all())
    assert torch.equal(res[-30:], last + last) and not bool(res[:-30].any())


def test_rows_refusals(hv, cuda):
    ops = hv.ops
    x = torch.zeros(3, 160, dtype=torch.bfloat16, device=cuda)
    w = torch.ones(160, dtype=torch.bfloat16, device=cuda)
    for bad in (x[:, :150], x[0], x.float(), x[:, :0]):
        with pytest.raises(ValueError):
            ops.quantize_rows_fp8(bad)
        with pytest.raises(ValueError):
            ops.rmsnorm_fp8(bad, w, 1e-6)
    for weight, res in ((w[:144], None), (w.float(), None), (w, x[:2]), (w, x.float()),
                        (w, x[:1].expand(3, 160)), (w, x.cpu())):
        with pytest.raises(ValueError):
            ops.rmsnorm_fp8(x, weight, 1e-6, residual=res)
    for rows in (ops.quantize_rows_fp8(x[:0]), ops.rmsnorm_fp8(x[:0], w, 1e-6)):
        assert rows.codes.shape == (0, 160) and rows.scales.shape == (0, 2)
