"""The 8-bit floating-point path on the host: the weight's layout and the refusals."""
import ctypes

import pytest
import torch

import fp8_ref as ref


def _unpack(w):
    """Codes and block scales back from the layout, by its definition."""
    tiles, steps = w.packed.shape[:2]
    codes = torch.zeros(tiles * 16, steps * 128, dtype=torch.uint8)
    for lane in range(64):
        for h in range(2):
            for j in range(16):
                k = 64 * h + 16 * (lane // 16) + j
                codes.view(tiles, 16, steps, 128)[:, lane % 16, :, k] = w.packed[:, :, h, lane, j]
    return codes, w.scales


@pytest.mark.parametrize("n,k", [(16, 128), (1, 16), (37, 352), (300, 144), (128, 256)])
def test_layout(hv, n, k):
    gen = torch.Generator().manual_seed(n)
    codes = torch.randint(0, 127, (n, k), generator=gen, dtype=torch.uint8)
    scales = torch.rand(-(-n // 128), -(-k // 128), generator=gen)
    w = hv.ops.pack_fp8(codes.view(torch.float8_e4m3fn), scales)
    assert (w.out_features, w.in_features) == (n, k)
    c, s = _unpack(w)
    assert torch.equal(c[:n, :k], codes)
    assert bool((c[n:] == 0).all() and (c[:, k:] == 0).all())
    for t in range(s.shape[0]):
        assert torch.equal(s[t], scales[t * 16 // 128])


def test_quantize_takes_the_nearest_code(hv):
    gen = torch.Generator().manual_seed(2)
    weight = torch.randn(200, 272, generator=gen) * 3
    weight[:128, :128] = 0
    weight[150, 130] = -1000
    w = hv.ops.quantize_fp8(weight)
    c, s = _unpack(w)
    c = c.view(torch.float8_e4m3fn).double()[:200, :272]
    s = s.double().repeat_interleave(16, 0).repeat_interleave(128, 1)[:200, :272]
    off = (c * s - weight.double()).abs()
    # half a step of the code, and the quotient's rounding
    step = torch.maximum(weight.double().abs() * 2.0 ** -4, s * 2.0 ** -10)
    assert bool((off <= step + weight.double().abs() * 2.0 ** -22).all())
    assert bool((c[:128, :128] == 0).all()) and bool(torch.isfinite(s).all())


def test_the_reference_knows_e4m3():
    """The oracle's rounding against torch's own conversion, over every bf16 value."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    x = x[(x.abs() <= 448) | ~torch.isfinite(x)]
    assert torch.equal(ref.e4m3(x.double()).nan_to_num(nan=1e9),
                       x.to(torch.float8_e4m3fn).double().nan_to_num(nan=1e9))


def test_arguments_are_checked(hv):
    ops = hv.ops
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    codes, scales = torch.zeros(40, 160).to(f8), torch.ones(1, 2)
    w = ops.pack_fp8(codes, scales)
    for c, s, err in ((codes.float(), scales, TypeError), (codes, scales.bfloat16(), TypeError),
                      (codes, torch.ones(2, 2), ValueError), (codes, torch.ones(1, 1), ValueError),
                      (codes[:, :150], scales, ValueError), (codes[0], scales, ValueError),
                      (codes[:0], torch.ones(0, 2), ValueError)):
        with pytest.raises(err):
            ops.pack_fp8(c, s)
    for bad in (torch.zeros(4, 60), torch.zeros(64), torch.zeros(4, 64, dtype=torch.int32),
                torch.zeros(0, 16)):
        with pytest.raises(ValueError):
            ops.quantize_fp8(bad)
    x = torch.zeros(3, 160, dtype=torch.bfloat16)
    rows = ops.Fp8Rows(torch.zeros(3, 160).to(f8), torch.ones(3, 2).to(e8))
    for call in (lambda: ops.linear_fp8(x, w), lambda: ops.linear_fp8(rows, w),
                 lambda: ops.quantize_rows_fp8(x),
                 lambda: ops.rmsnorm_fp8(x, torch.ones(160, dtype=torch.bfloat16), 1e-6)):
        with pytest.raises(ValueError):  # not on a GPU
            call()


def test_refusals(hv):
    lib = hv._lib.lib()
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 63) // 64 * 64

    def linear(x=p, xs=4096, xe=p, xes=32, w=p, s=p, rows=4, k=4096, n=4096, epi=0, out=p,
               ys=4096, ye=p, yes=32, ws=None, ws_bytes=0):
        return lib.hs_linear_fp8(x, xs, xe, xes, w, s, rows, k, n, epi, out, ys, ye, yes, ws,
                                 ws_bytes, None)

    assert linear(rows=0, x=None) == 0
    assert linear(x=None) == linear(w=None) == linear(s=None) == linear(out=None) == -1
    assert linear(epi=2, ye=None) == linear(rows=-1) == linear(k=0) == linear(n=0) == -1
    assert linear(epi=3) == linear(epi=-1) == -1
    assert linear(k=4088) == linear(xs=4088) == linear(xs=4104) == linear(x=p + 8) == -4
    assert linear(xs=(1 << 22) + 16) == linear(rows=(1 << 20) + 1) == linear(k=(1 << 22) + 16) == -4
    assert linear(xes=28) == linear(xes=34) == linear(xe=p + 2) == linear(xe=None, xs=4100) == -4
    assert linear(ys=4095) == linear(w=p + 8) == linear(s=p + 2) == linear(out=p + 1) == -4
    assert linear(n=24, epi=1) == linear(n=24, epi=2) == linear(n=(1 << 24) + 16) == -4
    assert linear(epi=2, ys=4104) == linear(epi=2, out=p + 8) == linear(epi=2, yes=31) == -4
    for bf16, epi, rows in ((1, 0, 64), (0, 2, 4), (1, 2, 64)):
        need = lib.hs_linear_fp8_workspace_size(rows, 4096, 4096, epi, bf16)
        xe = None if bf16 else p
        assert need > 0 and linear(rows=rows, xe=xe, epi=epi) == -2
        assert linear(rows=rows, xe=xe, epi=epi, ws=p, ws_bytes=need - 1) == -2
        assert linear(rows=rows, xe=xe, epi=epi, ws=p + 8, ws_bytes=need) == -4
    assert lib.hs_linear_fp8_workspace_size(0, 4096, 4096, 0, 0) == 0
    assert lib.hs_linear_fp8_workspace_size(4, 4096, 4096, 3, 0) == 0
    for sizes in (((1 << 20) + 1, 4096, 4096), (64, (1 << 31) - 1, 4096), (64, 4096, (1 << 31) - 1)):
        assert lib.hs_linear_fp8_workspace_size(*sizes, 2, 1) == 0

    def quantize(x=p, xs=256, rows=2, k=256, c=p, cs=256, s=p, ss=2):
        return lib.hs_quantize_rows_fp8(x, xs, rows, k, c, cs, s, ss, None)

    def norm(x=p, xs=256, res=p, rs=256, w=p, rows=2, k=256, c=p, cs=256, s=p, ss=2):
        return lib.hs_rmsnorm_fp8(x, xs, res, rs, w, 1e-6, rows, k, c, cs, s, ss, None)

    for f in (quantize, norm):
        assert f(rows=0, x=None) == 0
        assert f(x=None) == f(c=None) == f(s=None) == f(rows=-1) == f(k=0) == -1
        assert f(k=248) == f(xs=248) == f(xs=260) == f(cs=248) == f(cs=260) == f(ss=1) == -4
        assert f(x=p + 8) == f(c=p + 4) == f(rows=1 << 22) == -4
    assert quantize(rows=(1 << 22) - 1, k=1 << 20, xs=1 << 20, cs=1 << 20, ss=1 << 13) == -4
    assert norm(w=None) == -1
    assert norm(w=p + 8) == norm(res=p + 8) == norm(rs=248) == norm(rs=260) == -4
