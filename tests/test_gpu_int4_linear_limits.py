"""4-bit projections at the ends of the number range, against the same sums in 64 bits."""
import pytest
import torch

from test_gpu_int4_linear import _reference, _tolerance

pytestmark = pytest.mark.gpu

# inputs, features, group, rows, swiglu: every kernel and way of sharing out steps
_CASES = [
    (32, 16, 32, 1, False), (4096, 200, 128, 4, False), (12288, 64, 64, 16, False),
    (512, 16400, 32, 3, False), (256, 49200, 64, 2, False), (1024, 2048, 128, 7, True),
    (1024, 1001, 64, 17, False), (4096, 4096, 128, 63, False), (2048, 512, 32, 300, False),
    (12288, 4096, 64, 64, False), (512, 208, 64, 64, True), (4096, 8208, 128, 64, True),
]


def _check(hv, cuda, case, x, codes, scales):
    k, n, group, rows, swiglu = case
    got = hv.ops.linear_int4(x.to(cuda), hv.ops.pack_int4(codes.to(cuda), scales.to(cuda)),
                             swiglu=swiglu)
    y, size = _reference(x, codes, scales, group)
    tol = _tolerance(size, k, group)
    if swiglu:
        g, u = y[:, :n], y[:, n:]
        y = torch.nn.functional.silu(g) * u
        act = torch.nn.functional.silu(g).abs()
        # silu's slope is below 1.1; its exponential and quotient are good to 2^-18 here
        tol = 1.1 * tol[:, :n] * (u.abs() + tol[:, n:]) + act * tol[:, n:] + 2.0 ** -18 * y.abs()
    tol = tol + 2.0 ** -8 * y.abs()
    err = (got.double().cpu() - y).abs()
    assert bool(got.isfinite().all()), int((~got.isfinite()).sum())
    assert bool((err <= tol).all()), float((err / tol).max())
    # half of the gates lie far below 0, where silu is 0 in 32 bits
    assert bool((got != 0).float().mean() > (0.4 if swiglu else 0.9))


def _codes(gen, case):
    k, n, group, rows, swiglu = case
    m = 2 * n if swiglu else n
    return torch.randint(0, 16, (m, k), generator=gen, dtype=torch.uint8), \
        torch.rand(m, k // group, generator=gen) + 0.5


@pytest.mark.parametrize("case", _CASES, ids=["-".join(map(str, c)) for c in _CASES])
def test_largest_inputs(hv, cuda, case):
    """Inputs up to the largest finite bf16: the result is finite where the sum is, though 24
    times an input, or 31 times, is not."""
    k, n, group, rows, swiglu = case
    print("int4 linear, largest inputs", case, flush=True)
    gen = torch.Generator().manual_seed(k + n + rows)
    codes, scales = _codes(gen, case)
    # sums below k * 8 * 1.5e-5 / 2 of the largest input, or for SwiGLU of ordinary size
    scales = (scales * (2e-38 if swiglu else 1e-5 * min(1.0, 5000 / k))).to(torch.bfloat16)
    x = 3.38e38 * (torch.rand(rows, k, generator=gen) * 2 - 1).to(torch.float32)
    x = x.to(torch.bfloat16)
    x[0, 0], x[-1, -1] = 3.3895e38, -3.3895e38
    assert bool(x.isfinite().all())
    _check(hv, cuda, case, x, codes, scales)


@pytest.mark.parametrize("case", _CASES, ids=["-".join(map(str, c)) for c in _CASES])
def test_smallest_inputs(hv, cuda, case):
    """Inputs next to the smallest normal bf16, and below it, under large scales: a product
    with a code is a multiple of 2^-145, which f32 holds."""
    k, n, group, rows, swiglu = case
    print("int4 linear, smallest inputs", case, flush=True)
    gen = torch.Generator().manual_seed(k + n + rows + 1)
    codes, scales = _codes(gen, case)
    scales = (scales * 2.0 ** 120).to(torch.bfloat16)
    x = torch.randn(rows, k, generator=gen).double() * 2.0 ** -124
    x = x.to(torch.bfloat16)
    _check(hv, cuda, case, x, codes, scales)
