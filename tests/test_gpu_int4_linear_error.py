"""4-bit projections: single inputs exactly, and the error's size over many outputs."""
import math

import pytest
import torch

from test_gpu_int4_linear import _reference, _weights

pytestmark = pytest.mark.gpu

# inputs, features, group, rows: every kernel and way of sharing out steps
_CASES = [
    (352, 2000, 32, 5), (4096, 4096, 128, 4), (12288, 512, 64, 16), (512, 16400, 32, 3),
    (256, 49200, 64, 2), (1024, 1001, 64, 17), (4096, 4096, 128, 63), (2048, 512, 32, 300),
    (12288, 4096, 64, 64), (4096, 8208, 128, 64), (1056, 30000, 32, 20),
]


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("case", _CASES, ids=["-".join(map(str, c)) for c in _CASES])
def test_single_inputs(hv, cuda, case, swiglu):
    """One input of 1 a row picks a column of weights out: (c - 8) s has 12 bits at most, and
    every sum on the way to it is exact. At the first and last input and around the ends of
    groups, steps and their shares."""
    k, n, group, rows = case
    n = n // 32 * 16 if swiglu else n
    print("int4 linear, single inputs", case, swiglu, flush=True)
    gen = torch.Generator().manual_seed(k + rows)
    codes, scales = _weights(gen, 2 * n if swiglu else n, k, group)
    w = hv.ops.pack_int4(codes.to(cuda), scales.to(cuda))
    edges = sorted({min(max(e + d, 0), k - 1) for e in [0, 32, 64, 128, 256, 512, k // 3 // 128 * 128,
                                                        k // 2 // 128 * 128, k // 2, k - 128, k - group,
                                                        k] for d in (-1, 0, 1)})
    edges += torch.randint(k, (max(0, rows - len(edges)),), generator=gen).tolist()
    for at in range(0, len(edges), rows):
        part = (edges[at:at + rows] + edges[:rows])[:rows]
        x = torch.zeros(rows, k, dtype=torch.bfloat16)
        x[torch.arange(rows), torch.tensor(part)] = 1
        got = hv.ops.linear_int4(x.to(cuda), w, swiglu=swiglu).cpu()
        col = torch.tensor(part)
        y = ((codes[:, col].double() - 8) * scales[:, col // group].double()).t()
        if swiglu:
            y = torch.nn.functional.silu(y[:, :n]) * y[:, n:]
            # silu's exponential and quotient are good to 2^-18, then one rounding
            assert bool(((got.double() - y).abs() <= (2.0 ** -8 + 2.0 ** -17) * y.abs()).all())
        else:
            assert torch.equal(got, y.to(torch.bfloat16))


@pytest.mark.parametrize("case", _CASES, ids=["-".join(map(str, c)) for c in _CASES])
def test_mean_error(hv, cuda, case):
    """The error's root mean square is that of rounding the exact sums to bf16, and the 32-bit
    sums' own: a group's partial sums, random walks of size 24 sqrt(group) |x| at most, lose at
    most 2^-23 of it in each of up to 2 group additions, and the groups' errors are
    independent. 5 % above their root sum of squares leaves room for the sample's own spread,
    not for one more rounding to bf16 on the way (a third more where it is the weights')."""
    k, n, group, rows = case
    print("int4 linear, mean error", case, flush=True)
    gen = torch.Generator().manual_seed(k + n)
    codes, scales = _weights(gen, n, k, group)
    x = torch.randn(rows, k, generator=gen).to(torch.bfloat16)
    w = hv.ops.pack_int4(codes.to(cuda), scales.to(cuda))
    got = hv.ops.linear_int4(x.to(cuda), w).double().cpu()
    y, _ = _reference(x, codes, scales, group)

    def rms(t):
        return float(t.double().square().mean().sqrt())

    rounding = rms(y.to(torch.bfloat16).double() - y)
    sums = 2.0 ** -23 * 2 * group * 24 * math.sqrt(group) * rms(x) * rms(scales) * \
        math.sqrt(k / group)
    assert rms(got - y) <= 1.05 * math.hypot(rounding, sums), (rms(got - y), rounding, sums)
