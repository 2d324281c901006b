"""e4m3 weights of values that are not finite (on the host)."""
import pytest
import torch

import fp8_ref as ref


def _values(w):
    """The weight that the layout stands for: lane 16 g + f of a step holds feature f, inputs
    64 h + 16 g .. + 15."""
    tiles, steps = w.packed.shape[:2]
    c = w.packed.view(tiles, steps, 2, 4, 16, 16).permute(0, 4, 1, 2, 3, 5)
    c = c.reshape(tiles * 16, -1).view(torch.float8_e4m3fn)
    c = c[:w.out_features, :w.in_features]
    return ref.weight(c, w.scales[::8]), w.scales


@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("n,k", [(16, 16), (200, 272), (130, 128)])
def test_nonfinite_weights_stay_by_themselves(hv, n, k, bad):
    """A NaN or an infinity is NaN and takes no part in its block's scale: all other values are
    those of the weight without it."""
    weight = torch.randn(n, k, generator=torch.Generator().manual_seed(n))
    weight[n // 2, k // 2] = 0
    want, scales = _values(hv.ops.quantize_fp8(weight))
    weight[n // 2, k // 2] = float(bad)
    got, s = _values(hv.ops.quantize_fp8(weight))
    assert torch.equal(s, scales)
    assert bool(got[n // 2, k // 2].isnan())
    got[n // 2, k // 2] = 0
    assert torch.equal(got, want)


def test_a_block_of_nothing_finite(hv):
    """The least scale, and NaN; the next block is untouched."""
    weight = torch.ones(128, 256)
    weight[:, :128] = float("inf")
    got, s = _values(hv.ops.quantize_fp8(weight))
    assert bool((s[:, 0] == 2.0 ** -126).all())
    assert bool(got[:, :128].isnan().all())
    assert bool(((got[:, 128:] - 1).abs() <= 2.0 ** -22).all())


@pytest.mark.gpu
def test_the_device_quantises_alike(hv, cuda):
    """The same NaN, and values within half a step of the weight's. A block's scale is the host's
    to 2^-23: on the device the division by 448 is a product with its rounded inverse."""
    weight = torch.randn(200, 272, generator=torch.Generator().manual_seed(3))
    for i, bad in enumerate(("nan", "inf", "-inf")):
        weight[i * 70, i * 130] = float(bad)
    fine = torch.isfinite(weight)
    w = hv.ops.quantize_fp8(weight.to(cuda))
    got, scales = _values(w._replace(packed=w.packed.cpu(), scales=w.scales.cpu()))
    want = hv.ops.quantize_fp8(weight).scales.double()
    assert bool(((scales - want).abs() <= want * 2.0 ** -23).all())
    assert torch.equal(got.isnan(), ~fine)
    s = scales.double().repeat_interleave(16, 0).repeat_interleave(128, 1)[:200, :272]
    size = weight.double().abs()
    half = torch.maximum(size * 2.0 ** -4, s * 2.0 ** -10) + size * 2.0 ** -22
    assert bool(((got - weight).abs() <= half)[fine].all())
