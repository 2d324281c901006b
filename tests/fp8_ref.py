"""Plain restatements, in 64 bits on the host, of rows in 8 bits and of the projections over
them."""
import torch

GROUP = 128


def pow2(e):
    return torch.ldexp(torch.ones((), dtype=torch.float64), e)


def scale_of(amax):
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    m, e = torch.frexp(amax.double())  # m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return pow2(torch.where(m > 0, e, -126).clamp(min=-126))


def e4m3(x):
    """The e4m3 value nearest to each |x| <= 448, ties to the even one; NaN and infinities
    are NaN."""
    fine = torch.isfinite(x)
    _, e = torch.frexp(torch.where(fine, x, 1.0))
    step = pow2((e - 4).clamp(min=-9))
    return torch.where(fine, torch.round(x / step) * step, float("nan"))


def groups(x):
    """[rows, groups, 128], padded with zeros."""
    pad = -x.shape[1] % GROUP
    return torch.nn.functional.pad(x.double(), (0, pad)).view(x.shape[0], -1, GROUP)


def rows(x):
    """Codes (as values) and scales of rows x, all in 64 bits."""
    g = groups(x)
    s = scale_of(torch.where(torch.isfinite(g), g.abs(), 0.0).amax(-1))
    return e4m3(g / s[..., None]).view(x.shape[0], -1)[:, :x.shape[1]], s


def values(codes, scales):
    """The rows that codes and scales stand for, in 64 bits."""
    s = scales.double().repeat_interleave(GROUP, 1)[:, :codes.shape[1]]
    return codes.double() * s


def weight(codes, scales):
    s = scales.double().repeat_interleave(GROUP, 0).repeat_interleave(GROUP, 1)
    return codes.double() * s[:codes.shape[0], :codes.shape[1]]


def check_rows(codes, scales, y, tol):
    """codes and scales (from the GPU) of rows whose values are y (64 bits), computed to
    within tol: every scale is that of an amax within reach, and every value is off by at
    most half a step of its code beside tol."""
    amax, most = groups(y).abs().amax(-1), groups(tol).amax(-1)
    s = scales.double().cpu()
    low, high = scale_of((amax - most).clamp(min=0)), scale_of(amax + most)
    assert bool(((s >= low) & (s <= high)).all())
    off = (values(codes.cpu(), scales.cpu()) - y).abs()
    # half a step: 2^-4 of the value, and 2^-10 of the scale among e4m3's subnormals
    half = torch.maximum((y.abs() + tol) * 2.0 ** -4,
                         s.repeat_interleave(GROUP, 1)[:, :y.shape[1]] * 2.0 ** -10)
    assert bool((off <= half + tol).all()), float((off / (half + tol)).max())
