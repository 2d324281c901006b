"""RMSNorm to 8 bits with a residual of any layout whose elements are apart."""
import importlib

import pytest
import torch


def _layouts(m, k):
    """Strided views [m, k] of their own storage, by name: as a function of a device."""
    def of(shape, pick):
        return lambda dev: pick(torch.full(shape, 7.0, dtype=torch.bfloat16, device=dev))
    return {
        "columns first": of((k, m), lambda t: t.t()),
        "columns first, apart": of((k, m + 3), lambda t: t.t()[:m]),
        "every second value": of((m, 2 * k), lambda t: t[:, ::2]),
        # rows that follow each other by less than twice their length
        "every second value, close": of((m * (2 * k - 1) + 1,),
                                        lambda t: t.as_strided((m, k), (2 * k - 1, 2))),
    }


_OVERLAPS = [((3, 160), (0, 1)), ((3, 160), (160, 0)), ((3, 160), (159, 1)), ((3, 160), (16, 16)),
             ((3, 160), (1, 2)), ((3, 160), (318, 2)), ((1, 160), (160, 0))]


def test_overlaps():
    """The check takes what is apart, and names every layout whose addresses meet."""
    check = importlib.import_module("hilda-vllm_amd.ops")._overlaps
    base = torch.zeros(4096, dtype=torch.bfloat16)
    for m, k in ((1, 16), (2, 16), (3, 160), (5, 32)):
        for make in _layouts(m, k).values():
            assert not check(make("cpu"))
    for shape, stride in _OVERLAPS:
        assert check(base.as_strided(shape, stride))
    for shape in ((1, 1), (1, 6), (4, 1), (2, 3), (3, 5)):
        for row in range(13):
            for col in range(13):
                at = {i * row + j * col for i in range(shape[0]) for j in range(shape[1])}
                apart = len(at) == shape[0] * shape[1]
                # (a step in between may be refused though the addresses differ)
                assert apart or check(base.as_strided(shape, (row, col)))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(1, 160), (3, 160), (70, 1024)])
@pytest.mark.parametrize("name", list(_layouts(1, 1)))
def test_residuals_of_any_layout(hv, cuda, size, name):
    """The rows and the updated residual are those of a contiguous one; what lies between its
    values stays."""
    gen = torch.Generator().manual_seed(size[1])
    x = torch.randn(*size, generator=gen).to(torch.bfloat16).to(cuda)
    r = torch.randn(*size, generator=gen).mul(5).to(torch.bfloat16).to(cuda)
    w = torch.rand(size[1], generator=gen).to(torch.bfloat16).to(cuda)
    want_r = r.clone()
    want = hv.ops.rmsnorm_fp8(x, w, 1e-6, residual=want_r)
    res = _layouts(*size)[name](cuda)
    res.copy_(r)
    got = hv.ops.rmsnorm_fp8(x, w, 1e-6, residual=res)
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(res, want_r)
    taken = torch.zeros_like(res._base, dtype=torch.bool)
    taken.as_strided(res.shape, res.stride(), res.storage_offset()).fill_(True)
    assert bool((res._base[~taken] == 7).all())


@pytest.mark.gpu
def test_overlapping_residuals_are_refused(hv, cuda):
    base = torch.zeros(4096, dtype=torch.bfloat16, device=cuda)
    for shape, stride in _OVERLAPS:
        x = torch.zeros(shape, dtype=torch.bfloat16, device=cuda)
        w = torch.ones(shape[1], dtype=torch.bfloat16, device=cuda)
        with pytest.raises(ValueError):
            hv.ops.rmsnorm_fp8(x, w, 1e-6, residual=base.as_strided(shape, stride))
