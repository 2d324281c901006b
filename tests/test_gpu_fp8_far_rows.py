"""RMSNorm to 8 bits of rows whose squares pass the range of 32 bits."""
import pytest
import torch

import fp8_ref as ref
from test_gpu_fp8_rows import _norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("size", [(5, 128), (6, 1024), (6, 2048), (9, 4096), (6, 8192), (6, 16384),
                                  (6, 40960)], ids=lambda c: "-".join(map(str, c)))
def test_rows_of_any_size(hv, cuda, size, residual):
    """Rows of ordinary size, of sizes around the one whose sum of squares is f32's largest, and
    of bf16's largest values (with a residual: of half of them), beside each other. A row that is
    summed in units of 2^80 loses squares below 2^-149 of them: none that counts."""
    m, k = size
    print("far rows", size, residual, flush=True)
    gen = torch.Generator().manual_seed(k)
    scale = torch.tensor([1.0, 2.0 ** 50, 2.0 ** 58, 2.0 ** 63, 2.0 ** 90] * 2)[:m]
    x = (torch.randn(m, k, generator=gen).clamp(-1.9, 1.9) * scale[:, None]).to(torch.bfloat16)
    x[-1] = torch.finfo(torch.bfloat16).max * (0.49 if residual else 1.0)
    x[-1, ::3] *= -1
    x[3, k // 2:] = 0.25  # far below the row's root mean square
    r = x.roll(1, 1) if residual else None
    w = (torch.rand(k, generator=gen) * 3 - 1).to(torch.bfloat16)
    h, y, tol = _norm(x, r, w, 1e-6)
    res = r.to(cuda) if residual else None
    got = hv.ops.rmsnorm_fp8(x.to(cuda), w.to(cuda), 1e-6, residual=res)
    assert bool(torch.isfinite(got.codes.float()).all())
    ref.check_rows(got.codes, got.scales, y, tol)
    if residual:
        assert torch.equal(res.cpu(), h.float().to(torch.bfloat16))


def test_an_infinity_stays_in_its_row(hv, cuda):
    """As in rows of ordinary size: it is NaN, the row's other values are zeros."""
    x = torch.ones(4, 4096, dtype=torch.bfloat16, device=cuda)
    w = torch.ones(4096, dtype=torch.bfloat16, device=cuda)
    want = hv.ops.rmsnorm_fp8(x, w, 1e-6)
    x[1, 9], x[2, 8] = float("inf"), float("nan")
    got = hv.ops.rmsnorm_fp8(x, w, 1e-6)
    for i in (0, 3):
        assert torch.equal(got.codes[i].view(torch.uint8), want.codes[i].view(torch.uint8))
    values = got.codes.float()
    assert bool(values[1, 9].isnan()) and int((values[1] != 0).sum()) == 1
    assert bool(values[2].isnan().all())
