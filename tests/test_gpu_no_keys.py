"""Calls whose sequences have no keys at all."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [[1], [4, 0, 2], [700, 900]])
def test_rows_without_keys(hv, cuda, rows):
    """Every sequence is empty and so is the declared longest: zeros, as for any row that sees
    no key."""
    print("attention without keys", rows, flush=True)
    n, B = sum(rows), len(rows)
    kc = torch.full((2, 64, 8, 128), 0x7f, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    ks = torch.full((2, 2, 8), float("nan"), device=cuda)
    q = torch.randn(n, 16, 128, device=cuda).to(torch.bfloat16)
    cu = torch.tensor([0] + torch.tensor(rows).cumsum(0).tolist(), dtype=torch.int32, device=cuda)
    out = hv.ops.verify_attention_scaled(q, kc, kc, ks, ks, torch.full((B, 1), -1, dtype=torch.int32,
                                                                       device=cuda),
                                         cu, torch.zeros_like(cu), max(rows), 0, 0.1)
    assert bool((out == 0).all())


def test_a_negative_bound_is_refused(hv, cuda):
    print("negative bound on the keys", flush=True)
    kc = torch.zeros((2, 64, 8, 128), dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    ks = torch.ones((2, 2, 8), device=cuda)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    with pytest.raises(RuntimeError):
        hv.ops.verify_attention_scaled(torch.zeros(1, 16, 128, dtype=torch.bfloat16, device=cuda), kc,
                                       kc, ks, ks, torch.zeros((1, 1), dtype=torch.int32, device=cuda),
                                       cu, cu, 1, -1, 0.1)
