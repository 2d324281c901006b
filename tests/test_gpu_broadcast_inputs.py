"""Broadcast rows, and single rows with a stride of their own, of the quantised path's
calls."""
import pytest
import torch

import test_gpu_scaled_kv as kv

pytestmark = pytest.mark.gpu


def test_logits(hv, cuda):
    print("log-probabilities of broadcast rows", flush=True)
    x = torch.randn(1, 5003, generator=torch.Generator().manual_seed(1)).to(cuda)
    tokens = torch.tensor([7, 5002, 0], device=cuda)
    want = hv.ops.token_logprobs(x.repeat(3, 1), tokens, top=5)
    got = hv.ops.token_logprobs(x.expand(3, 5003), tokens, top=5)
    column = x[0][:, None]  # [5003, 1]: its transpose is one row with a stride of 1
    assert column.t().stride() == (1, 1)
    one = hv.ops.token_logprobs(column.t(), tokens[:1], top=5)
    for k, v in want.items():
        assert torch.equal(got[k], v) and torch.equal(one[k], v[:1])


def test_block_tables(hv, cuda):
    """Sequences that share all of their blocks, and a single table with a stride of 1."""
    print("attention over broadcast tables", flush=True)
    case = ("shared-blocks", 16, 8, 64, 32, [2, 1, 3], [700, 300, 650], 1024)
    host, x = kv._attend_inputs(cuda, case)
    # a table of its own for the longest sequence, whose blocks hold every key
    table = x["bt"][:1, :11].contiguous()
    want = kv._run(hv, case, dict(x, bt=table.repeat(3, 1)))
    got = kv._run(hv, case, dict(x, bt=table.expand(3, 11)))
    assert torch.equal(got, want)
    one = ("one", 16, 8, 64, 32, [2], [700], 1024)
    first = dict(x, q=x["q"][:2], cu_q=x["cu_q"][:2], cu_k=x["cu_k"][:2])
    column = table[0][:, None]
    assert column.t().stride() == (1, 1)
    assert torch.equal(kv._run(hv, one, dict(first, bt=column.t())), want[:2])
