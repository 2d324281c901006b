"""Log-probabilities at their limits: not-a-number far below the row's
maximum, and rows that are certain."""
import pytest
import torch

from test_gpu_token_logprobs import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [9, 200])
def test_nan_far_below_the_maximum(hv, cuda, rows, dtype):
    """A NaN reaches its row's results wherever it lies: alone in a chunk, among masked
    tokens, among values too far below the row's maximum to weigh anything, and under a
    temperature that puts them there. (9 rows run with 8 values a thread, 200 with 16:
    chunks of 2048 and 4096 logits.)"""
    print("NaN far below", rows, dtype, flush=True)
    V, inf, nan = 20001, float("inf"), float("nan")
    chunk = 2048 if rows == 9 else 4096
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, V, generator=gen)
    x[0, chunk:2 * chunk] = nan  # a whole chunk
    x[1, chunk:2 * chunk] = -inf  # masked but for a NaN
    x[1, chunk + 77] = nan
    x[2, 2 * chunk:3 * chunk] -= 200  # far below
    x[2, 2 * chunk + 5] = nan
    x[3, 2 * chunk:3 * chunk] -= 10  # far below at the row's temperature
    x[3, 3 * chunk - 1] = nan
    x[4, (V - 1) // chunk * chunk:] = nan  # the last, short chunk
    x[5] = -inf  # nothing but masked tokens, one value and a NaN in another chunk
    x[5, [3, V - 1]] = torch.tensor([1.0, nan])
    x[6, :chunk] = -inf  # no NaN at all
    x = x.to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    tokens = torch.randint(V, (rows,), generator=gen)
    temps = torch.ones(rows)
    temps[3] = 0.05
    for top in (0, 20):
        got = hv.ops.token_logprobs(x.to(cuda), tokens.to(cuda), top=top,
                                    temperatures=temps.to(cuda))
        for r in range(6):
            assert bool(got["logprobs"][r].isnan() and got["entropy"][r].isnan()), (r, top)
        _check(got, x, tokens, top, temps)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [224, 2000])
def test_certain_rows(hv, cuda, rows, dtype):
    """Where one token has all of the probability its log-probability and the entropy are 0,
    and where nearly all, the log-probability is never above 0: every difference from the
    maximum is exact or rounds below it, the maximum's own term is exp(0) = 1, and sums of
    terms that are not negative stay at 1 or more. (224 rows run with 8 values a thread,
    2000 with 16.)"""
    print("certain rows", rows, dtype, flush=True)
    V = 2501
    gen = torch.Generator().manual_seed(rows)
    m = torch.linspace(0.37, 88.0, rows).to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    x = torch.full((rows, V), -float("inf"), dtype=m.dtype)
    at = torch.randint(V, (rows,), generator=gen)
    x[torch.arange(rows), at] = m
    for temps in (None, torch.rand(rows, generator=gen) * 2 + 0.05):
        t = None if temps is None else temps.to(cuda)
        got = hv.ops.token_logprobs(x.to(cuda), at.to(cuda), top=1, temperatures=t)
        assert bool((got["logprobs"] == 0).all()), float(got["logprobs"].abs().max())
        assert bool((got["top_logprobs"] == 0).all() and (got["entropy"] == 0).all())
        assert torch.equal(got["top_ids"][:, 0].cpu(), at)
        # the others 5 to 40 below
        y = m[:, None].float() - 5 - 35 * torch.rand(rows, V, generator=gen)
        y = y.to(m.dtype)
        y[torch.arange(rows), at] = m
        got = hv.ops.token_logprobs(y.to(cuda), at.to(cuda), top=1, temperatures=t)
        assert bool((got["logprobs"] <= 0).all()), float(got["logprobs"].max())
        assert bool((got["top_logprobs"] <= 0).all() and (got["entropy"] >= 0).all())
        _check(got, y, at, 1, temps)


def test_nearly_certain_tokens(hv, cuda):
    """One other token d below the certain one: log p = -log(1 + exp(-d)), to what 32 bits
    hold of a sum next to 1 (half a step of 2^-23, as much for the exponential and the
    logarithm together: 2^-22)."""
    d = torch.linspace(6, 15, 64)
    gen = torch.Generator().manual_seed(3)
    m = torch.rand(64, generator=gen) * 60 + 1
    x = torch.full((64, 5000), -float("inf"))
    x[:, 4000], x[:, 17] = m, m - d
    d = x[:, 4000].double() - x[:, 17].double()
    got = hv.ops.token_logprobs(x.to(cuda), torch.full((64,), 4000, device=cuda))
    err = (got["logprobs"].double().cpu() + torch.log1p(torch.exp(-d))).abs()
    assert float(err.max()) <= 2.0 ** -22, float(err.max())
