"""Log-probabilities where a row's chunks differ most: not-a-number far below the row's
maximum."""
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
