"""Every kernel for projections of rows in 8 bits, by the sizes of fp8_cases, against the same
sums in 64 bits."""
import pytest
import torch

import fp8_ref as ref
from fp8_cases import CASES, ids, plan
from test_gpu_fp8_linear import _reference, _same

pytestmark = pytest.mark.gpu

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _codes(x):
    return x.clamp(-448, 448).to(E4M3)


class Setup:
    """Weights, row codes and exponents of a case, on the GPU; the codes lie in wider rows and
    the exponents in words whose other bytes are NaN."""

    def __init__(self, hv, cuda, case, spread=4):
        self.ops, (self.k, self.n, self.rows, self.epilogue) = hv.ops, case
        k, rows, steps = self.k, self.rows, -(-self.k // 128)
        self.gate = self.epilogue != "plain"
        self.how = dict(swiglu=self.gate, quantize=self.epilogue == "eight")
        gen = torch.Generator(device=cuda).manual_seed(k + self.n + rows)
        rand = lambda *size: torch.randn(*size, generator=gen, device=cuda)  # noqa: E731
        features = self.n * (2 if self.gate else 1)
        self.wcodes = _codes(rand(features, k) * 100)
        self.wscales = rand(-(-features // 128), steps).abs() * 2e-3 + 1e-5
        self.w = hv.ops.pack_fp8(self.wcodes, self.wscales)
        wide = torch.full((rows, k + 32), 0x7f, dtype=torch.uint8, device=cuda).view(E4M3)
        wide[:, 16:16 + k] = _codes(rand(rows, k) * 60)
        self.codes = wide[:, 16:16 + k]
        self.bytes = torch.full((rows, -(-steps // 4) * 4 + 4), 255, dtype=torch.uint8, device=cuda)
        e = torch.randint(-spread, 1, (rows, steps), generator=gen, device=cuda)
        self.bytes[:, :steps] = (e + 120).to(torch.uint8)
        self.steps = steps

    def exponents(self):
        return self.bytes[:, :self.steps]

    def x(self):
        return self.ops.Fp8Rows(self.codes, self.exponents().view(E8M0))

    def run(self, x=None, **more):
        return self.ops.linear_fp8(self.x() if x is None else x, self.w, **self.how, **more)

    def reference(self):
        s = torch.exp2(self.exponents().double() - 127)
        x = ref.values(self.codes, s)
        return _reference(x, self.wcodes, self.wscales, self.epilogue, self.n)

    def check(self, got, y, tol):
        if self.epilogue == "eight":
            ref.check_rows(got.codes, got.scales, y.cpu(), tol.cpu())
            return
        err, tol = (got.double() - y).abs(), tol + 2.0 ** -8 * (y.abs() + tol)
        assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_every_kernel(hv, cuda, case):
    print("fp8 kernel", case, plan(hv, *case), flush=True)
    s = Setup(hv, cuda, case)
    got, (y, tol) = s.run(), s.reference()
    s.check(got, y, tol)
    assert _same(s.run(), got)
    if s.epilogue != "eight":  # an output off the 16-byte pieces, between others' values
        wide = torch.full((s.rows + 1, s.n + 5), 7.0, dtype=torch.bfloat16, device=cuda)
        out = wide[:s.rows, 3:3 + s.n]
        assert s.run(out=out) is out and _same(out, got)
        assert bool((wide[s.rows] == 7).all() and (wide[:, :3] == 7).all())
        assert bool((wide[:, 3 + s.n:] == 7).all())
    # bf16 rows: those that the codes of some others stand for
    x = s.codes.float().mul(torch.exp2(torch.randint(-8, 9, (s.rows, 1), device=cuda).float()))
    x = x.to(torch.bfloat16)
    assert _same(s.run(x), s.run(s.ops.quantize_rows_fp8(x)))


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_rows_do_not_meet_in_any_kernel(hv, cuda, case):
    """A NaN code, or a scale that is NaN (byte 255), makes its row NaN; the least scales (bytes 0
    and 1) make theirs less than 2^-95; the other rows keep their bits. (The bytes behind a row's
    last scale are 255 all along.)"""
    print("fp8 rows", case, plan(hv, *case), flush=True)
    s = Setup(hv, cuda, case)
    want = s.run()
    s.codes.view(torch.uint8)[1, s.k - 3] = 0x7f
    s.exponents()[s.rows - 1, s.steps // 2] = 255
    s.exponents()[0] = torch.arange(s.steps, device=cuda) % 2
    got = s.run()
    if s.epilogue == "eight":
        values = got.codes.float()
        least = values[0] * got.scales[0].float().repeat_interleave(128)[:s.n]
        kept = _same(s.ops.Fp8Rows(got.codes[2:-1], got.scales[2:-1]),
                     s.ops.Fp8Rows(want.codes[2:-1], want.scales[2:-1]))
        assert bool((got.scales[[1, s.rows - 1]].float() == 2.0 ** -126).all())
    else:
        values, least, kept = got, got[0], _same(got[2:-1], want[2:-1])
    assert kept
    assert bool(values[[1, s.rows - 1]].isnan().all())
    assert bool((least.abs() < 2.0 ** -95).all())


_BATCHES = (1, 3, 8, 9, 16, 17, 24, 32, 33, 48, 64, 65, 96, 129, 200, 256, 257, 300, 400, 512, 513,
            640, 777, 1024, 1100, 1500, 2051)


@pytest.mark.parametrize("k,n,epilogue", [
    (1040, 528, "plain"), (1040, 4099, "plain"), (12288, 4096, "plain"), (2064, 8200, "plain"),
    (1040, 2064, "swiglu"), (4096, 4112, "swiglu"), (1040, 2064, "eight"), (4096, 4112, "eight")])
def test_a_row_in_many_batches(hv, cuda, k, n, epilogue):
    """All rows of every batch are within their bounds, and a row has the same bits in every batch
    of one plan, wherever it lies in it: first and last rows are shared between batches."""
    print("fp8 batches", k, n, epilogue, flush=True)
    s = Setup(hv, cuda, (k, n, _BATCHES[-1], epilogue))
    y, tol = s.reference()
    plans = {}
    for m in _BATCHES:
        last = slice(s.rows - m, s.rows)
        first = s.run(s.ops.Fp8Rows(s.codes[:m], s.exponents().view(E8M0)[:m]))
        other = s.run(s.ops.Fp8Rows(s.codes[last], s.exponents().view(E8M0)[last]))
        s.check(first, y[:m], tol[:m])
        s.check(other, y[last], tol[last])
        plans.setdefault(plan(hv, k, n, m, epilogue), []).append((m, first, other))
    part = (lambda t, at: s.ops.Fp8Rows(t.codes[at], t.scales[at])) if epilogue == "eight" else \
        (lambda t, at: t[at])
    for same in plans.values():
        for (m, first, other), (more, longer, late) in zip(same, same[1:]):
            assert _same(part(longer, slice(0, m)), first)
            assert _same(part(late, slice(more - m, more)), other)
            if more + m > s.rows:  # rows that the first `more` and the last m share
                both = more + m - s.rows
                assert _same(part(longer, slice(more - both, more)), part(other, slice(0, both)))
    assert len(plans) >= 3


# calls that split their steps, and so have a workspace of sums, or one of codes beside it
_SPLITS = [(12288, 4096, 64, "plain"), (12288, 1030, 300, "plain"), (12288, 1024, 128, "swiglu"),
           (6160, 2080, 66, "eight"), (12288, 4096, 64, "plain")]


def test_captured_splits_share_nothing(hv, cuda):
    """Graphs of calls that split their steps, of rows in 8 bits and of bf16 rows, replayed at
    once on two streams over and over with new inputs, with eager calls on both between them."""
    calls = []
    for case in _SPLITS:
        p = plan(hv, *case)
        assert p[3] < -(-case[0] // 128), (case, p)
        s = Setup(hv, cuda, case)
        raw = s.codes.view(torch.uint8)
        sets = [raw.clone(), raw.flip(0), raw.roll(3, 0)]
        bf16 = s.codes.to(torch.bfloat16)
        graphs = []
        for x in (s.x(), bf16):
            s.run(x)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = s.run(x)
            graphs.append((g, y))
        calls.append((s, sets, bf16, graphs))
    side = torch.cuda.Stream()
    whole = lambda y: y if isinstance(y, torch.Tensor) else y.codes.view(torch.uint8)  # noqa: E731
    for turn in range(4):
        want = []
        for s, sets, bf16, graphs in calls:
            s.codes.view(torch.uint8).copy_(sets[turn % 3])
            bf16.copy_(s.codes)
            want.append([s.run(), s.run(bf16)])
            for _, y in graphs:
                whole(y).zero_()
        torch.cuda.synchronize()
        beside, eager = [], []
        for s, _, bf16, graphs in calls:
            graphs[0][0].replay()
            with torch.cuda.stream(side):
                graphs[1][0].replay()
                beside.append([s.run(), s.run(bf16)])
            eager.append([s.run(bf16), s.run()])
        torch.cuda.synchronize()
        for (s, _, _, graphs), w, b, e in zip(calls, want, beside, eager):
            assert _same(graphs[0][1], w[0]) and _same(graphs[1][1], w[1])
            assert _same(b[0], w[0]) and _same(b[1], w[1])
            assert _same(e[0], w[1]) and _same(e[1], w[0])
