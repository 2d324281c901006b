"""Which kernel serves a projection of rows in 8 bits, on the host."""
import ctypes

from fp8_cases import CASES, EPILOGUES, plan, variant


def test_cases_reach_every_variant(hv):
    """Every variant that some size of a wide grid is launched with is among the sizes that the
    GPU tests run, so that a change of the rules cannot leave one without."""
    tested, reached = {variant(hv, *c) for c in CASES}, {}
    for k in (16, 128, 640, 1040, 2064, 4096, 4112, 6160, 8192, 8464, 12288, 16400):
        for n in (16, 37, 208, 528, 1040, 2064, 4096, 4112, 6144, 8192, 12288, 24576, 60000,
                  131072):
            for rows in (1, 2, 4, 8, 9, 16, 17, 24, 32, 33, 48, 64, 65, 100, 128, 192, 256, 300,
                         384, 512, 531, 600, 768, 1000, 1100, 1500, 2048, 4096, 20000):
                for epilogue in EPILOGUES:
                    size = (k, n if epilogue == "plain" else -(-n // 16) * 16, rows, epilogue)
                    reached.setdefault(variant(hv, *size), size)
    assert {v: size for v, size in reached.items() if v not in tested} == {}


def test_splits_have_a_workspace(hv):
    """Parts of split steps, f32 sums of every row, are what the workspace holds, and with bf16
    rows their codes."""
    size = hv._lib.lib().hs_linear_fp8_workspace_size
    for k, n, rows, epilogue in CASES:
        features, _, _, split = plan(hv, k, n, rows, epilogue)
        parts = -(-(-(-k // 128)) // split)
        need = 0
        if parts > 1 or epilogue == "eight" and features < 256:
            need = parts * rows * -(-n // 16) * (32 if epilogue != "plain" else 16) * 4
        got = size(rows, k, n, EPILOGUES.index(epilogue), 0)
        assert need <= got < need + 256 and (need or not got)


def test_refusals_of_a_plan(hv):
    ask, out = hv._lib.lib().hs_linear_fp8_plan, (ctypes.c_int * 4)()
    at = ctypes.addressof(out)
    assert ask(4, 4096, 4096, 0, 0, at) == 0 and min(out) > 0
    assert ask(4, 4096, 4096, 0, 0, None) == ask(0, 4096, 4096, 0, 0, at) == -1
    assert ask(4, 0, 4096, 0, 0, at) == ask(4, 4096, 0, 0, 0, at) == -1
    assert ask(4, 4096, 4096, 3, 0, at) == -1
    big = (1 << 31) - 1
    assert ask((1 << 20) + 1, 4096, 4096, 0, 0, at) == -4
    assert ask(4, big, 4096, 0, 0, at) == ask(4, 4096, big, 2, 1, at) == -4
