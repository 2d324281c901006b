"""Sizes of projections of rows in 8 bits that reach every kernel there is for them, each with the
epilogues and ways of sharing the steps that it can be launched with, in ragged sizes (inputs,
features, rows, epilogue), and what such a call launches."""
import ctypes

EPILOGUES = ("plain", "swiglu", "eight")

CASES = [
    (1040, 37, 13, "plain"), (8464, 37, 13, "plain"), (1040, 37, 3, "plain"),
    (8464, 37, 3, "plain"), (1040, 37, 1537, "plain"), (8464, 37, 1537, "plain"),
    (1040, 37, 2050, "plain"), (1040, 50001, 13, "plain"), (8464, 50001, 13, "plain"),
    (1040, 50001, 19, "plain"), (8464, 50001, 19, "plain"), (1040, 530, 515, "plain"),
    (8464, 530, 1100, "plain"), (8464, 201, 605, "plain"), (1040, 530, 2050, "plain"),
    (8464, 2070, 605, "plain"), (8464, 37, 2050, "plain"), (1040, 1045, 2050, "plain"),
    (8464, 1045, 2050, "plain"), (12288, 37, 2050, "plain"), (1040, 16390, 131, "plain"),
    (8464, 16390, 131, "plain"), (16400, 4099, 131, "plain"), (1040, 16390, 390, "plain"),
    (8464, 16390, 390, "plain"), (1040, 48, 3, "swiglu"), (8464, 48, 3, "swiglu"),
    (1040, 48, 1537, "swiglu"), (1040, 1056, 101, "swiglu"), (8464, 208, 1537, "swiglu"),
    (4112, 1056, 101, "swiglu"), (1040, 208, 2050, "swiglu"), (8464, 2080, 257, "swiglu"),
    (8464, 48, 1537, "swiglu"), (1040, 8208, 66, "swiglu"), (8464, 4112, 195, "swiglu"),
    (6160, 2080, 66, "swiglu"), (1040, 16400, 35, "swiglu"), (8464, 16400, 35, "swiglu"),
    (16400, 2080, 131, "swiglu"), (1040, 16400, 131, "swiglu"), (8464, 16400, 131, "swiglu"),
    (1040, 48, 3, "eight"), (8464, 48, 3, "eight"), (1040, 48, 1537, "eight"),
    (1040, 208, 777, "eight"), (8464, 8208, 19, "eight"), (1040, 1056, 101, "eight"),
    (1040, 208, 2050, "eight"), (8464, 8208, 35, "eight"), (2064, 2080, 35, "eight"),
    (2064, 8208, 66, "eight"), (8464, 4112, 301, "eight"), (6160, 2080, 66, "eight"),
    (1040, 544, 1537, "eight"), (8464, 16400, 35, "eight"), (6160, 8208, 66, "eight"),
    (1040, 16400, 131, "eight"), (8464, 16400, 131, "eight"), (2064, 6150, 2053, "plain"),
    (2064, 4112, 2053, "swiglu"), (2064, 4112, 2053, "eight"), (1040, 4099, 1100, "plain"),
]


def ids(case):
    return "-".join(map(str, case))


def plan(hv, k, n, rows, epilogue, bf16_rows=False):
    """Features and rows of a workgroup, its waves, and the steps it adds."""
    out = (ctypes.c_int * 4)()
    status = hv._lib.lib().hs_linear_fp8_plan(rows, k, n, EPILOGUES.index(epilogue), bf16_rows,
                                              ctypes.addressof(out))
    assert status == 0
    return tuple(out)


def variant(hv, k, n, rows, epilogue):
    """What the tests tell apart: the kernel's sizes, the epilogue, and whether the steps are
    split over workgroups, or more than the 64 whose scales a workgroup of a tile holds at once."""
    p, steps = plan(hv, k, n, rows, epilogue), -(-k // 128)
    how = "split" if p[3] < steps else "long" if steps > 64 else ""
    return (epilogue, *p[:3], how)
