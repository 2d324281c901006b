"""4-bit projections on the host: the weight's layout and the refusals."""
import ctypes

import pytest
import torch


def _unpack(w):
    """Codes and scales back from the layout, by its definition."""
    tiles, steps = w.packed.shape[:2]
    codes = torch.full((tiles * 16, steps * 128), -1)
    for lane in range(64):
        for i in range(4):
            for e in range(8):
                word = w.packed[:, :, lane, i]
                c = (word >> (4 * (e // 2) + 16 * (e % 2))) & 15
                k = 32 * i + 8 * (lane // 16) + e
                codes.view(tiles, 16, steps, 128)[:, lane % 16, :, k] = c
    scales = w.scales.permute(0, 2, 1).reshape(tiles * 16, -1)
    return codes, scales


@pytest.mark.parametrize("n,k,group", [(16, 128, 128), (1, 32, 32), (37, 352, 32), (48, 320, 64)])
def test_layout(hv, n, k, group):
    gen = torch.Generator().manual_seed(n)
    codes = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.uint8)
    scales = torch.rand(n, k // group, generator=gen).to(torch.bfloat16)
    w = hv.ops.pack_int4(codes, scales)
    c, s = _unpack(w)
    assert torch.equal(c[:n, :k], codes.long()) and torch.equal(s[:n, :k // group], scales)
    assert bool((c[n:] == 8).all() and (c[:, k:] == 8).all())
    assert bool((s[n:] == 0).all() and (s[:, k // group:] == 0).all())


def test_quantize_takes_the_nearest_code(hv):
    gen = torch.Generator().manual_seed(2)
    weight = torch.randn(20, 128, generator=gen) * 3
    w = hv.ops.quantize_int4(weight, 32)
    c, s = _unpack(w)
    s = s[:20].double().repeat_interleave(32, 1)
    off = ((c[:20].double() - 8) * s - weight.double()).abs()
    # half a step, and where 7 steps fall short of the group's largest value by rounding
    assert bool((off <= 0.5 * s + 7 * s * 2.0 ** -8).all())


def test_weights_are_checked(hv):
    ops = hv.ops
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.bfloat16)
    for c, s, err in ((codes + 16, scales, ValueError), (codes, scales.float(), TypeError),
                      (codes.float(), scales, TypeError), (codes, scales[:3], ValueError),
                      (codes, scales[:, :0], ValueError), (codes[:, :63], scales, ValueError),
                      (codes, torch.zeros(4, 4, dtype=torch.bfloat16), ValueError)):
        with pytest.raises(err):
            ops.pack_int4(c, s)
    for bad, group in ((torch.zeros(4, 60), 32), (torch.zeros(4, 64), 16), (torch.zeros(64), 64),
                       (torch.zeros(4, 64, dtype=torch.int32), 64)):
        with pytest.raises(ValueError):
            ops.quantize_int4(bad, group)
    with pytest.raises(ValueError):  # not on a GPU
        ops.linear_int4(torch.zeros(1, 64, dtype=torch.bfloat16), ops.pack_int4(codes, scales))


def test_refusals(hv):
    lib = hv._lib.lib()
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 63) // 64 * 64

    def call(x=p, xs=4096, w=p, s=p, rows=4, k=4096, n=4096, group=128, epi=0, out=p, ys=4096,
             ws=None, ws_bytes=0):
        return lib.hs_linear_int4(x, xs, w, s, rows, k, n, group, epi, out, ys, ws, ws_bytes, None)

    assert call(rows=0, x=None) == 0
    assert call(x=None) == call(w=None) == call(s=None) == call(out=None) == -1
    assert call(rows=-1) == call(k=0) == call(n=0) == call(group=16) == call(epi=2) == -1
    assert call(k=4000, group=128) == -1
    assert call(xs=4088) == call(xs=4100) == call(ys=4095) == call(x=p + 8) == call(s=p + 4) == -4
    assert call(n=24, epi=1) == call(rows=1 << 21) == -4
    need = lib.hs_linear_int4_workspace_size(64, 4096, 4096, 0)
    assert need > 0 and lib.hs_linear_int4_workspace_size(16, 4096, 4096, 0) == 0
    assert call(rows=64) == call(rows=64, ws=p, ws_bytes=need - 1) == -2
