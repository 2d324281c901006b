"""Refusals of the 8-bit cache's entry points (host checks: no GPU is touched) and of their
torch wrappers."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def ptr():
    buf = ctypes.create_string_buffer(4096 + 64)
    base = ctypes.addressof(buf)
    yield (base + 63) // 64 * 64
    del buf


def test_store_refusals(hv, ptr):
    lib = hv._lib.lib()

    def call(key=ptr, scales=ptr, st=256, csb=256 * 256, group=32, n=3, heads=2, d=128, bs=256,
             nb=4, slots=ptr):
        return lib.hs_store_kvcache_scaled(key, st, 128, ptr, st, 128, ptr, ptr, csb, 256, 128,
                                           scales, ptr, 16, 2, 1, group, slots, n, heads, d, bs,
                                           nb, None)

    assert call(n=0, key=None) == 0
    assert call(key=None) == call(scales=None) == call(slots=None) == -1
    assert call(n=-1) == call(heads=0) == call(bs=0) == call(nb=0) == call(group=0) == -1
    assert call(group=96) == -1  # does not divide the block
    assert call(bs=48, group=48) == call(bs=512, group=512) == call(group=16) == -4
    assert call(d=64) == -4
    assert call(st=252) == call(key=ptr + 8) == call(csb=100) == -4
    assert call(scales=ptr + 2) == -4


def test_attention_refusals(hv, ptr):
    lib = hv._lib.lib()

    def call(q=ptr, bt=ptr, scales=ptr, qst=4096, csb=256 * 1024, cst=1024, group=32, width=8,
             bt_stride=8, nb=4, B=1, mq=4, mk=320, hq=32, hkv=8, d=128, bs=256, ws=ptr,
             ws_bytes=1 << 30):
        return lib.hs_verify_attention_scaled(
            q, qst, 128, ptr, ptr, csb, cst, 128, scales, ptr, 64, 8, 1, group, bt, bt_stride,
            width, nb, ptr, ptr, B, mq, mk, hq, hkv, d, bs, 0.1, ptr, 4096, 128, ws, ws_bytes,
            None)

    assert call(q=None) == call(bt=None) == call(scales=None) == -1
    assert call(B=0) == call(mq=0) == call(mk=0) == call(nb=0) == call(width=0) == -1
    assert call(bt_stride=4) == call(hq=20) == call(group=96) == -1
    assert call(d=64) == call(bs=16, group=16) == call(hq=32, hkv=1) == -4
    assert call(qst=4100) == call(csb=1000) == call(cst=1 << 26) == call(q=ptr + 8) == -4
    assert call(B=65536) == -4
    need = lib.hs_verify_attention_scaled_workspace_size(1, 32, 8, 4, 40960)
    assert need > 0
    assert call(mk=40960, ws_bytes=need - 1) == call(mk=40960, ws=None) == -2
    assert lib.hs_verify_attention_scaled_workspace_size(0, 32, 8, 4, 320) == 0


def test_wrappers_refuse_what_is_not_such_a_cache(hv):
    ops = hv.ops
    c = torch.zeros(2, 256, 2, 128).to(torch.float8_e4m3fn)
    s = torch.zeros(2, 8, 2)
    assert ops._scaled_cache(c, c, s, s)[3] == 32
    with pytest.raises(TypeError):
        ops._scaled_cache(c.to(torch.bfloat16), c, s, s)
    with pytest.raises(TypeError):
        ops._scaled_cache(c, c, s.double(), s)
    for bad in (s[:1], s[:, :, :1], torch.zeros(2, 7, 2), s[:, :0], torch.zeros(2, 16, 2)[:, ::2]):
        with pytest.raises(ValueError):
            ops._scaled_cache(c, c, s, bad)
    with pytest.raises(ValueError):
        ops._scaled_cache(c, c[:, :128], s, s)
    with pytest.raises(ValueError):  # not on a GPU
        ops.store_kvcache_scaled(torch.zeros(1, 2, 128), torch.zeros(1, 2, 128), c, c, s, s,
                                 torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.verify_attention_scaled(torch.zeros(1, 4, 128), c, c, s, s,
                                    torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2),
                                    torch.zeros(2), 1, 1, 1.0)
