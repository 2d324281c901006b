"""Refusals of the log-probabilities' entry points (host checks: no GPU is touched)."""
import ctypes

import pytest
import torch


def test_refusals(hv):
    lib = hv._lib.lib()
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 63) // 64 * 64

    def call(x=p, dtype=1, stride=1000, rows=2, V=1000, tokens=p, temps=None, top=5, lp=p, ent=p,
             ids=p, tlp=p, ws=p, ws_bytes=1 << 30):
        return lib.hs_token_logprobs(x, dtype, stride, rows, V, tokens, temps, top, lp, ent, ids,
                                     tlp, ws, ws_bytes, None)

    assert call(rows=0, x=None) == 0
    assert call(x=None) == call(rows=-1) == call(V=0) == call(dtype=2) == call(stride=999) == -1
    assert call(top=33) == call(top=-1) == call(V=4, top=5) == -1
    assert call(tokens=None) == call(lp=None) == call(ids=None) == call(tlp=None) == -1
    assert call(rows=65536) == call(V=(1 << 21) + 1, stride=1 << 22) == call(x=p + 1) == -4
    need = lib.hs_token_logprobs_workspace_size(2, 1000, 5)
    assert need > 0 and lib.hs_token_logprobs_workspace_size(2, 1000, 33) == 0
    assert call(ws=None) == call(ws_bytes=need - 1) == -2
    assert call(ws=p + 8) == -4


def test_wrapper_refusals(hv):
    with pytest.raises(ValueError):  # not on a GPU
        hv.ops.token_logprobs(torch.zeros(2, 10))
