"""The training entry points of the C ABI reject malformed arguments on the host, before any
CUDA call (no GPU needed)."""
import ctypes

import pytest

from tensorcx_b200 import _abi

B = ctypes.c_void_p(1024)  # stands for a buffer; every call below is refused before it is read
INF, NAN = float("inf"), float("nan")


def norm(x=B, y=B, total=B, mean=B, rows=4, cols=8, eps=1e-5, p=0.0, residual=None):
    return _abi.lib().tcx_sm100_layernorm_forward(None, x, residual, None, None, y, total, mean, B, rows, cols, eps, p,
                                                  0, 0, None)


def norm_back(dx=B, dw=B, db=B, rows=4, cols=8, p=0.0, ws=None, ws_bytes=0, dres=B):
    return _abi.lib().tcx_sm100_layernorm_backward(None, B, B, B, B, None, None, dres, dx, dw, db, rows, cols, p, 0, 0,
                                                   None, ws, ws_bytes)


def rec(form=0, gate=B, h=B, batch=2, time=3, channels=4, ws=None, ws_bytes=0):
    return _abi.lib().tcx_sm100_recurrence_forward(None, form, gate, B, None, None, h, None, batch, time, channels, ws,
                                                   ws_bytes)


def rec_back(form=0, x=B, h=B, dx=B, batch=2, time=3, channels=4):
    return _abi.lib().tcx_sm100_recurrence_backward(None, form, B, B, x, h, None, None, None, B, dx, None, batch, time,
                                                    channels, None, 0)


def drop(x=B, out=B, count=4, p=0.5):
    return _abi.lib().tcx_sm100_dropout(None, x, None, out, count, p, 0, 0, None)


@pytest.mark.parametrize("call,word", [
    (lambda: drop(count=-1), b"negative"), (lambda: drop(p=-0.1), b"probability"),
    (lambda: drop(p=1.1), b"probability"), (lambda: drop(p=NAN), b"probability"), (lambda: drop(x=None), b"buffer"), (lambda: drop(out=None), b"buffer"),
    (lambda: norm(rows=-1), b"negative"), (lambda: norm(cols=0), b"non-empty"), (lambda: norm(eps=-1.0), b"epsilon"),
    (lambda: norm(eps=NAN), b"epsilon"), (lambda: norm(eps=INF), b"epsilon"), (lambda: norm(p=2.0), b"probability"),
    (lambda: norm(x=None), b"buffer"), (lambda: norm(mean=None), b"buffer"),
    (lambda: norm(total=None, residual=B), b"total"), (lambda: norm(total=None, p=0.5), b"total"),
    (lambda: norm(rows=1 << 40, cols=1 << 40), b"overflows"),
    (lambda: norm_back(rows=-1), b"negative"), (lambda: norm_back(db=None), b"together"),
    (lambda: norm_back(dx=None, p=0.5), b"dropout"), (lambda: norm_back(dres=None), b"buffer"),
    (lambda: norm_back(p=NAN), b"probability"), (lambda: norm_back(), b"workspace"),
    (lambda: norm_back(ws_bytes=1 << 30), b"workspace"), (lambda: rec(time=300), b"workspace"),
    (lambda: rec(time=300, ws_bytes=1 << 30), b"workspace"),
    (lambda: rec(time=300, ws=ctypes.c_void_p(1028), ws_bytes=1 << 30), b"aligned"),
    (lambda: rec(form=2), b"form"), (lambda: rec(batch=-1), b"negative"), (lambda: rec(gate=None), b"buffer"),
    (lambda: rec(h=None), b"buffer"), (lambda: rec(batch=1 << 30, time=1 << 30, channels=1 << 30), b"overflows"),
    (lambda: rec_back(form=-1), b"form"), (lambda: rec_back(form=1, x=None), b"needs x"),
    (lambda: rec_back(h=None), b"buffer"), (lambda: rec_back(dx=None), b"buffer"),
])
def test_refusals(call, word):
    assert call() == _abi.INVALID_ARGUMENT
    assert word in _abi.lib().tcx_sm100_last_error(), _abi.lib().tcx_sm100_last_error()


def test_nothing_to_do():
    lib = _abi.lib()
    assert lib.tcx_sm100_dropout(None, None, None, None, 0, 0.5, 0, 0, None) == _abi.OK
    assert norm(rows=0) == _abi.OK
    assert rec(batch=0) == _abi.OK and rec(channels=0) == _abi.OK and rec_back(batch=0) == _abi.OK
    assert lib.tcx_sm100_layernorm_backward_workspace_bytes(0, 8) == 0
    assert lib.tcx_sm100_layernorm_backward_workspace_bytes(1000, 4096) >= 2 * 4096 * 4
