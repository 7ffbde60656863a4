"""Argument checks of the RMS norm's entry points, which run before any device work (no GPU)."""
import ctypes

import pytest

from glaucis_b200 import _lib

P = ctypes.c_void_p(16)   # never dereferenced: validation fails first
ODD = ctypes.c_void_p(24)


def _err():
    return _lib.load().gl_last_error().decode()


def _fwd(x=P, res=None, w=P, eps=1e-6, M=4, K=256, h=None, y=P, q=None, s=None):
    return _lib.load().gl_rms_norm_fwd(x, res, w, 0, eps, M, K, h, y, q, s, None, None, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(K=100), "multiple of 8"), (dict(K=0), "multiple of 8"),
    (dict(K=16392), "16384"), (dict(M=-1), "M"), (dict(M=1 << 31), "M"), (dict(res=P), "residual"),
    (dict(h=P), "residual"), (dict(q=P), "q and s"), (dict(y=None), "neither"),
    (dict(q=P, s=P, K=264), "128"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(x=ODD), "aligned"), (dict(y=ODD), "aligned"), (dict(w=ODD), "aligned"), (dict(res=P, h=ODD), "aligned"),
])
def test_forward_rejects(kw, msg):
    assert _fwd(**kw) == _lib.GL_EINVAL and msg in _err(), _err()


def test_no_rows_is_no_launch():
    assert _fwd(M=0, x=None, y=None) == _lib.GL_OK
    assert _lib.load().gl_rms_norm_bwd_workspace_bytes(0, 256) == 0
    assert _lib.load().gl_rms_norm_bwd_workspace_bytes(4, 100) == 0


def test_backward_rejects():
    def bwd(dy=P, dh=None, h=P, w=P, M=4, K=256, dx=P, dw=P):
        return _lib.load().gl_rms_norm_bwd(dy, dh, h, w, 0, P, M, K, dx, dw, None, 0, None, None)
    for kw, msg in [(dict(dy=None), "null"), (dict(dw=None), "null"), (dict(K=12), "multiple of 8"),
                    (dict(dx=ODD), "aligned"), (dict(dh=ODD), "aligned")]:
        assert bwd(**kw) == _lib.GL_EINVAL and msg in _err(), _err()
