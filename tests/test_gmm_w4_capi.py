"""Argument checks of the 4-bit products' entry points, which run before any device work (no GPU)."""
import ctypes

import pytest

from glaucis_b200 import _lib

P = ctypes.c_void_p(16)   # never dereferenced: validation fails first
ODD = ctypes.c_void_p(24)


def _err():
    return _lib.load().gl_last_error().decode()


def _gmm(x=P, w=P, s=P, gs=P, G=4, M=8, K=256, N=64, out=P, dt=0, flags=0, ws=P, n=1 << 30):
    return _lib.load().gl_gmm_w4_fwd(x, w, s, gs, G, M, K, N, out, dt, flags, ws, n, None, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(gs=None), "null"), (dict(out=None), "null"),
    (dict(G=0), "G"), (dict(G=1025), "G"), (dict(K=200), "128"), (dict(N=48), "32"), (dict(M=-1), "M"),
    (dict(M=65537), "rows"), (dict(dt=5), "out_dtype"), (dict(flags=2), "flags"), (dict(x=ODD), "aligned"),
    (dict(s=ODD), "aligned"), (dict(ws=None), "workspace"), (dict(ws=ODD), "aligned"),
])
def test_product_rejects(kw, msg):
    assert _gmm(**kw) == _lib.GL_EINVAL and msg in _err(), _err()


def test_workspace_and_quantiser():
    lib = _lib.load()
    assert lib.gl_gmm_w4_workspace_bytes(8, 200) == 0
    assert lib.gl_gmm_w4_workspace_bytes(0, 256) == 0
    assert _gmm(M=0, x=None, out=None, ws=None) == _lib.GL_OK
    q = lambda w, G, K, N: lib.gl_quant_w4_128x1(w, G, K, N, P, P, None, None)  # noqa: E731
    for args, msg in [((None, 1, 128, 32), "null"), ((P, 0, 128, 32), "G"), ((P, 1, 100, 32), "128"),
                      ((P, 1, 128, 16), "32"), ((ODD, 1, 128, 32), "aligned")]:
        assert q(*args) == _lib.GL_EINVAL and msg in _err(), _err()
