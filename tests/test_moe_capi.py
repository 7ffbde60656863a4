"""Argument checks of the router's and the exchange's entry points, which run before any device work (no GPU)."""
import ctypes

import pytest

from glaucis_b200 import _lib

P = ctypes.c_void_p(16)   # never dereferenced: validation fails first
ODD = ctypes.c_void_p(24)


def _err():
    return _lib.load().gl_last_error().decode()


def _route(T=4, E=16, k=2, z=P, ids=P, counts=P, ws=P, n=1 << 30):
    return _lib.load().gl_moe_route_fwd(z, 1, None, T, E, k, 1, ids, P, counts, P, P, P, ws, n, None, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=-1), "T"), (dict(T=1 << 31), "T"), (dict(E=0), "E"), (dict(E=1025, k=1), "E"), (dict(k=0), "topk"),
    (dict(k=17), "topk"), (dict(E=64, k=33), "topk"), (dict(T=1 << 30, k=2), "31 bits"), (dict(z=None), "null"),
    (dict(ids=None), "null"), (dict(counts=None), "null"), (dict(T=5000, ws=None), "workspace"), (dict(T=5000, n=16), "workspace"),
    (dict(T=5000, ws=ctypes.c_void_p(18)), "4-byte"),
])
def test_route_rejects(kw, msg):
    assert _route(**kw) == _lib.GL_EINVAL and msg in _err(), _err()


def test_route_workspace_and_backward():
    lib = _lib.load()
    assert lib.gl_moe_route_workspace_bytes(4, 0) == 0 and lib.gl_moe_route_workspace_bytes(4, 2000) == 0
    assert lib.gl_moe_route_workspace_bytes(5000, 128) >= 2 * 128 * 4
    assert lib.gl_moe_route_workspace_bytes(4, 128) == 0  # one CTA takes them all
    bwd = lambda T, E, k, z: lib.gl_moe_route_bwd(z, 1, None, P, P, P, P, None, None, T, E, k, 1, P, None, None)  # noqa: E731
    assert bwd(4, 16, 20, P) == _lib.GL_EINVAL and "topk" in _err()
    assert bwd(4, 16, 2, None) == _lib.GL_EINVAL and "null" in _err()
    assert bwd(0, 16, 2, None) == _lib.GL_OK


def _dispatch(x=P, rb=256, s=None, sc=0, pos=P, gs=P, G=8, T=4, k=2, rows=8, out=P, out_s=None):
    return _lib.load().gl_moe_dispatch(x, rb, s, sc, pos, gs, G, T, k, rows, out, out_s, None, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(rb=0), "row_bytes"), (dict(rb=24), "row_bytes"), (dict(x=None), "null"), (dict(pos=None), "null"),
    (dict(gs=None), "null"), (dict(out=None), "null"), (dict(G=0), "G"), (dict(G=1025), "G"), (dict(T=-1), "T"),
    (dict(k=33), "topk"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(s=P, sc=0), "scales"),
    (dict(s=P, sc=2), "together"), (dict(sc=2, out_s=P), "together"), (dict(x=ODD), "aligned"),
    (dict(out=ODD), "aligned"), (dict(T=1 << 30, k=4), "2^31"),
])
def test_dispatch_rejects(kw, msg):
    assert _dispatch(**kw) == _lib.GL_EINVAL and msg in _err(), _err()


def test_dispatch_and_combine_of_nothing_launch_nothing():
    assert _dispatch(T=0, rows=0, x=None, pos=None, out=None) == _lib.GL_OK
    assert _combine(T=0, y=None, out=None) == _lib.GL_OK


def _combine(y=P, pos=P, res=None, T=4, k=2, K=256, rows=8, out=P):
    return _lib.load().gl_moe_combine(y, 0, pos, None, res, T, k, K, rows, out, None, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(K=100), "multiple of 8"), (dict(K=16392), "16384"), (dict(y=None), "null"), (dict(pos=None), "null"),
    (dict(out=None), "null"), (dict(res=ODD), "aligned"), (dict(y=ODD), "aligned"), (dict(k=0), "topk"),
])
def test_combine_rejects(kw, msg):
    assert _combine(**kw) == _lib.GL_EINVAL and msg in _err(), _err()


def test_combine_backward_rejects():
    def bwd(dout=P, K=256, G=8, dy=P, T=4):
        return _lib.load().gl_moe_combine_bwd(dout, P, 0, P, P, P, G, T, 2, K, 8, dy, P, None, None)
    for kw, msg in [(dict(dout=None), "null"), (dict(dy=None), "null"), (dict(K=4), "multiple of 8"), (dict(G=0), "G"),
                    (dict(dout=ODD), "aligned"), (dict(T=-2), "T")]:
        assert bwd(**kw) == _lib.GL_EINVAL and msg in _err(), _err()
