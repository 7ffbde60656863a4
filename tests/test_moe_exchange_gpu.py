"""Rows into expert order and back, and their gradients, against indexing in 64 bits.

Dispatch copies: equal bit for bit.  A combine rounds its product-sums in
fp32, at most 2 (k + 1) half-ulps (2^-24) of the terms' magnitudes, then once
to bf16 (2^-8).  A weight's gradient is a sum over K features: at most
K / 256 terms a thread in vectors of 8, then 13 additions of a tree."""
import pytest
import torch

from glaucis_b200 import _lib, ops

pytestmark = pytest.mark.gpu

BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
U, HALF_BF16 = 2.0 ** -24, 2.0 ** -8


def _routing(cuda, T, E, k, seed, drop=0.0):
    """pos and group_sizes of random distinct choices; a share of them dropped."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    ids = torch.rand((T, E), generator=g, device=cuda).argsort(1)[:, :k]
    gone = torch.rand((T, k), generator=g, device=cuda) < drop
    flat = torch.where(gone, E, ids).reshape(-1)
    order = torch.sort(flat, stable=True).indices
    pos = torch.empty_like(flat)
    pos[order] = torch.arange(flat.numel(), device=cuda)
    pos = torch.where(flat == E, -1, pos).int().reshape(T, k)
    return pos, torch.bincount(flat, minlength=E + 1)[:E].int()


def _rand(cuda, *shape, seed=0, dtype=BF16):
    return torch.randn(shape, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).to(dtype)


SHAPES = [(1, 8, 1, 8), (1, 128, 8, 7168), (4, 128, 8, 7168), (37, 60, 4, 264), (130, 8, 2, 1024), (65, 64, 6, 2056),
          (700, 256, 8, 512), (9, 40, 32, 4096), (2100, 8, 2, 4096), (3, 16, 3, 16384),
          (600, 12, 3, 264), (650, 8, 2, 5120), (601, 8, 1, 16)]


@pytest.mark.parametrize("T,E,k,K", SHAPES)
@pytest.mark.parametrize("drop,extra", [(0.0, 0), (0.2, 0), (0.2, 77)])
def test_dispatch(cuda, T, E, k, K, drop, extra):
    pos, sizes = _routing(cuda, T, E, k, seed=T, drop=drop)
    rows = T * k + extra
    t, j = torch.nonzero(pos >= 0, as_tuple=True)
    for dtype in (BF16, F32):
        x = _rand(cuda, T, K, seed=1, dtype=dtype)
        want = torch.zeros((rows, K), dtype=dtype, device=cuda)
        want[pos[t, j].long()] = x[t]
        out = torch.full((rows, K), float("nan"), dtype=dtype, device=cuda)
        assert ops.moe_dispatch_fwd(x, pos, sizes, rows, out=out) is out
        assert torch.equal(out, want)
    if K % 128 == 0:
        q = (_rand(cuda, T, K, seed=2, dtype=F32) * 50).to(E4M3)
        s = _rand(cuda, T, K // 128, seed=3, dtype=F32).abs()
        a_q, a_s = ops.moe_dispatch_quant(q, s, pos, sizes, rows)
        wq = torch.zeros((rows, K), dtype=torch.uint8, device=cuda)
        ws = torch.ones((rows, K // 128), device=cuda)
        wq[pos[t, j].long()] = q.view(torch.uint8)[t]
        ws[pos[t, j].long()] = s[t]
        assert torch.equal(a_q.view(torch.uint8), wq) and torch.equal(a_s, ws)
    assert ops.device_status() == 0


@pytest.mark.parametrize("T,E,k,K", SHAPES)
@pytest.mark.parametrize("f32,residual,drop", [(False, True, 0.2), (True, False, 0.0), (True, True, 0.2)])
def test_combine_and_its_gradients(cuda, T, E, k, K, f32, residual, drop):
    pos, sizes = _routing(cuda, T, E, k, seed=T + 1, drop=drop)
    rows = T * k + 5
    y = _rand(cuda, rows, K, seed=4, dtype=F32 if f32 else BF16)
    y[int(sizes.sum()):] = float("nan")  # rows of no group are of no meaning
    w = torch.softmax(_rand(cuda, T, k, seed=5, dtype=F32), 1)
    w = torch.where(pos < 0, float("nan"), w)  # nor are weights without a row
    res = _rand(cuda, T, K, seed=6) if residual else None
    dout = _rand(cuda, T, K, seed=7)
    t, j = torch.nonzero(pos >= 0, as_tuple=True)
    at, wt = pos[t, j].long(), w[t, j].to(F64)[:, None]
    base = res.to(F64) if residual else torch.zeros((T, K), dtype=F64, device=cuda)
    ref = base.index_add(0, t, y.to(F64)[at] * wt)
    mag = base.abs().index_add(0, t, (y.to(F64)[at] * wt).abs())
    out = ops.moe_combine_fwd(y, pos, w, residual=res)
    assert ((out.to(F64) - ref).abs() <= HALF_BF16 * ref.abs() + 2 * (k + 1) * U * mag).all()

    dy, dw = ops.moe_combine_bwd(dout, y, pos, w, sizes)
    ref_dy = torch.zeros((rows, K), dtype=F64, device=cuda)
    ref_dy[at] = dout.to(F64)[t] * wt
    assert ((dy.to(F64) - ref_dy).abs() <= (U if f32 else HALF_BF16 + U) * ref_dy.abs()).all()
    prod = y.to(F64)[at] * dout.to(F64)[t]
    ref_dw = torch.zeros((T, k), dtype=F64, device=cuda)
    tol = torch.zeros((T, k), dtype=F64, device=cuda)
    ref_dw[t, j] = prod.sum(1)
    tol[t, j] = (K / 256 + 8 + 13) * U * prod.abs().sum(1)
    assert ((dw.to(F64) - ref_dw).abs() <= tol).all()

    # the dispatch's gradient: a token's rows added up
    dxs = torch.where(torch.isnan(y), 0, y)
    dx = ops.moe_dispatch_bwd(dxs, pos)
    ref = torch.zeros((T, K), dtype=F64, device=cuda).index_add(0, t, dxs.to(F64)[at])
    mag = torch.zeros((T, K), dtype=F64, device=cuda).index_add(0, t, dxs.to(F64)[at].abs())
    assert ((dx.to(F64) - ref).abs() <= HALF_BF16 * ref.abs() + (k + 1) * U * mag).all()
    assert ops.device_status() == 0


def test_gradients_against_differences(cuda):
    T, E, k, K = 12, 8, 2, 256
    pos, sizes = _routing(cuda, T, E, k, seed=3)
    y, w = _rand(cuda, T * k, K, dtype=F32), torch.softmax(_rand(cuda, T, k, seed=1, dtype=F32), 1)
    dout = _rand(cuda, T, K, seed=2)
    dy, dw = ops.moe_combine_bwd(dout, y, pos, w, sizes)
    dirs = _rand(cuda, T * k, K, seed=3, dtype=F64), _rand(cuda, T, k, seed=4, dtype=F64)

    def value(yy, ww):
        return ((yy[pos.long()] * ww[:, :, None]).sum(1) * dout.to(F64)).sum()

    y64, w64, h = y.to(F64), w.to(F64), 1e-3  # bilinear: central differences are exact
    for got, d, lo, hi in [(dy, dirs[0], (y64 - h * dirs[0], w64), (y64 + h * dirs[0], w64)),
                           (dw, dirs[1], (y64, w64 - h * dirs[1]), (y64, w64 + h * dirs[1]))]:
        diff = float((value(*hi) - value(*lo)) / (2 * h))
        terms = got.to(F64) * d
        assert abs(diff - float(terms.sum())) <= 1e-5 * float(terms.abs().sum())


def test_autograd(cuda):
    T, E, k, K = 50, 16, 4, 384
    pos, sizes = _routing(cuda, T, E, k, seed=9, drop=0.1)
    x = _rand(cuda, T, K).requires_grad_()
    w = torch.where(pos < 0, 0, torch.softmax(_rand(cuda, T, k, seed=1, dtype=F32), 1)).requires_grad_()
    res = _rand(cuda, T, K, seed=2).requires_grad_()
    xs = ops.moe_dispatch(x, pos, sizes)
    out = ops.moe_combine(xs, pos, w, sizes, residual=res)
    dout = _rand(cuda, T, K, seed=3)
    gx, gw, gr = torch.autograd.grad(out, (x, w, res), dout)
    dy, dw = ops.moe_combine_bwd(dout, xs.detach(), pos, w.detach(), sizes)
    assert torch.equal(gr, dout) and torch.equal(gw, dw)
    assert torch.equal(gx, ops.moe_dispatch_bwd(dy, pos))
    # a gradient that is broadcast, and the residual alone
    out = ops.moe_combine(xs.detach(), pos, w.detach(), sizes, residual=res)
    gr, = torch.autograd.grad(out.sum(), res)
    assert (gr == 1).all()


def test_out_may_be_the_residual(cuda):
    pos, sizes = _routing(cuda, 33, 8, 2, seed=2)
    y, w = _rand(cuda, 66, 512), torch.rand((33, 2), device=cuda)
    res = _rand(cuda, 33, 512, seed=1)
    want = ops.moe_combine_fwd(y, pos, w, residual=res)
    assert torch.equal(ops.moe_combine_fwd(y, pos, w, residual=res, out=res), want)


def test_rows_past_two_billion_elements(cuda):
    # offsets in a long output pass 32 bits: 600,000 rows of 4096 (4.9 GB)
    T, K, rows = 3, 4096, 600_000
    x = _rand(cuda, T, K)
    pos = torch.tensor([[0], [rows - 2], [rows - 1]], dtype=torch.int32, device=cuda)
    sizes = torch.tensor([rows], dtype=torch.int32, device=cuda)
    out = torch.zeros((rows, K), dtype=BF16, device=cuda)
    ops.moe_dispatch_fwd(x, pos, sizes, rows, out=out)
    assert torch.equal(out[pos[:, 0].long()], x)
    back = ops.moe_combine_fwd(out, pos, torch.ones((T, 1), device=cuda))
    assert torch.equal(back, x)
    assert int((out[1:rows - 2].view(torch.int16) != 0).sum()) == 0


def test_no_tokens(cuda):
    pos = torch.empty((0, 4), dtype=torch.int32, device=cuda)
    sizes = torch.zeros(8, dtype=torch.int32, device=cuda)
    x = torch.empty((0, 256), dtype=BF16, device=cuda)
    assert ops.moe_dispatch_fwd(x, pos, sizes).shape == (0, 256)
    assert (ops.moe_dispatch_fwd(x, pos, sizes, 10) == 0).all()
    w = torch.empty((0, 4), device=cuda)
    assert ops.moe_combine_fwd(x, pos, w).shape == (0, 256)
    dy, dw = ops.moe_combine_bwd(x, torch.ones((6, 256), dtype=BF16, device=cuda), pos, w, sizes)
    assert (dy == 0).all() and dw.shape == (0, 4)
    # tokens, none of them routed
    pos = torch.full((5, 2), -1, dtype=torch.int32, device=cuda)
    x = _rand(cuda, 5, 256)
    assert (ops.moe_dispatch_fwd(x, pos, sizes) == 0).all()
    assert torch.equal(ops.moe_combine_fwd(x[:0], pos, torch.ones((5, 2), device=cuda), residual=x), x)
    assert ops.device_status() == 0


def test_bad_rows_and_sizes_are_reported(cuda):
    # the kernels skip such a row themselves and say so in the error word
    T, K, rows = 4, 256, 8
    x, w = _rand(cuda, T, K), torch.ones((T, 2), device=cuda)
    pos = torch.tensor([[0, 1], [2, 8], [4, 5], [6, 2 ** 31 - 1]], dtype=torch.int32, device=cuda)
    sizes = torch.tensor([8], dtype=torch.int32, device=cuda)
    out = torch.zeros((rows, K), dtype=BF16, device=cuda)
    ops.moe_dispatch_fwd(x, pos, sizes, out=out)
    assert ops.device_status() == 3 and ops.device_status() == 0
    assert torch.equal(out[[0, 1, 2, 4, 5, 6]], x[[0, 0, 1, 2, 2, 3]]) and (out[[3, 7]] == 0).all()
    back = ops.moe_combine_fwd(out, pos, w)
    assert ops.device_status() == 3
    assert torch.equal(back[1], x[1]) and torch.equal(back[3], x[3])
    dy, dw = ops.moe_combine_bwd(x, out, pos, w, sizes)
    assert ops.device_status() == 3 and dw[1, 1] == 0 and dw[3, 1] == 0
    ok = torch.tensor([[0, 1], [2, 3], [4, 5], [6, 7]], dtype=torch.int32, device=cuda)
    for bad in ([9], [-1], [4, -2]):
        ops.moe_dispatch_fwd(x, ok, torch.tensor(bad, dtype=torch.int32, device=cuda), out=out)
        assert ops.device_status() == 2
        assert torch.equal(out, x.repeat_interleave(2, 0))


def test_no_tokens_but_rows_of_a_capacity(cuda):
    K, rows, k = 256, 40, 2
    pos = torch.empty((0, k), dtype=torch.int32, device=cuda)
    sizes = torch.zeros(4, dtype=torch.int32, device=cuda)
    q = torch.empty((0, K), dtype=torch.float8_e4m3fn, device=cuda)
    s = torch.empty((0, K // 128), device=cuda)
    out = torch.full((rows, K), float("nan"), device=cuda).to(torch.float8_e4m3fn)
    out_s = torch.full((rows, K // 128), float("nan"), device=cuda)
    ops.moe_dispatch_quant(q, s, pos, sizes, rows, out=out, out_s=out_s)
    assert (out.float() == 0).all() and (out_s == 1).all()
    y = torch.ones((rows, K), device=cuda)
    dy, dw = ops.moe_combine_bwd(torch.empty((0, K), dtype=torch.bfloat16, device=cuda), y, pos,
                                 torch.empty((0, k), device=cuda), sizes)
    assert (dy == 0).all() and dw.shape == (0, k)
    assert ops.device_status() == 0


@pytest.mark.parametrize("T", [1, 3])
def test_few_tokens_in_rows_of_a_capacity(cuda, T):
    # more rows than the choices can fill: the rest is zero, its scales 1
    E, k, K, rows = 8, 2, 512, 5000
    pos, sizes = _routing(cuda, T, E, k, seed=50)
    g = torch.Generator(device=cuda).manual_seed(51)
    x = torch.randn((T, K), generator=g, device=cuda).to(BF16)
    named = pos.reshape(-1).long()
    junk = lambda *s, dtype=BF16: torch.full(s, float("nan"), device=cuda).to(dtype)  # noqa: E731
    out = ops.moe_dispatch_fwd(x, pos, sizes, rows, junk(rows, K))
    assert torch.equal(out[named], x.repeat_interleave(k, 0)) and (out[T * k:] == 0).all()
    q, s = ops.quant_act_1x128(x)
    oq, os_ = ops.moe_dispatch_quant(q, s, pos, sizes, rows, junk(rows, K, dtype=E4M3), junk(rows, K // 128, dtype=F32))
    assert torch.equal(os_[named], s.repeat_interleave(k, 0)) and (os_[T * k:] == 1).all()
    assert torch.equal(oq[named].view(torch.uint8), q.view(torch.uint8).repeat_interleave(k, 0))
    assert (oq[T * k:].float() == 0).all()
    y = torch.randn((rows, K), generator=g, device=cuda).to(BF16)
    w = torch.rand((T, k), generator=g, device=cuda)
    dy, dw = ops.moe_combine_bwd(x, y, pos, w, sizes)
    assert (dy[T * k:] == 0).all()
    assert torch.equal(dy[named], (w.reshape(-1, 1) * x.float().repeat_interleave(k, 0)).to(BF16))
    assert ops.device_status() == 0


def test_refusals(cuda):
    T, K = 4, 256
    x, pos = _rand(cuda, T, K), torch.zeros((T, 2), dtype=torch.int32, device=cuda)
    sizes, w = torch.tensor([8], dtype=torch.int32, device=cuda), torch.ones((T, 2), device=cuda)
    y = _rand(cuda, 8, K)
    with pytest.raises(ValueError, match="x must be"):
        ops.moe_dispatch(x[:2], pos, sizes)
    with pytest.raises(ValueError, match="x must be"):
        ops.moe_dispatch(x.half(), pos, sizes)
    with pytest.raises(ValueError, match="pos"):
        ops.moe_dispatch(x, pos.long(), sizes)
    with pytest.raises(ValueError, match="group_sizes"):
        ops.moe_dispatch(x, pos, sizes.long())
    with pytest.raises(ValueError, match="s must be"):
        ops.moe_dispatch_quant(x.to(E4M3), w[:2], pos, sizes)
    with pytest.raises(ValueError, match="weights"):
        ops.moe_combine(y, pos, w.to(BF16), sizes)
    with pytest.raises(ValueError, match="residual"):
        ops.moe_combine(y, pos, w, sizes, residual=x[:2])
    with pytest.raises(ValueError, match="dout"):
        ops.moe_combine_bwd(x[:2], y, pos, w, sizes)
    with pytest.raises(ValueError, match="out must"):
        ops.moe_dispatch_fwd(x, pos, sizes, out=y[:4])
    with pytest.raises(_lib.GlaucisError, match="multiple of 16"):
        ops.moe_dispatch(x[:, :100].contiguous(), pos, sizes)
    with pytest.raises(_lib.GlaucisError, match="multiple of 8"):
        ops.moe_combine(y[:, :100].contiguous(), pos, w, sizes)
    with pytest.raises(_lib.GlaucisError, match="topk"):
        ops.moe_dispatch(x, torch.zeros((T, 33), dtype=torch.int32, device=cuda), sizes)
    with pytest.raises(ValueError, match="takes bf16"):
        ops.moe_dispatch(x.float().requires_grad_(), pos, sizes)
    with pytest.raises(ValueError, match="at most 16384"):  # which its gradient could not take
        ops.moe_dispatch(_rand(cuda, T, 16512).requires_grad_(), pos, sizes)
