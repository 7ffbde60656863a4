"""RMS norm with the residual's addition: outputs, 8-bit pair and gradients
against the formulas in 64 bits.

Tolerances.  A row's sum of squares is held in fp32: at most 16 terms a
thread, then 10 additions of a tree, so it is off by at most 27 half-ulps
(27 * 2^-24 = 1.6e-6 relative), its inverse root by half of that, and rsqrtf,
the two products and a division add at most 5 * 2^-23: F32 = 2e-6 bounds what
the norm is off before its one rounding.  That rounding adds half a step of
the output's type (bf16 2^-8, e4m3 2^-4 or half its smallest subnormal 2^-10).
A gradient's terms each carry F32 twice (the norm again, and the row's mean),
a weight gradient one more rounding for each row that one CTA sums."""
import pytest
import torch

from glaucis_b200 import _lib, ops

pytestmark = pytest.mark.gpu

BF16, F32T, F64 = torch.bfloat16, torch.float32, torch.float64
F32, HALF_BF16, HALF_E4M3, SUB_E4M3 = 2e-6, 2.0 ** -8, 2.0 ** -4, 2.0 ** -10
EPS = 1e-6


def _inputs(cuda, M, K, residual, w32, seed=0, scale=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    x = (r(M, K) * scale).to(BF16)
    res = (r(M, K) * 2 * scale).to(BF16) if residual else None
    w = (1 + 0.2 * r(K)).to(F32T if w32 else BF16)
    return x, res, w, (r(M, K) * 0.1).to(BF16), (r(M, K) * 0.1).to(BF16)


def _norm64(h, w, eps=EPS):
    h, w = h.to(F64), w.to(F64)
    rstd = 1 / (h.square().mean(1) + eps).sqrt()
    return h * rstd[:, None] * w, rstd


def _within(got, ref, tol, what):
    err = (got.to(F64) - ref).abs()
    assert torch.isfinite(err).all(), what
    bad = err > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max())}"


def _check_pair(q, s, y, K):
    blocks = y.reshape(y.shape[0], K // 128, 128)
    ref_s = blocks.abs().amax(2) / 448
    ref_s = torch.where(ref_s == 0, 1.0, ref_s)
    _within(s, ref_s, F32 * ref_s, "scales")
    deq = q.to(F64).reshape(blocks.shape) * s.to(F64)[:, :, None]
    tol = (HALF_E4M3 * blocks.abs() + SUB_E4M3 * ref_s[:, :, None]) * (1 + 1e-3)
    _within(deq, blocks, tol, "q * s")


SHAPES = [(1, 8), (3, 128), (37, 264), (8, 256), (9, 512), (5, 1024), (2, 1032), (300, 1920), (1, 7168),
          (33, 7168), (700, 4096), (2, 16384)]


@pytest.mark.parametrize("M,K", SHAPES)
@pytest.mark.parametrize("residual,w32", [(False, False), (True, False), (True, True)])
def test_forward(cuda, M, K, residual, w32):
    x, res, w, _, _ = _inputs(cuda, M, K, residual, w32)
    quant = K % 128 == 0
    f = ops.rms_norm_fwd(x, w, EPS, residual=res, output_quant=quant)
    if residual:
        assert torch.equal(f.h, (x.float() + res.float()).to(BF16))
    else:
        assert f.h is x
    y, rstd = _norm64(f.h, w)
    _within(f.y, y, (HALF_BF16 + 2 * F32) * y.abs(), "y")
    _within(f.rstd, rstd, F32 * rstd, "rstd")
    if quant:
        _check_pair(f.q, f.s, y, K)
        pair = ops.rms_norm_quant_1x128(x, w, EPS, residual=res)
        assert torch.equal(pair[0].view(torch.uint8), f.q.view(torch.uint8)) and torch.equal(pair[1], f.s)
        assert len(pair) == (3 if residual else 2)
        if residual:
            assert torch.equal(pair[2], f.h)


@pytest.mark.parametrize("M,K", [s for s in SHAPES] + [(5000, 512), (4099, 1536)])
@pytest.mark.parametrize("residual,w32", [(False, True), (True, False), (True, True)])
def test_backward(cuda, M, K, residual, w32):
    x, res, w, dy, dh = _inputs(cuda, M, K, residual, w32, seed=1)
    f = ops.rms_norm_fwd(x, w, EPS, residual=res)
    dx, dw = ops.rms_norm_bwd(dy, f.h, w, f.rstd, dh=dh if residual else None)
    h, w64, g = f.h.to(F64), w.to(F64), dy.to(F64)
    r = 1 / (h.square().mean(1, keepdim=True) + EPS).sqrt()
    u, xh = g * w64, h * r
    c = (u * xh).mean(1, keepdim=True)
    ref = r * (u - xh * c)
    terms = r * (u.abs() + xh.abs() * (u * xh).abs().mean(1, keepdim=True))
    if residual:
        ref = ref + dh.to(F64)
        terms = terms + dh.to(F64).abs()
    _within(dx, ref, HALF_BF16 * ref.abs() + 3 * F32 * terms, "dx")
    assert dw.dtype == w.dtype
    ref_w = (g * xh).sum(0)
    # at most ceil(M / 148) rows in one running sum, then 32 + 32 shares
    per_row = (-(-M // 148) + 64) * 2.0 ** -24 + 2 * F32
    tol = per_row * (g * xh).abs().sum(0) + (0 if w32 else HALF_BF16 * ref_w.abs())
    _within(dw, ref_w, tol, "dw")


def test_gradients_against_differences(cuda):
    M, K = 6, 384
    x, res, w, dy, dh = _inputs(cuda, M, K, True, True, seed=2)
    f = ops.rms_norm_fwd(x, w, EPS, residual=res)
    dx, dw = ops.rms_norm_bwd(dy, f.h, w, f.rstd, dh=dh)
    g = torch.Generator(device=cuda).manual_seed(3)
    d = torch.randn((M, K), generator=g, device=cuda, dtype=F64)
    e = torch.randn(K, generator=g, device=cuda, dtype=F64)

    def loss(h, wt):
        return (_norm64(h, wt)[0] * dy.to(F64)).sum() + (h * dh.to(F64)).sum()

    h, w64, t = f.h.to(F64), w.to(F64), 1e-5
    by_x = (loss(h + t * d, w64) - loss(h - t * d, w64)) / (2 * t)
    by_w = (loss(h, w64 + t * e) - loss(h, w64 - t * e)) / (2 * t)
    # the differences' own error is of t^2 and 2^-52 / t: below 1e-9 here
    assert abs(float((dx.to(F64) * d).sum() - by_x)) <= HALF_BF16 * float((dx.to(F64) * d).abs().sum())
    assert abs(float((dw.to(F64) * e).sum() - by_w)) <= 1e-5 * float((dw.to(F64) * e).abs().sum())


def test_weight_gradient_is_the_same_every_time(cuda):
    x, _, w, dy, _ = _inputs(cuda, 3000, 768, False, True, seed=4)
    f = ops.rms_norm_fwd(x, w)
    first = ops.rms_norm_bwd(dy, x, w, f.rstd)[1]
    for _ in range(3):
        assert torch.equal(ops.rms_norm_bwd(dy, x, w, f.rstd)[1], first)


@pytest.mark.parametrize("K", [256, 2048])
def test_rows_of_zeros_infinities_and_nan(cuda, K):
    x, _, w, _, _ = _inputs(cuda, 12, K, False, False, seed=5)
    clean = ops.rms_norm_fwd(x, w, EPS, output_quant=True)
    x = x.clone()
    x[2] = 0
    x[5, 3] = float("inf")
    x[7, 1] = float("nan")
    x[9] = 1e-30  # squares below fp32's range: eps alone
    f = ops.rms_norm_fwd(x, w, EPS, output_quant=True)
    others = [r for r in range(12) if r not in (2, 5, 7, 9)]
    assert torch.equal(f.y[others], clean.y[others]) and torch.equal(f.s[others], clean.s[others])
    assert (f.y[2] == 0).all() and (f.q[2].float() == 0).all() and (f.s[2] == 1).all()
    # an infinity: its row's inverse root is 0, itself inf * 0
    assert torch.isnan(f.y[5, 3]) and (f.y[5, :3] == 0).all() and (f.y[5, 4:] == 0).all()
    assert torch.isnan(f.y[7]).all() and torch.isnan(f.q[7].float()).all()
    y9 = _norm64(x[9:10], w)[0]
    _within(f.y[9:10], y9, (HALF_BF16 + 2 * F32) * y9.abs(), "tiny row")
    _check_pair(f.q[9:10], f.s[9:10], y9, K)


def test_tiny_outputs_divide(cuda):
    # scales whose reciprocal is past fp32's range take the division per element
    K = 256
    x = torch.randn((4, K), device=cuda, generator=torch.Generator(device=cuda).manual_seed(6)).to(BF16)
    w = torch.full((K,), 2.0 ** -110, device=cuda)
    q, s = ops.rms_norm_quant_1x128(x, w, EPS)
    _check_pair(q, s, _norm64(x, w)[0], K)


@pytest.mark.parametrize("M,K", [(64, 128), (9, 256), (33, 1024), (3, 2048), (40, 7168), (2, 16384)])
@pytest.mark.parametrize("residual,w32", [(False, True), (True, False), (True, True)])
def test_pair_is_the_rounded_quotient(cuda, M, K, residual, w32):
    # y as the kernel has it, in 32 bits: two rounded products with its own rstd.
    # From there the pair is the activation quantiser's, byte for byte: the scale
    # a correctly rounded quotient and q = e4m3(y / s) of another one.
    x, res, w, _, _ = _inputs(cuda, M, K, residual, w32, seed=12)
    x[0, ::5], w[3::7] = -0.0, 0.0
    f = ops.rms_norm_fwd(x, w, EPS, residual=res, output_quant=True)
    y = (f.h.float() * f.rstd[:, None]) * w.float()
    b = y.reshape(M, K // 128, 128)
    s = (b.abs().amax(2).double() / 448).float()
    s = torch.where(s == 0, 1.0, s)
    assert torch.equal(f.s, s)
    q = (b.double() / s.double()[:, :, None]).float().to(torch.float8_e4m3fn).reshape(M, K)
    assert torch.equal(f.q.view(torch.uint8), q.view(torch.uint8))


def test_sum_may_replace_an_input(cuda):
    x, res, w, _, _ = _inputs(cuda, 50, 2048, True, False, seed=7)
    q, s, h = ops.rms_norm_quant_1x128(x, w, residual=res)
    stream = res.clone()
    q2, s2, h2 = ops.rms_norm_quant_1x128(x, w, residual=stream, h=stream)
    assert h2 is stream and torch.equal(stream, h) and torch.equal(s2, s)
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8))


def test_autograd(cuda):
    x, res, w, dy, dh = _inputs(cuda, 21, 640, True, False, seed=8)
    x.requires_grad_(), res.requires_grad_(), w.requires_grad_()
    y, h = ops.rms_norm(x, w, residual=res)
    f = ops.rms_norm_fwd(x.detach(), w.detach(), residual=res.detach())
    assert torch.equal(y, f.y) and torch.equal(h, f.h)
    gx, gw, gr = torch.autograd.grad((y, h), (x, w, res), (dy, dh), retain_graph=True)
    dx, dw = ops.rms_norm_bwd(dy, f.h, w.detach(), f.rstd, dh=dh)
    assert torch.equal(gx, dx) and torch.equal(gr, dx) and torch.equal(gw, dw)
    # a gradient that reaches only one of the two outputs; one that is broadcast
    gx, = torch.autograd.grad(h, x, dh, retain_graph=True)
    assert torch.equal(gx, dh)
    gx, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(gx, ops.rms_norm_bwd(torch.ones_like(dy), f.h, w.detach(), f.rstd)[0])
    z = ops.rms_norm(x, w)
    assert z.requires_grad and torch.equal(z, ops.rms_norm_fwd(x.detach(), w.detach()).y)


def test_no_rows(cuda):
    x, res, w, _, _ = _inputs(cuda, 0, 256, True, True)
    q, s, h = ops.rms_norm_quant_1x128(x, w, residual=res)
    assert q.shape == (0, 256) and s.shape == (0, 2) and h.shape == (0, 256)
    f = ops.rms_norm_fwd(x, w, residual=res)
    dx, dw = ops.rms_norm_bwd(x, f.h, w, f.rstd)
    assert dx.shape == (0, 256) and (dw == 0).all()


def test_rows_of_a_larger_tensor_and_another_stream(cuda):
    x, _, w, _, _ = _inputs(cuda, 40, 512, False, False, seed=9)
    want = ops.rms_norm_fwd(x[7:20].clone(), w).y
    assert torch.equal(ops.rms_norm_fwd(x[7:20], w).y, want)
    out = torch.full((40, 512), 3.0, dtype=BF16, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.rms_norm_fwd(x[7:20], w, y=out[7:20])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out[7:20], want) and (out[:7] == 3).all() and (out[20:] == 3).all()


def test_offsets_past_32_bits(cuda):
    M, K = 600_000, 4096  # 2.46e9 elements
    x = torch.ones((M, K), dtype=BF16, device=cuda)
    tail, _, w, _, _ = _inputs(cuda, 200, K, False, True, seed=10)
    x[-200:] = tail
    q, s = ops.rms_norm_quant_1x128(x, w)
    want_q, want_s = ops.rms_norm_quant_1x128(tail, w)
    assert torch.equal(q[-200:].view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s[-200:], want_s)
    del q, s
    f = ops.rms_norm_fwd(x, w)
    want = ops.rms_norm_fwd(tail, w)
    assert torch.equal(f.y[-200:], want.y) and torch.equal(f.rstd[-200:], want.rstd)
    dx, _ = ops.rms_norm_bwd(f.y, f.h, w, f.rstd)
    assert torch.equal(dx[-200:], ops.rms_norm_bwd(want.y, tail, w, want.rstd)[0])


def test_refusals(cuda):
    x, res, w, dy, _ = _inputs(cuda, 4, 256, True, False)
    with pytest.raises(ValueError, match="2-D bf16"):
        ops.rms_norm_fwd(x.float(), w)
    with pytest.raises(ValueError, match="weight"):
        ops.rms_norm_fwd(x, w[:128])
    with pytest.raises(ValueError, match="residual"):
        ops.rms_norm_fwd(x, w, residual=res[:2])
    with pytest.raises(ValueError, match="contiguous"):
        ops.rms_norm_fwd(x.t().contiguous().t(), w)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rms_norm_fwd(x, w.cpu())
    with pytest.raises(ValueError, match="h goes with"):
        ops.rms_norm_quant_1x128(x, w, h=torch.empty_like(x))
    with pytest.raises(ValueError, match="dy"):
        ops.rms_norm_bwd(dy[:2], x, w, torch.ones(4, device=cuda))
    with pytest.raises(_lib.GlaucisError, match="multiple of 128"):
        ops.rms_norm_quant_1x128(x[:, :200].contiguous(), w[:200].contiguous())
    with pytest.raises(_lib.GlaucisError, match="multiple of 8"):
        ops.rms_norm_fwd(x[:, :100].contiguous(), w[:100].contiguous())
    with pytest.raises(_lib.GlaucisError, match="eps"):
        ops.rms_norm_fwd(x, w, -1.0)
    odd = torch.empty(4 * 256 + 1, dtype=BF16, device=cuda)[1:].view(4, 256)
    with pytest.raises(_lib.GlaucisError, match="aligned"):
        ops.rms_norm_fwd(odd, w)
