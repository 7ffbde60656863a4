"""The router: choices, counts, rows and balance loss, and the gradient of the
logits, against a numpy computation in 64 bits.

Tolerances.  With u = 2^-24: a softmax numerator is off by |z - max| u (the
subtraction) and 2 ulp of expf (4 u), the sum of E of them by (E / 32 + 5) u
more, reciprocal, products and division by 4 u each: EXP(row) =
(spread + E / 32 + 30) u relative.  The loss adds the running sums over a
warp's tokens, the CTA's warps and the CTAs (all terms positive)."""
import numpy as np
import pytest
import torch

from glaucis_b200 import _lib, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")


def _logits(cuda, T, E, bf16, seed, off=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    z = torch.randn((T, E), generator=g, device=cuda) * 2 + torch.randn(E, generator=g, device=cuda)
    if off:
        z[:, torch.randperm(E, generator=g, device=cuda)[:off]] = -INF
    return z.to(torch.bfloat16 if bf16 else torch.float32)


def _reference(logits, k, mask, renorm):
    z = logits.double().cpu().numpy()
    T, E = z.shape
    live = (z != -INF).any(1)
    if mask is not None:
        live &= mask.cpu().numpy()
    p = np.zeros((T, E))
    with np.errstate(invalid="ignore"):
        e = np.exp(z[live] - np.nanmax(z[live], axis=1, keepdims=True, initial=-INF))
    e[z[live] == -INF] = 0
    p[live] = e / e.sum(1, keepdims=True)
    order = np.argsort(-np.where(np.isnan(z), -INF, z), axis=1, kind="stable")[:, :k]
    ok = live[:, None] & (np.take_along_axis(np.where(np.isnan(z), -INF, z), order, 1) > -INF)
    ids = np.where(ok, order, -1)
    w = np.where(ok, np.take_along_axis(p, order, 1), 0)
    total = w.sum(1, keepdims=True)
    if renorm:
        w = np.divide(w, total, out=np.zeros_like(w), where=total != 0)
    counts = np.bincount(ids[ids >= 0], minlength=E)
    pos = np.full(T * k, -1)
    flat = ids.reshape(-1)
    valid = np.flatnonzero(flat >= 0)
    pos[valid[np.argsort(flat[valid], kind="stable")]] = np.arange(valid.size)
    n = max(1, int(live.sum()))
    f = counts / max(1, counts.sum())
    loss = E * float(f @ p.sum(0)) / n
    return dict(ids=ids, w=w, counts=counts, pos=pos.reshape(T, k), loss=loss, p=p, f=f, n=n, ok=ok,
                total=total, live=live)


def _exp_tol(logits):
    z = logits.double().cpu().numpy()
    fin = np.where(np.isfinite(z), z, np.nan)
    with np.errstate(all="ignore"):
        spread = np.nanmax(fin, 1) - np.nanmin(fin, 1) if z.size else np.zeros(0)
    return (np.nan_to_num(spread) + z.shape[1] / 32 + 30)[:, None] * U


def _check_forward(r, ref, logits):
    T, E = logits.shape
    assert np.array_equal(r.ids.cpu().numpy(), ref["ids"])
    assert np.array_equal(r.counts.cpu().numpy(), ref["counts"])
    assert np.array_equal(r.pos.cpu().numpy(), ref["pos"])
    tol = _exp_tol(logits)
    err = np.abs(r.weights.double().cpu().numpy() - ref["w"])
    assert (err <= 3 * tol * ref["w"] + 1e-40).all(), err.max() if err.size else 0
    sums = T / 32 + 32 + 148  # at least: tokens of a warp, warps, CTAs
    rel = (float(tol.max()) if T else 0) + (sums + 10) * U
    assert abs(float(r.balance_loss) - ref["loss"]) <= rel * ref["loss"]


CASES = [(1, 128, 8), (3, 128, 8), (64, 128, 8), (65, 128, 8), (100, 8, 2), (33, 1, 1), (257, 5, 3), (500, 60, 4),
         (129, 160, 6), (300, 256, 8), (2000, 33, 8), (70, 384, 8), (150, 512, 32), (40, 1000, 10), (600, 1024, 32),
         (10007, 128, 8), (20000, 64, 6), (60, 8, 2), (12, 1000, 2), (9000, 300, 4), (16000, 1000, 8)]


@pytest.mark.parametrize("T,E,k", CASES)
@pytest.mark.parametrize("bf16,renorm", [(False, True), (True, False)])
def test_forward(cuda, T, E, k, bf16, renorm):
    logits = _logits(cuda, T, E, bf16, seed=T + E, off=E // 32 if E // 32 + k <= E else 0)
    r = ops.moe_route_fwd(logits, k, renormalize=renorm)
    _check_forward(r, _reference(logits, k, None, renorm), logits)
    assert ops.device_status() == 0


@pytest.mark.parametrize("T,E,k", [(50, 128, 8), (3000, 60, 4), (5000, 256, 8)])
def test_mask_and_what_padding_holds(cuda, T, E, k):
    logits = _logits(cuda, T, E, False, seed=7)
    mask = torch.rand(T, generator=torch.Generator().manual_seed(1)).to(cuda) > 0.3
    clean = ops.moe_route_fwd(logits, k, mask=mask)
    _check_forward(clean, _reference(logits, k, mask, True), logits)
    junk = logits.clone()
    junk[~mask] = torch.tensor([float("nan"), INF, -INF, 3e38], device=cuda).repeat(E)[:E]
    r = ops.moe_route_fwd(junk, k, mask=mask)
    for a, b in zip(r[:6], clean[:6]):
        assert torch.equal(a, b)
    assert (r.ids[~mask] == -1).all() and (r.pos[~mask] == -1).all() and (r.weights[~mask] == 0).all()


@pytest.mark.parametrize("E", [1, 7, 32, 60, 128, 256, 500, 1024])
@pytest.mark.parametrize("bf16", [False, True])
def test_small_probabilities_keep_their_bits(cuda, E, bf16):
    # whole logits: subtracting the largest is exact, so a probability is off by
    # 2 ulp of the exponential (4 u) above and in the sum, by (E / 32 + 5) u of
    # the sum itself, 4 u of its reciprocal and u of the product, whatever its
    # size; and the loss as in _check_forward, without the subtraction's share.
    k, T = min(E, 8), 300
    g = torch.Generator(device=cuda).manual_seed(E)
    z = -torch.randint(0, 87, (T, E), generator=g, device=cuda).float()
    z[1] = -80
    z[1, 0] = 0
    z = z.to(torch.bfloat16) if bf16 else z
    r = ops.moe_route_fwd(z, k, renormalize=False)
    ref = _reference(z, k, None, False)
    tol = (E / 32 + 18) * U
    assert np.array_equal(r.ids.cpu().numpy(), ref["ids"])
    err = np.abs(r.weights.double().cpu().numpy() - ref["w"])
    assert (err <= tol * ref["w"]).all(), float((err / ref["w"]).max() / U)
    assert abs(float(r.balance_loss) - ref["loss"]) <= (tol + (T / 32 + 32 + 148 + 10) * U) * ref["loss"]
    # the gradient of the loss alone: p (c - sum p c), every p and the sum so
    dl = ops.moe_route_bwd(z, r, None, torch.ones((), device=cuda)).double().cpu().numpy()
    c = E * ref["f"] / ref["n"]
    mean = (ref["p"] * c).sum(1, keepdims=True)
    want = ref["p"] * (c - mean)
    bound = ref["p"] * (tol * np.abs(c - mean) + (2 * tol + (E / 32 + 12) * U) * (np.abs(c) + mean))
    # its rounding: half a step, of the type's subnormals 2^-133 (bf16) or of a
    # few products that end at 2^-149 (fp32)
    half = 2.0 ** -8 * np.abs(want) + 2.0 ** -134 if bf16 else U * np.abs(want)
    assert (np.abs(dl - want) <= bound + half + 8 * 2.0 ** -149).all()


def test_ties_go_to_the_lowest_expert(cuda):
    logits = torch.zeros((40, 128), device=cuda)
    logits[1::2] = -0.0
    logits[5, 64:] = 1.0
    logits[6, 3::7] = 2.0
    logits[7, ::2] = -0.0  # both zeros are one value
    r = ops.moe_route_fwd(logits, 8)
    _check_forward(r, _reference(logits, 8, None, True), logits)
    assert r.ids[5].tolist() == list(range(64, 72)) and r.ids[7].tolist() == list(range(8))


def test_even_split_has_loss_one(cuda):
    T, E = 512, 16
    logits = torch.full((T, E), -30.0, device=cuda)
    logits[torch.arange(T), torch.arange(T) % E] = 30.0
    assert abs(float(ops.moe_route_fwd(logits, 1).balance_loss) - 1) < 1e-5


@pytest.mark.parametrize("T", [9, 400])
def test_switched_off_experts_and_empty_rows(cuda, T):
    E, k = 40, 6
    logits = _logits(cuda, T, E, False, seed=11)
    logits[2] = -INF                      # nothing left: not routed
    logits[4] = -INF
    logits[4, [7, 30]] = torch.tensor([0.5, 1.5], device=cuda)  # fewer than k
    logits[6, 5:] = -INF
    r = ops.moe_route_fwd(logits, k)
    _check_forward(r, _reference(logits, k, None, True), logits)
    assert r.ids[4].tolist() == [30, 7, -1, -1, -1, -1] and (r.ids[2] == -1).all()
    dl = ops.moe_route_bwd(logits, r, torch.ones_like(r.weights), torch.ones((), device=cuda))
    assert torch.isfinite(dl).all() and (dl[2] == 0).all() and (dl[logits == -INF] == 0).all()


def test_nothing_routed(cuda):
    for logits, mask in [(torch.zeros((0, 16), device=cuda), None),
                         (torch.full((70, 16), -INF, device=cuda), None),
                         (torch.zeros((200, 16), device=cuda), torch.zeros(200, dtype=torch.bool, device=cuda))]:
        r = ops.moe_route_fwd(logits, 2, mask=mask)
        assert float(r.balance_loss) == 0 and (r.counts == 0).all() and (r.ids == -1).all() and (r.pos == -1).all()
        dl = ops.moe_route_bwd(logits, r, torch.ones_like(r.weights), torch.ones((), device=cuda))
        assert (dl == 0).all()


def test_nan_shows_and_stays_in_its_row(cuda):
    logits = _logits(cuda, 80, 64, False, seed=13)
    clean = ops.moe_route_fwd(logits, 4)
    logits[3, 9] = float("nan")
    logits[5] = float("nan")
    r = ops.moe_route_fwd(logits, 4)
    others = [t for t in range(80) if t not in (3, 5)]
    assert torch.equal(r.ids[others], clean.ids[others]) and torch.equal(r.weights[others], clean.weights[others])
    assert 9 not in r.ids[3].tolist() and (r.ids[3] >= 0).all() and torch.isnan(r.weights[3]).all()
    assert (r.ids[5] == -1).all() and torch.isnan(r.balance_loss)


def _gradient(ref, dw, dloss, renorm, k):
    """dlogits and the sum of its terms' magnitudes."""
    E = ref["p"].shape[1]
    p, ids = ref["p"], np.maximum(ref["ids"], 0)
    sel = np.where(ref["ok"], dw, 0)
    mag = np.abs(sel)
    if renorm:
        total = np.where(ref["total"] == 0, 1, ref["total"])
        mag = np.where(ref["ok"], (mag + (mag * ref["w"]).sum(1, keepdims=True)) / total, 0)
        sel = np.where(ref["ok"], (sel - (sel * ref["w"]).sum(1, keepdims=True)) / total, 0)
    c = dloss * E / ref["n"] * ref["f"]
    dp, dm = np.tile(c, (len(p), 1)), np.tile(np.abs(c), (len(p), 1))
    for j in range(k):
        np.put_along_axis(dp, ids[:, j:j + 1], np.take_along_axis(dp, ids[:, j:j + 1], 1) + sel[:, j:j + 1], 1)
        np.put_along_axis(dm, ids[:, j:j + 1], np.take_along_axis(dm, ids[:, j:j + 1], 1) + mag[:, j:j + 1], 1)
    dz = p * (dp - (p * dp).sum(1, keepdims=True))
    return np.where(ref["live"][:, None], dz, 0), p * (dm + (p * dm).sum(1, keepdims=True))


@pytest.mark.parametrize("T,E,k", CASES)
@pytest.mark.parametrize("bf16,renorm", [(False, True), (False, False), (True, True)])
def test_backward(cuda, T, E, k, bf16, renorm):
    logits = _logits(cuda, T, E, bf16, seed=2 * T + E, off=E // 32 if E // 32 + k <= E else 0)
    mask = torch.arange(T, device=cuda) % 5 != 3
    r = ops.moe_route_fwd(logits, k, mask=mask, renormalize=renorm)
    g = torch.Generator(device=cuda).manual_seed(5)
    dw = torch.randn((T, k), generator=g, device=cuda)
    dloss = torch.tensor(0.7, device=cuda)
    ref = _reference(logits, k, mask, renorm)
    dz, terms = _gradient(ref, dw.double().cpu().numpy(), float(dloss), renorm, k)
    got = ops.moe_route_bwd(logits, r, dw, dloss)
    assert got.dtype == logits.dtype
    tol = 6 * _exp_tol(logits) * terms + (2.0 ** -8 if bf16 else 0) * np.abs(dz) + 1e-30
    err = np.abs(got.double().cpu().numpy() - dz)
    assert (err <= tol).all(), float((err - tol).max())
    # each of the two gradients alone
    a = ops.moe_route_bwd(logits, r, dw, None).double().cpu().numpy()
    b = ops.moe_route_bwd(logits, r, None, dloss).double().cpu().numpy()
    half = (2.0 ** -8 if bf16 else 0) * (np.abs(a) + np.abs(b))
    assert (np.abs(a + b - dz) <= 2 * tol + half).all()


@pytest.mark.parametrize("T,E", [(50, 7), (3000, 128)])
def test_a_single_choice_has_weight_one_and_no_gradient(cuda, T, E):
    logits = _logits(cuda, T, E, False, seed=23)
    r = ops.moe_route_fwd(logits, 1)
    assert (r.weights == 1).all()
    dw = torch.randn((T, 1), device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)) * 1e3
    assert (ops.moe_route_bwd(logits, r, dw, None) == 0).all()


def test_gradient_against_differences(cuda):
    T, E, k = 24, 20, 3
    logits = _logits(cuda, T, E, False, seed=17)
    r = ops.moe_route_fwd(logits, k)
    g = torch.Generator(device=cuda).manual_seed(6)
    dw, d = torch.randn((T, k), generator=g, device=cuda), torch.randn((T, E), generator=g, device=cuda)
    got = ops.moe_route_bwd(logits, r, dw, torch.tensor(1.3, device=cuda))
    ids, counts = r.ids.long(), r.counts.double()

    def value(z):
        p = torch.softmax(z, 1)
        w = p.gather(1, ids)
        loss = E * (counts / counts.sum() * p.mean(0)).sum()
        return (w / w.sum(1, keepdim=True) * dw.double()).sum() + 1.3 * loss

    z, t = logits.double(), 1e-5
    diff = float((value(z + t * d.double()) - value(z - t * d.double())) / (2 * t))
    want = float((got.double() * d.double()).sum())
    assert abs(diff - want) <= 1e-5 * float((got.double() * d.double()).abs().sum())


def test_autograd(cuda):
    logits = _logits(cuda, 90, 32, True, seed=19).requires_grad_()
    r = ops.moe_route(logits, 4)
    assert r.weights.requires_grad and r.balance_loss.requires_grad and not r.counts.requires_grad
    g = torch.randn_like(r.weights)
    got, = torch.autograd.grad((r.weights * g).sum() + 0.01 * r.balance_loss, logits, retain_graph=True)
    plain = ops.moe_route_fwd(logits.detach(), 4)
    assert torch.equal(plain.weights, r.weights) and torch.equal(plain.pos, r.pos)
    want = ops.moe_route_bwd(logits.detach(), plain, g, torch.tensor(0.01, device=cuda))
    assert torch.equal(got, want)
    only, = torch.autograd.grad(r.balance_loss, logits)
    assert torch.equal(only, ops.moe_route_bwd(logits.detach(), plain, None, torch.ones((), device=cuda)))


@pytest.mark.parametrize("T", [40, 3000])
def test_the_same_every_time_and_on_two_streams(cuda, T):
    logits = [_logits(cuda, T, 128, False, seed=s) for s in (1, 2)]
    want = [ops.moe_route_fwd(z, 8) for z in logits]
    streams = [torch.cuda.Stream() for _ in logits]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.moe_route_fwd(logits[i], 8))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r[:6], want[i][:6]))


def test_offsets_past_32_bits(cuda):
    T, E, k = 2_200_000, 1024, 4  # 2.25e9 logits
    logits = torch.zeros((T, E), dtype=torch.bfloat16, device=cuda)
    logits[:, 3:7] = 1
    logits[-500:] = _logits(cuda, 500, E, True, seed=29)
    r = ops.moe_route_fwd(logits, k)
    tail = ops.moe_route_fwd(logits[-500:].clone(), k)
    assert torch.equal(r.ids[-500:], tail.ids) and torch.equal(r.weights[-500:], tail.weights)
    want = torch.bincount(r.ids.reshape(-1).long(), minlength=E).int()
    assert torch.equal(r.counts, want) and (r.ids[:-500] == torch.arange(3, 7, device=cuda)).all()
    rows = torch.zeros(T * k, dtype=torch.bool, device=cuda)
    rows[r.pos.reshape(-1).long()] = True
    assert rows.all()  # every row once
    start = want.cumsum(0) - want
    assert ((r.pos >= start[r.ids.long()]) & (r.pos < (start + want)[r.ids.long()])).all()
    dl = ops.moe_route_bwd(logits, r, torch.ones_like(r.weights), None)
    assert torch.isfinite(dl[-500:].float()).all()


def test_gradient_past_32_bits_is_that_of_its_rows(cuda):
    # the last tokens' logits lie past 2^31 elements and 2^32 bytes; without the
    # loss a token's gradient depends on its own row alone
    T, E, k, n = 2_200_000, 1024, 4, 500
    logits = torch.zeros((T, E), dtype=torch.bfloat16, device=cuda)
    logits[:, 3:7] = 1
    logits[-n:] = _logits(cuda, n, E, True, seed=31)
    dw = torch.randn((T, k), generator=torch.Generator(device=cuda).manual_seed(32), device=cuda)
    for renorm in (True, False):
        r = ops.moe_route_fwd(logits, k, renormalize=renorm)
        dl = ops.moe_route_bwd(logits, r, dw, None)
        tail = logits[-n:].clone()
        rt = ops.moe_route_fwd(tail, k, renormalize=renorm)
        want = ops.moe_route_bwd(tail, rt, dw[-n:].contiguous(), None)
        assert want.float().abs().amax(1).min() > 0
        assert torch.equal(dl[-n:], want)
        del dl, r


def test_backward_refuses_another_routings_types(cuda):
    z = torch.zeros((4, 16), device=cuda)
    r = ops.moe_route_fwd(z, 2)
    dw = torch.zeros((4, 2), device=cuda)
    for bad in (dict(ids=r.ids.long()), dict(counts=r.counts.long()), dict(weights=r.weights.double()),
                dict(routed=r.routed.double()), dict(routed=r.routed.expand(2).contiguous()),
                dict(counts=r.counts[:8].contiguous())):
        with pytest.raises(ValueError, match="belong"):
            ops.moe_route_bwd(z, r._replace(**bad), dw, None)


def test_refusals(cuda):
    z = torch.zeros((4, 16), device=cuda)
    for bad in (z.half(), z[0], z.double()):
        with pytest.raises(ValueError, match="logits"):
            ops.moe_route_fwd(bad, 2)
    with pytest.raises(ValueError, match="contiguous"):
        ops.moe_route_fwd(z.t(), 2)
    with pytest.raises(ValueError, match="mask"):
        ops.moe_route_fwd(z, 2, mask=torch.ones(3, dtype=torch.bool, device=cuda))
    with pytest.raises(ValueError, match="mask"):
        ops.moe_route_fwd(z, 2, mask=torch.ones(4, device=cuda))
    for k in (0, 17, 33):
        with pytest.raises(_lib.GlaucisError, match="topk"):
            ops.moe_route_fwd(z, k)
    with pytest.raises(_lib.GlaucisError, match="1024"):
        ops.moe_route_fwd(torch.zeros((2, 1025), device=cuda), 2)
    r = ops.moe_route_fwd(z, 2)
    with pytest.raises(ValueError, match="dweights"):
        ops.moe_route_bwd(z, r, torch.zeros((4, 3), device=cuda), None)
    with pytest.raises(ValueError, match="dloss"):
        ops.moe_route_bwd(z, r, None, torch.zeros(2, device=cuda))
    with pytest.raises(ValueError, match="belong"):
        ops.moe_route_bwd(z[:3].contiguous(), r, None, None)
