"""The operators around the experts' products run together, as a layer uses them:
norm, router, rows into expert order, products, weighted sum onto the residual;
for a prompt in e4m3, for generated tokens with 4-bit weights inside a CUDA
graph, and for training through autograd."""
import pytest
import torch

from glaucis_b200 import ops

pytestmark = pytest.mark.gpu

BF16, F64 = torch.bfloat16, torch.float64


def _rand(cuda, *shape, seed=0, scale=1.0, dtype=BF16):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=cuda) * scale).to(dtype)


def _experts64(rows, sizes, weight):
    """rows (fp64, expert order) times each expert's fp64 weight; zeros past the last group."""
    out = torch.zeros((rows.shape[0], weight(0).shape[1]), dtype=F64, device=rows.device)
    at = 0
    for g, n in enumerate(sizes):
        if n:
            out[at:at + n] = rows[at:at + n] @ weight(g)
            at += n
    return out


@pytest.mark.parametrize("T,E,k,K,N,pad", [(300, 16, 4, 1024, 512, 0), (129, 8, 2, 512, 256, 40), (1, 8, 2, 256, 128, 0)])
def test_prompt_in_e4m3(cuda, T, E, k, K, N, pad):
    x, res = _rand(cuda, T, K, seed=1), _rand(cuda, T, K, seed=2)
    w = (1 + 0.1 * _rand(cuda, K, seed=3, dtype=torch.float32))
    wg, rhs = _rand(cuda, K, E, seed=4, scale=0.05, dtype=torch.float32), _rand(cuda, E, K, N, seed=5, scale=0.02)
    down = _rand(cuda, E, N, K, seed=6, scale=0.02)
    mask = torch.arange(T, device=cuda) < T - pad if pad else None
    f = ops.rms_norm_fwd(x, w, residual=res, output_quant=True)
    r = ops.moe_route_fwd(f.y.float() @ wg, k, mask=mask)
    a_q, a_s = ops.moe_dispatch_quant(f.q, f.s, r.pos, r.counts)
    up = ops.gmm_fp8_fwd(a_q, a_s, *ops.quant_w_128x128(rhs), r.counts, out_dtype=BF16)
    rows = int(r.counts.sum())
    up[rows:] = 0
    mid_q, mid_s = ops.quant_act_1x128(torch.nn.functional.silu(up))
    y = ops.gmm_fp8_fwd(mid_q, mid_s, *ops.quant_w_128x128(down), r.counts, out_dtype=BF16)
    y[rows:] = float("nan")  # rows of no group are not read
    out = ops.moe_combine(y, r.pos, r.weights, r.counts, residual=f.h)
    assert ops.device_status() == 0 and torch.isfinite(out).all()
    assert rows == (T - pad) * k
    if pad:
        assert torch.equal(out[T - pad:], f.h[T - pad:])

    # the same products on the same quantised operands in 64 bits
    def deq(q, s):
        return q.to(F64) * s.to(F64).repeat_interleave(128, -1)

    def weights(t):
        q, s = ops.quant_w_128x128(t)
        return lambda g: q[g].to(F64) * s[g].to(F64).repeat_interleave(128, 0).repeat_interleave(128, 1)

    sizes = r.counts.tolist()
    # a product of e4m3 blocks: fp32 sums of 128 terms, then of K / 128 blocks; bf16 out
    ref_up = _experts64(deq(a_q, a_s), sizes, weights(rhs))
    mag = _experts64(deq(a_q, a_s).abs(), sizes, lambda g: weights(rhs)(g).abs())
    assert ((up.to(F64) - ref_up).abs() <= 2.0 ** -8 * ref_up.abs() + 2.0 ** -13 * mag).all()
    ref_y = _experts64(deq(mid_q, mid_s), sizes, weights(down))
    mag = _experts64(deq(mid_q, mid_s).abs(), sizes, lambda g: weights(down)(g).abs())
    assert ((y[:rows].to(F64) - ref_y[:rows]).abs() <= 2.0 ** -8 * ref_y[:rows].abs() + 2.0 ** -13 * mag[:rows]).all()
    at = r.pos.clamp_min(0).long()
    part = torch.where((r.pos >= 0)[:, :, None], y.to(F64)[at] * r.weights.to(F64)[:, :, None], 0)
    ref = f.h.to(F64) + part.sum(1)
    mag = f.h.to(F64).abs() + part.abs().sum(1)
    assert ((out.to(F64) - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -20 * mag).all()


def test_rows_are_quantised_once_or_per_choice_alike(cuda):
    T, E, k, K = 200, 16, 4, 512
    x, w = _rand(cuda, T, K), torch.ones(K, dtype=BF16, device=cuda)
    f = ops.rms_norm_fwd(x, w, output_quant=True)
    r = ops.moe_route_fwd(_rand(cuda, T, E, seed=1, dtype=torch.float32), k)
    a_q, a_s = ops.moe_dispatch_quant(*ops.quant_act_1x128(f.y), r.pos, r.counts)
    b_q, b_s = ops.quant_act_1x128(ops.moe_dispatch(f.y, r.pos, r.counts))
    assert torch.equal(a_q.view(torch.uint8), b_q.view(torch.uint8)) and torch.equal(a_s, b_s)


def test_generated_tokens_in_a_graph(cuda):
    T, E, k, K, N = 3, 32, 4, 1024, 512
    w = torch.ones(K, dtype=BF16, device=cuda)
    wg = _rand(cuda, K, E, seed=1, scale=0.05, dtype=torch.float32)
    up, down = (ops.quant_w4_128x1(_rand(cuda, E, a, b, seed=s, scale=0.02)) for a, b, s in ((K, N, 2), (N, K, 3)))

    def layer(x, res):
        f = ops.rms_norm_fwd(x, w, residual=res)
        r = ops.moe_route(f.y.float() @ wg, k)
        xs = ops.moe_dispatch(f.y, r.pos, r.counts)
        mid = torch.nn.functional.silu(ops.gmm_w4_fwd(xs, *up, r.counts, out_dtype=BF16))
        y = ops.gmm_w4_fwd(mid, *down, r.counts)
        return ops.moe_combine(y, r.pos, r.weights, r.counts, residual=f.h)

    x, res = _rand(cuda, T, K, seed=4), _rand(cuda, T, K, seed=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, res)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, res)
    for seed in range(6, 12):
        x.copy_(_rand(cuda, T, K, seed=seed))
        res.copy_(_rand(cuda, T, K, seed=seed + 100))
        graph.replay()
        torch.cuda.synchronize()
        assert ops.device_status() == 0
        assert torch.equal(out, layer(x, res))


def _train_inputs(cuda, T, E, K, N):
    p = dict(x=_rand(cuda, T, K, seed=1), res=_rand(cuda, T, K, seed=2),
             w=1 + 0.1 * _rand(cuda, K, seed=3, dtype=torch.float32),
             wg=_rand(cuda, K, E, seed=4, scale=0.05, dtype=torch.float32), rhs=_rand(cuda, E, K, N, seed=5, scale=0.02))
    return p, _rand(cuda, T, N, seed=6, scale=0.1)


def _train_forward(p, k, mask, rows):
    y, h = ops.rms_norm(p["x"], p["w"], residual=p["res"])
    logits = y.float() @ p["wg"]
    r = ops.moe_route(logits, k, mask=mask)
    xs = ops.moe_dispatch(y, r.pos, r.counts, rows)
    e = ops.gmm_fp8_blockwise(xs, p["rhs"], r.counts, out_dtype=BF16)
    return y, h, logits, r, xs, e, ops.moe_combine(e, r.pos, r.weights, r.counts, residual=h)


@pytest.mark.parametrize("T,E,k,K,pad", [(192, 8, 2, 512, 0), (256, 16, 4, 256, 50)])
def test_training_step(cuda, T, E, k, K, pad):
    """Autograd through the layer gives bit for bit what the operators' own
    backward calls give, chained by hand (each of which its own tests hold to
    the formulas and to differences)."""
    p, dout = _train_inputs(cuda, T, E, K, K)
    leaves = {n: t.clone().requires_grad_() for n, t in p.items()}
    mask = torch.arange(T, device=cuda) < T - pad if pad else None
    rows = (T * k + 127) // 128 * 128
    y, h, logits, r, xs, e, out = _train_forward(leaves, k, mask, rows)
    loss = (out.float() * dout.float()).sum() + 0.01 * r.balance_loss
    got = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))

    with torch.no_grad():
        f = ops.rms_norm_fwd(p["x"], p["w"], residual=p["res"])
        rt = ops.moe_route_fwd(f.y.float() @ p["wg"], k, mask=mask)
        assert torch.equal(f.y, y) and torch.equal(f.h, h) and torch.equal(rt.pos, r.pos)
        de, dweights = ops.moe_combine_bwd(dout, e.detach(), rt.pos, rt.weights, rt.counts)
        dxs, drhs = ops.gmm_fp8_blockwise_bwd(xs.detach(), p["rhs"], rt.counts, de)
        dlogits = ops.moe_route_bwd(logits.detach(), rt, dweights, torch.tensor(0.01, device=cuda))
        dy = ops.moe_dispatch_bwd(dxs, rt.pos) + (dlogits @ p["wg"].t()).to(BF16)
        dx, dw = ops.rms_norm_bwd(dy, f.h, p["w"], f.rstd, dh=dout)
        dwg = f.y.float().t() @ dlogits
    assert torch.equal(got["rhs"], drhs) and torch.equal(got["wg"], dwg)
    assert torch.equal(got["x"], dx) and torch.equal(got["res"], dx) and torch.equal(got["w"], dw)
    if pad:  # padding reaches neither the router nor the experts: its gradient is the residual's
        assert (dlogits[T - pad:] == 0).all()
        assert torch.equal(dy[T - pad:], torch.zeros_like(dy[T - pad:]))
    assert ops.device_status() == 0


def test_training_step_in_a_graph(cuda):
    """Forward and backward captured together replay to the eager gradients."""
    T, E, k, K = 128, 8, 2, 256
    p, dout = _train_inputs(cuda, T, E, K, K)
    leaves = {n: t.clone().requires_grad_() for n, t in p.items()}

    def step():
        r, out = _train_forward(leaves, k, None, T * k)[3::3]
        return torch.autograd.grad((out.float() * dout.float()).sum() + 0.01 * r.balance_loss, list(leaves.values()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (20, 21):
        with torch.no_grad():
            leaves["x"].copy_(_rand(cuda, T, K, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [g.clone() for g in got]
        for a, b in zip(replayed, step()):
            assert torch.equal(a, b)


def test_second_derivatives_are_refused(cuda):
    p, dout = _train_inputs(cuda, 128, 8, 256, 256)
    x = p["x"].requires_grad_()
    y = ops.rms_norm(x, p["w"])
    g, = torch.autograd.grad(y, x, dout.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()


def test_calls_on_many_streams(cuda):
    """The same calls under way on several streams at once give what they give alone."""
    T, E, k, K = 500, 64, 6, 512
    w = torch.ones(K, dtype=BF16, device=cuda)
    xs = [_rand(cuda, T, K, seed=i) for i in range(4)]
    zs = [_rand(cuda, T, E, seed=10 + i, dtype=torch.float32) for i in range(4)]
    w4 = ops.quant_w4_128x1(_rand(cuda, E, K, 128, seed=30, scale=0.02))

    def chain(x, z):
        f = ops.rms_norm_fwd(x, w)
        dx, dw = ops.rms_norm_bwd(x, f.h, w, f.rstd)
        r = ops.moe_route_fwd(z, k)
        rows = ops.moe_dispatch(f.y, r.pos, r.counts)
        y = ops.gmm_w4_fwd(rows, *w4, r.counts, out_dtype=BF16)
        return dx, dw, r.pos, r.balance_loss, ops.moe_combine(y, r.pos, r.weights, r.counts)

    want = [chain(x, z) for x, z in zip(xs, zs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(chain(xs[i], zs[i]))
    torch.cuda.synchronize()
    for i in range(4):
        for res in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(res, want[i]))
    assert ops.device_status() == 0


def _buffers(cuda, T, E, k, K):
    g = torch.Generator(device=cuda).manual_seed(5)
    r = ops.moe_route_fwd(torch.randn((T, E), generator=g, device=cuda), k)
    w4, s = ops.quant_w4_128x1(_rand(cuda, E, K, K, seed=6, scale=K ** -0.5))
    h = _rand(cuda, T, K, seed=7)
    return dict(r=r, w4=w4, s=s, h=h, h0=h.clone(), xs=torch.empty((T * k, K), dtype=BF16, device=cuda),
                y=torch.empty((T * k, K), dtype=BF16, device=cuda))


@pytest.mark.parametrize("T,E,k,K", [(1, 8, 2, 512), (16, 8, 2, 1024), (300, 16, 2, 2048)])
def test_each_call_sees_the_one_before(cuda, T, E, k, K):
    """Calls that read what the call just before them wrote over its own input,
    one after the other without a pause and in a graph, give what they give with
    the device idle between them."""
    b = _buffers(cuda, T, E, k, K)
    r = b["r"]

    def chain(between):
        for i in range(12):
            ops.moe_dispatch_fwd(b["h"], r.pos, r.counts, out=b["xs"])
            between()
            ops.gmm_w4_fwd(b["xs"], b["w4"], b["s"], r.counts, out=b["y"])
            between()
            ops.moe_combine_fwd(b["y"], r.pos, r.weights, residual=b["h"], out=b["h"])
            between()
            if i % 3 == 2:  # else the next dispatch follows at once
                b["h"].mul_(0.25)
                between()

    chain(torch.cuda.synchronize)
    want = b["h"].clone()
    assert torch.isfinite(want).all()
    for _ in range(5):
        b["h"].copy_(b["h0"])
        chain(lambda: None)
        assert torch.equal(b["h"], want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b["h"].copy_(b["h0"])
        chain(lambda: None)
    for _ in range(5):
        b["h"].zero_()
        graph.replay()
        assert torch.equal(b["h"], want)
    assert ops.device_status() == 0


def test_captured_after_anything(cuda):
    """A call captured first, after copies, fills, forks and joins of streams."""
    b = _buffers(cuda, 16, 8, 2, 1024)
    r, src, other = b["r"], _rand(cuda, 32, 1024, seed=8), torch.cuda.Stream()
    z, x = torch.zeros(1 << 20, device=cuda), src.clone()

    def call():
        return ops.gmm_w4_fwd(x, b["w4"], b["s"], r.counts)

    want = call()

    def after_copy():
        x.copy_(src)
        return [call()]

    def after_fill():
        z.zero_()
        return [call()]

    def after_join():
        cur = torch.cuda.current_stream()
        z.add_(1)
        other.wait_stream(cur)
        with torch.cuda.stream(other):
            torch.mul(src, 1, out=x)
        z.add_(1)
        cur.wait_stream(other)
        return [call()]

    def in_a_fork():
        cur = torch.cuda.current_stream()
        torch.mul(src, 1, out=x)
        other.wait_stream(cur)
        with torch.cuda.stream(other):
            a = call()
        c = call()
        cur.wait_stream(other)
        return [a, c]

    for step in (lambda: [call()], lambda: [call(), call()], after_copy, after_fill, after_join, in_a_fork):
        assert all(torch.equal(o, want) for o in step())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for _ in range(5):
            if step in (after_copy, after_join, in_a_fork):
                x.zero_()
            for o in out:
                o.zero_()
            graph.replay()
            assert all(torch.equal(o, want) for o in out)
        x.copy_(src)
    assert ops.device_status() == 0


@pytest.mark.parametrize("T,K", [(1, 512), (16, 1024), (300, 1024)])
def test_norm_and_router_see_the_call_before(cuda, T, K):
    """The norm reads what the combine just wrote and adds it to the stream in
    place; the router takes the norm's output as it comes."""
    E, k = 8, 2
    b = _buffers(cuda, T, E, k, K)
    r, w = b["r"], torch.ones(K, dtype=BF16, device=cuda)
    x, n = b["h0"].clone(), torch.empty_like(b["h0"])

    def chain(between):
        ids = []
        x.copy_(b["h0"])
        b["h"].copy_(b["h0"])
        for _ in range(8):
            ops.rms_norm_fwd(x, w, residual=b["h"], y=n, h=b["h"])
            between()
            ids.append(ops.moe_route_fwd(n, 4).ids)
            between()
            ops.moe_dispatch_fwd(n, r.pos, r.counts, out=b["xs"])
            between()
            ops.gmm_w4_fwd(b["xs"], b["w4"], b["s"], r.counts, out=b["y"])
            between()
            ops.moe_combine_fwd(b["y"], r.pos, r.weights, out=x)
            between()
        return torch.stack(ids)

    ids = chain(torch.cuda.synchronize)
    want = b["h"].clone()
    assert torch.isfinite(want).all()
    for _ in range(5):
        assert torch.equal(chain(lambda: None), ids) and torch.equal(b["h"], want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(lambda: None)
    for _ in range(5):
        b["h"].zero_()
        graph.replay()
        assert torch.equal(got, ids) and torch.equal(b["h"], want)
    assert ops.device_status() == 0


def _one_expert(cuda, T=4, K=256, N=64):
    g = torch.Generator(device=cuda).manual_seed(40)
    x = torch.randn((T, K), generator=g, device=cuda).to(torch.bfloat16)
    w4 = torch.randint(-2 ** 31, 2 ** 31, (1, K // 8, N), generator=g, device=cuda, dtype=torch.int32)
    return x, w4, torch.ones((1, K // 128, N), device=cuda), torch.tensor([T], dtype=torch.int32, device=cuda)


def test_a_gradient_that_does_not_exist_is_an_error(cuda):
    # a call that takes part in a recorded computation but has no backward says
    # so when the gradient is asked for; without one it runs as ever
    x, w4, s, sizes = _one_expert(cuda)
    w = torch.ones(x.shape[1], device=cuda)
    pos = torch.arange(4, dtype=torch.int32, device=cuda)[:, None].contiguous()
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    clean = ops.gmm_w4_fwd(x, w4, s, sizes)
    out = ops.gmm_w4_fwd(xg, w4, s, sizes)
    assert torch.equal(out, clean) and not clean.requires_grad
    with pytest.raises(RuntimeError, match="gmm_w4_fwd"):
        out.sum().backward()
    q, sc = ops.quant_act_1x128(x)
    scg = sc.clone().requires_grad_()
    _, moved = ops.moe_dispatch_quant(q, scg, pos, sizes)
    assert torch.equal(moved, sc)
    with pytest.raises(RuntimeError, match="moe_dispatch_quant"):
        moved.sum().backward()
    for a, b in ((xg, w), (x, wg)):
        pair = ops.rms_norm_quant_1x128(a, b, residual=x)
        with pytest.raises(RuntimeError, match="rms_norm_quant_1x128"):
            pair[2].float().sum().backward()
    assert xg.grad is None and wg.grad is None
    # a given output cannot carry that: refused where a gradient is recorded
    own = torch.empty_like(clean)
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.gmm_w4_fwd(xg, w4, s, sizes, out=own)
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.rms_norm_quant_1x128(xg, w, residual=x, h=torch.empty_like(x))
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.moe_dispatch_quant(q, scg, pos, sizes, out_s=torch.empty_like(sc))
    with torch.no_grad():
        assert torch.equal(ops.gmm_w4_fwd(xg, w4, s, sizes, out=own), clean)
        assert not ops.rms_norm_quant_1x128(xg, wg)[1].requires_grad


def test_forward_mode_tangents_are_refused(cuda):
    from torch.autograd import forward_ad as fw
    x, w4, s, sizes = _one_expert(cuda)
    w = torch.ones(x.shape[1], device=cuda)
    pos = torch.arange(4, dtype=torch.int32, device=cuda)[:, None].contiguous()
    one = torch.ones((4, 1), device=cuda)
    q, sc = ops.quant_act_1x128(x)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for name, call in [("rms_norm", lambda: ops.rms_norm(dual(x), w)),
                           ("rms_norm", lambda: ops.rms_norm(x, w, residual=dual(x))),
                           ("rms_norm_quant_1x128", lambda: ops.rms_norm_quant_1x128(x, dual(w))),
                           ("moe_route", lambda: ops.moe_route(dual(x[:, :8].float().contiguous()), 2)),
                           ("moe_dispatch", lambda: ops.moe_dispatch(dual(x), pos, sizes)),
                           ("moe_dispatch_quant", lambda: ops.moe_dispatch_quant(q, dual(sc), pos, sizes)),
                           ("moe_combine", lambda: ops.moe_combine(x, pos, dual(one), sizes)),
                           ("gmm_w4_fwd", lambda: ops.gmm_w4_fwd(dual(x), w4, s, sizes))]:
            with pytest.raises(RuntimeError, match=f"{name}.*forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match=f"{name}.*forward-mode"):
                call()
        assert torch.equal(ops.rms_norm(x, w), ops.rms_norm_fwd(x, w).y)  # no tangent, no refusal


def test_combine_refuses_early_what_its_gradient_could_not_take(cuda):
    T, K = 4, 64
    y = torch.ones((T, K), device=cuda, requires_grad=True)
    pos = torch.arange(T, dtype=torch.int32, device=cuda)[:, None].contiguous()
    w = torch.ones((T, 1), device=cuda)
    sizes = torch.tensor([T], dtype=torch.int32, device=cuda)
    for bad in (sizes.long(), sizes.cpu(), sizes[None], torch.zeros(1025, dtype=torch.int32, device=cuda),
                torch.zeros(0, dtype=torch.int32, device=cuda)):
        with pytest.raises(ValueError, match="group_sizes|CUDA"):
            ops.moe_combine(y, pos, w, bad)
        with pytest.raises(ValueError, match="group_sizes|CUDA"):
            ops.moe_combine(y.detach(), pos, w.clone().requires_grad_(), bad)
    ops.moe_combine(y, pos, w, sizes).sum().backward()
    assert (y.grad == 1).all()
