"""Grouped products with 4-bit weights and their quantiser, against 64 bits.

Tolerances.  The quantiser is exact arithmetic: equal bit for bit.  The
product of a nibble and x is exact; the matrix unit adds 16 of them at a time
in fp32, 8 times a block, each addition off by at most 2^-22 of what it adds
(a half-ulp rounding gives 2^-24, truncation 2^-23; the offset's share counts
as a term).  Blocks then add up in fp32 with 3 roundings each.  So with
A = sum_k s (|q| + 16) |x| an output is within
(8 * 2^-22 + (K / 128 + 16) * 2^-24) A, and half a step of bf16 when it is
bf16."""
import pytest
import torch

from glaucis_b200 import _lib, ops

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _weights(cuda, G, K, N, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    w4 = torch.randint(-2 ** 31, 2 ** 31, (G, K // 8, N), generator=g, device=cuda, dtype=torch.int32)
    s = (torch.rand((G, K // 128, N), generator=g, device=cuda) + 0.1) * 0.01
    return w4, s


def _unpack(w4):
    G, K8, N = w4.shape
    u = w4.to(torch.int64)[:, :, None, :] >> (4 * torch.arange(8, device=w4.device))[:, None]
    return ((u & 15) - 8).reshape(G, K8 * 8, N)


def _x(cuda, M, K, seed=1):
    return torch.randn((M, K), generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda).to(BF16)


def _check(out, x, w4, s, sizes, K):
    row = 0
    for g, n in enumerate(sizes):
        if not n:
            continue
        q = _unpack(w4[g:g + 1])[0].to(F64)
        sc = s[g].to(F64).repeat_interleave(128, 0)
        xr = x[row:row + n].to(F64)
        ref, mag = xr @ (q * sc), xr.abs() @ ((q.abs() + 16) * sc)
        tol = (8 * 2.0 ** -22 + (K / 128 + 16) * 2.0 ** -24) * mag
        if out.dtype == BF16:
            tol = tol + 2.0 ** -8 * ref.abs()
        err = (out[row:row + n].to(F64) - ref).abs()
        assert (err <= tol).all(), (g, n, float((err - tol).max()), float(err.max()))
        row += n


CASES = [
    (128, 32, [1]), (128, 32, [3]), (1024, 1024, [1, 0, 0, 1, 0, 0, 0, 0]), (1152, 96, [0, 2, 7, 8, 9, 0, 17, 1]),
    (256, 160, [0, 0, 33]), (4096, 256, [1] * 8 + [0] * 56), (7168, 64, [0] * 100 + [4] + [0] * 27),
    (2048, 512, [5, 0, 1] * 50), (640, 128, [1] * 300), (512, 64, [0] * 1000 + [2, 0, 1] + [0] * 21),
    (14336, 64, [2]), (384, 2048, [64]),
]


@pytest.mark.parametrize("K,N,sizes", CASES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_product(cuda, K, N, sizes, dtype):
    G, rows = len(sizes), sum(sizes)
    w4, s = _weights(cuda, G, K, N)
    x = _x(cuda, rows + 3, K)  # three rows of no group
    gs = torch.tensor(sizes, dtype=torch.int32, device=cuda)
    out = ops.gmm_w4_fwd(x, w4, s, gs, out_dtype=dtype)
    assert out.dtype == dtype and (out[rows:] == 0).all()
    _check(out, x, w4, s, sizes, K)
    own = torch.full((rows + 3, N), 7.0, dtype=dtype, device=cuda)
    assert ops.gmm_w4_fwd(x, w4, s, gs, out=own) is own
    assert torch.equal(own[:rows], out[:rows]) and (own[rows:] == 7).all()
    assert ops.device_status() == 0


def test_every_nibble_at_every_place(cuda):
    # one-hot rows read single weights back: 8 places of a word, 16 values each
    K, N = 128, 32
    q = (torch.arange(K * N, device=cuda).reshape(K, N) * 7 + torch.arange(K, device=cuda)[:, None]) % 16
    word = torch.zeros((K // 8, N), dtype=torch.int64, device=cuda)
    for j in range(8):
        word |= q[j::8] << (4 * j)
    w4 = torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)[None].contiguous()
    s = torch.ones((1, 1, N), device=cuda)
    out = ops.gmm_w4_fwd(torch.eye(K, device=cuda).to(BF16), w4, s, torch.tensor([K], dtype=torch.int32, device=cuda))
    assert torch.equal(out, (q - 8).float())


@pytest.mark.parametrize("scale", [2.0 ** -130, 2.0 ** -118, 1e-30, 1e-3, 1e4, 2.0 ** 60, 2.0 ** 115])
def test_rows_of_any_magnitude(cuda, scale):
    K, N = 512, 64
    w4, s = _weights(cuda, 2, K, N, seed=3)
    x = (_x(cuda, 6, K, seed=4).float() * scale).to(BF16)
    x[1, 128:256] = 0
    x[2, ::2] = (x[2, ::2].float() * 2.0 ** -20).to(BF16)  # far apart within a block
    if scale > 1:
        x[3, :128] = (x[3, :128].float() / scale).to(BF16)  # blocks far apart
    out = ops.gmm_w4_fwd(x, w4, s, torch.tensor([2, 4], dtype=torch.int32, device=cuda))
    if scale >= 1e-30:
        _check(out, x, w4, s, [2, 4], K)
    else:  # sums near fp32's smallest values: half a subnormal step for each of the roundings
        q = torch.cat([(_unpack(w4[g:g + 1])[0].to(F64) * s[g].to(F64).repeat_interleave(128, 0))[None]
                       for g in (0, 1)])
        ref = torch.cat([x[:2].to(F64) @ q[0], x[2:].to(F64) @ q[1]])
        mag = torch.cat([x[:2].to(F64).abs() @ q[0].abs(), x[2:].to(F64).abs() @ q[1].abs()])
        assert ((out.to(F64) - ref).abs() <= 2.0 ** -16 * mag + 24 * 2.0 ** -149).all()


def test_non_finite_rows_stay_alone(cuda):
    K, N = 1024, 96
    w4, s = _weights(cuda, 1, K, N, seed=5)
    x = _x(cuda, 12, K, seed=6)
    gs = torch.tensor([12], dtype=torch.int32, device=cuda)
    clean = ops.gmm_w4_fwd(x, w4, s, gs)
    x[4, 7], x[9, 1000] = float("nan"), float("inf")
    out = ops.gmm_w4_fwd(x, w4, s, gs)
    assert not torch.isfinite(out[[4, 9]]).any()
    keep = [r for r in range(12) if r not in (4, 9)]
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("G,K,N", [(1, 128, 32), (3, 256, 96), (2, 1024, 320)])
def test_quantiser(cuda, G, K, N):
    w = (torch.randn((G, K, N), generator=torch.Generator(device=cuda).manual_seed(8), device=cuda) * 0.02).to(BF16)
    w[0, :128, 5] = 0
    w[0, 3, 6] = 1.0
    w4, s = ops.quant_w4_128x1(w)
    b = w.float().reshape(G, K // 128, 128, N)
    want_s = (b.abs().amax(2).double() / 7).float()  # the correctly rounded quotient
    want_s = torch.where(want_s == 0, 1.0, want_s)
    assert torch.equal(s, want_s)
    want_q = torch.round(b / want_s[:, :, None]).reshape(G, K, N).long()
    q = _unpack(w4)
    assert torch.equal(q, want_q) and int(q.min()) >= -7 and int(q.max()) == 7
    # the pair goes into the product: within the quantiser's half step of w
    x = _x(cuda, G * 2, K, seed=9)
    out = ops.gmm_w4_fwd(x, w4, s, torch.full((G,), 2, dtype=torch.int32, device=cuda))
    _check(out, x, w4, s, [2] * G, K)


def test_no_rows_and_no_groups_in_use(cuda):
    w4, s = _weights(cuda, 4, 256, 64)
    zero = torch.zeros(4, dtype=torch.int32, device=cuda)
    assert ops.gmm_w4_fwd(_x(cuda, 0, 256), w4, s, zero).shape == (0, 64)
    assert (ops.gmm_w4_fwd(_x(cuda, 9, 256), w4, s, zero) == 0).all()
    assert ops.device_status() == 0


def test_bad_sizes_are_reported(cuda):
    # row ranges are clipped to x's rows by the kernels themselves
    w4, s = _weights(cuda, 3, 256, 64)
    x = _x(cuda, 6, 256)
    for bad in ([3, 3, 1], [-1, 2, 2], [2 ** 31 - 1, 2 ** 31 - 1, 5], [0, 0, 7]):
        ops.gmm_w4_fwd(x, w4, s, torch.tensor(bad, dtype=torch.int32, device=cuda))
        assert ops.device_status() == 2, bad
    out = ops.gmm_w4_fwd(x, w4, s, torch.tensor([2, 0, 4], dtype=torch.int32, device=cuda))
    assert ops.device_status() == 0
    _check(out, x, w4, s, [2, 0, 4], 256)


def test_weights_past_four_gigabytes(cuda):
    # the last groups' words lie past 2^32 bytes
    G, K, N = 40, 7168, 8192
    w4 = torch.zeros((G, K // 8, N), dtype=torch.int32, device=cuda)
    s = torch.ones((G, K // 128, N), device=cuda)
    small, _ = _weights(cuda, 1, K, N, seed=11)
    w4[G - 1] = small[0]
    x = _x(cuda, 1, K, seed=12)
    sizes = torch.zeros(G, dtype=torch.int32, device=cuda)
    sizes[G - 1] = 1
    out = ops.gmm_w4_fwd(x, w4, s, sizes)
    want = ops.gmm_w4_fwd(x, small, s[:1], torch.ones(1, dtype=torch.int32, device=cuda))
    assert torch.equal(out, want)


def test_graph_replays_share_nothing(cuda):
    """Two captured products on two streams, each with its own workspace."""
    w4, s = _weights(cuda, 8, 1024, 256)
    gs = torch.tensor([1, 0, 2, 0, 0, 1, 0, 0], dtype=torch.int32, device=cuda)
    xs = [_x(cuda, 4, 1024, seed=i) for i in (1, 2)]
    want = [ops.gmm_w4_fwd(x, w4, s, gs) for x in xs]
    graphs, outs = [], []
    for x in xs:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.gmm_w4_fwd(x, w4, s, gs)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.gmm_w4_fwd(x, w4, s, gs))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def _weighs_only_what_it_meets(out, x, q, s, sizes):
    """_check with |q| for |q| + 16: an x whose weight is 0 adds nothing, also no error."""
    row, K = 0, x.shape[1]
    for g, n in enumerate(sizes):
        sc = s[g].to(F64).repeat_interleave(128, 0)
        xr = x[row:row + n].to(F64)
        ref, mag = xr @ (q[g].to(F64) * sc), xr.abs() @ (q[g].abs().to(F64) * sc)
        tol = (8 * 2.0 ** -22 + (K / 128 + 16) * 2.0 ** -24) * mag
        err = (out[row:row + n].to(F64) - ref).abs()
        assert (err <= tol).all(), (g, float((err / mag).max()))
        row += n


@pytest.mark.parametrize("large", [1e2, 1e4, 1e6, 1e20, 1e38])
@pytest.mark.parametrize("K,N,sizes", [(128, 32, [1]), (1024, 96, [3, 0, 9]), (7168, 512, [1])])
def test_large_x_against_weights_of_zero(cuda, K, N, sizes, large):
    # outliers in some features, as in front of a down projection: their weights
    # are 0 in every column, so the output is that of the other features
    w4, s = _weights(cuda, len(sizes), K, N, seed=15)
    at = torch.arange(0, K, 37, device=cuda)
    for k in at.tolist():
        word, bit = w4[:, k // 8], 4 * (k % 8)
        eight = 8 << bit
        w4[:, k // 8] = (word & ~torch.tensor(15 << bit, device=cuda).to(torch.int32)) | \
            torch.tensor(eight - 2 ** 32 if eight >= 2 ** 31 else eight, device=cuda).to(torch.int32)
    q = _unpack(w4)
    assert (q[:, at] == 0).all()
    x = _x(cuda, sum(sizes), K, seed=16)
    gs = torch.tensor(sizes, dtype=torch.int32, device=cuda)
    x[:, at] = (x[:, at].float().sign() * large).to(BF16)
    out = ops.gmm_w4_fwd(x, w4, s, gs)
    _weighs_only_what_it_meets(out, x, q, s, sizes)
    x[:, at] = 0
    assert torch.equal(ops.gmm_w4_fwd(x, w4, s, gs), out)
    assert ops.device_status() == 0


def test_small_x_beside_large_ones(cuda):
    # a column reads features 2^-20 to 2^-45 of the block's largest: every one in full
    K, N = 128, 32
    x = torch.full((8, K), 3.0, device=cuda)
    small = (1 + torch.arange(8, device=cuda) / 128) * 2.0 ** -torch.arange(20, 52, 4, device=cuda)
    x[:, 40:48] = small
    x = x.to(BF16)
    q = torch.zeros((K, N), dtype=torch.int64, device=cuda)
    q[40:48] = torch.eye(8, dtype=torch.int64, device=cuda).repeat(1, 4) * 5  # column n reads feature 40 + n % 8
    word = torch.zeros((K // 8, N), dtype=torch.int64, device=cuda)
    for j in range(8):
        word |= (q[j::8] + 8) << (4 * j)
    w4 = torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)[None].contiguous()
    out = ops.gmm_w4_fwd(x, w4, torch.ones((1, 1, N), device=cuda), torch.tensor([8], dtype=torch.int32, device=cuda))
    want = x[:, 40:48].float().repeat(1, 4) * 5
    assert torch.equal(out, want)


@pytest.mark.parametrize("K,N,sizes", [(14336, 512, [1]), (7168, 512, [8]), (7168, 1024, [3, 0, 2, 5])])
def test_jobs_of_many_ctas_are_the_same_every_time(cuda, K, N, sizes):
    # every tile's k is cut among CTAs, and whichever of them is last adds all parts
    w4, s = _weights(cuda, len(sizes), K, N, seed=13)
    x = _x(cuda, sum(sizes), K, seed=14)
    gs = torch.tensor(sizes, dtype=torch.int32, device=cuda)
    first = ops.gmm_w4_fwd(x, w4, s, gs)
    _check(first, x, w4, s, sizes, K)
    busy = torch.empty(1 << 27, dtype=torch.uint8, device=cuda)
    for i in range(100):
        if i % 2:
            busy.fill_(i)  # the parts leave the caches, the CTAs start at other times
        assert torch.equal(ops.gmm_w4_fwd(x, w4, s, gs), first)
    assert ops.device_status() == 0


def test_refusals(cuda):
    w4, s = _weights(cuda, 2, 256, 64)
    x, gs = _x(cuda, 4, 256), torch.tensor([2, 2], dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="x must"):
        ops.gmm_w4_fwd(x.float(), w4, s, gs)
    with pytest.raises(ValueError, match="w4 must"):
        ops.gmm_w4_fwd(x[:, :128].contiguous(), w4, s, gs)
    with pytest.raises(ValueError, match="s must"):
        ops.gmm_w4_fwd(x, w4, s[:, :1].contiguous(), gs)
    with pytest.raises(ValueError, match="group_sizes"):
        ops.gmm_w4_fwd(x, w4, s, gs[:1])
    with pytest.raises(ValueError, match="group_sizes"):
        ops.gmm_w4_fwd(x, w4, s, gs.long())
    with pytest.raises(ValueError, match="out_dtype"):
        ops.gmm_w4_fwd(x, w4, s, gs, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="out must"):
        ops.gmm_w4_fwd(x, w4, s, gs, out=torch.empty((3, 64), device=cuda))
    with pytest.raises(ValueError, match="3-D bf16"):
        ops.quant_w4_128x1(x)
    with pytest.raises(_lib.GlaucisError, match="128"):
        ops.quant_w4_128x1(torch.zeros((1, 200, 64), dtype=BF16, device=cuda))
    with pytest.raises(_lib.GlaucisError, match="32"):
        ops.quant_w4_128x1(torch.zeros((1, 256, 40), dtype=BF16, device=cuda))
