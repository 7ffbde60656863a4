"""Measured cases of the operators around the experts' products of a mixture-of-experts layer:

  norm      RMS norm with the residual's addition, output in e4m3 with 1x128 scales; training in bf16
  route     top-k routing with counts, rows in expert order and the balance loss; and its gradients
  exchange  rows into expert order and back (weighted sum), in bf16 and as e4m3 with scales; and its gradients
  w4        grouped products with 4-bit weights and 128x1 scales for few rows

`run` computes the plain form in 32 bits with elementary torch operations, or, with `own` set, calls
the package's operators.  Sizes are those of the package's configurations (gmm_small, gmm_moe_up,
gmm_dense_expert) and ragged ones between them.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn


def listed():
    return [
        # one generated token, the residual stream added, ready for the experts' first product
        dict(name="norm_quant_decode", op="norm", mode="quant", M=1, K=7168, residual=True, w32=False),
        # the prompt batch of the activation quantiser's own measurements
        dict(name="norm_quant_prefill", op="norm", mode="quant", M=16384, K=7168, residual=True, w32=False),
        # training step of a ragged batch, master weights in 32 bits
        dict(name="norm_train", op="norm", mode="train", M=4099, K=4096, residual=True, w32=True),
        # three sequences generating, 128 experts, top 8
        dict(name="route_decode", op="route", mode="serve", T=3, E=128, k=8, bf16=False, renorm=True, off=4, pad=0.0),
        # the 4096 tokens of gmm_moe_up, bf16 logits, a sixteenth of the rows padding
        dict(name="route_prefill", op="route", mode="serve", T=4096, E=128, k=8, bf16=True, renorm=True, off=4, pad=0.0625),
        # training step of a large batch, loss and weights differentiated
        dict(name="route_train", op="route", mode="train", T=32771, E=128, k=8, bf16=False, renorm=True, off=0, pad=0.0),
        # four sequences generating: rows out and weighted sum back onto the residual
        dict(name="exchange_decode", op="exchange", mode="serve", T=4, k=8, K=7168, E=128, y32=False, pad=0.0),
        # the rows of gmm_moe_up as the experts' first product takes them
        dict(name="exchange_fp8_prefill", op="exchange", mode="fp8", T=4096, k=8, K=7168, E=128, y32=False, pad=0.0),
        # training step with 8 dense experts, top 2, a ragged batch with padding
        dict(name="exchange_train", op="exchange", mode="train", T=16387, k=2, K=4096, E=8, y32=False, pad=0.03),
        # one token through two of 8 small experts: latency
        dict(name="w4_small", op="w4", M=2, G=8, K=1024, N=1024, topk=2, out32=False),
        # one token through 8 of 128 experts
        dict(name="w4_one_token", op="w4", M=8, G=128, K=7168, N=2048, topk=8, out32=False),
        # sixteen sequences generating
        dict(name="w4_batch", op="w4", M=128, G=128, K=7168, N=2048, topk=8, out32=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "route", "exchange", "w4"])
    if op == "norm":
        mode = rng.choice(["quant", "train"])
        # the 8-bit output has blocks of 128 features; the bf16 one takes vectors of 8
        K = 128 * _log_int(rng, 4, 64) if mode == "quant" else 8 * _log_int(rng, 16, 1024)
        most = 16384 * 7168 if mode == "quant" else 8192 * 4096
        M = _log_int(rng, 1, min(32768, most // K))
        return dict(op=op, mode=mode, M=M, K=K, residual=rng.random() < 0.75, w32=rng.random() < 0.5)
    if op == "route":
        mode = rng.choice(["serve", "train"])
        E = _log_int(rng, 4, 384)
        T = _log_int(rng, 1, min(65536, 32771 * 128 // E))
        off = rng.choice([0, 0, E // 32])
        return dict(op=op, mode=mode, T=T, E=E, k=rng.randint(1, min(8, E - off)), bf16=rng.random() < 0.5,
                    renorm=rng.random() < 0.7, off=off, pad=rng.choice([0.0, 0.0, 0.1, 0.5]))
    if op == "exchange":
        mode = rng.choice(["serve", "fp8", "train"])
        k, E = rng.choice([(1, 8), (2, 8), (4, 60), (6, 64), (8, 128), (8, 256)])
        K = 128 * _log_int(rng, 4, 64) if mode == "fp8" else 8 * _log_int(rng, 64, 1024)
        most = (2 if mode == "fp8" else 1) * 16387 * 2 * 4096 // (k * K)
        return dict(op=op, mode=mode, T=_log_int(rng, 1, min(16384, most)), k=k, K=K, E=E,
                    y32=mode != "fp8" and rng.random() < 0.4, pad=rng.choice([0.0, 0.0, 0.1]))
    G, topk = rng.choice([(1, 1), (8, 2), (60, 4), (64, 6), (128, 8)])
    K, N = 128 * _log_int(rng, 4, 56), 128 * _log_int(rng, 4, 56)
    while G * K * N > 128 * 7168 * 2048:
        K, N = max(128, K // 256 * 128), max(128, N // 256 * 128)
    M = _log_int(rng, 1, max(1, min(128, 128 * 7168 * 2048 // (K * N))))
    return dict(op=op, M=M, G=G, K=K, N=N, topk=topk, out32=rng.random() < 0.4)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _popularity(g, E):
    """Logit of each expert's popularity: rank^-1.2 over a seeded order."""
    rank = torch.rand(E, generator=g, device="cuda").argsort().float() + 1.0
    return -1.2 * rank.log()


def _choices(g, T, E, k, pad):
    """Distinct choices of every token by popularity (int64 [T, k]); padding rows have -1."""
    u = torch.rand((T, E), generator=g, device="cuda").clamp_min(1e-20)
    ids = (_popularity(g, E) - (-u.log()).log()).topk(k, dim=1).indices
    if pad:
        ids[int(T * (1 - pad)):] = -1
    return ids


def _order(ids, E):
    """Rows of the choices in expert order, -1 for none (int32, as ids), and int32 [E] counts."""
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, E, flat)
    row = torch.empty_like(flat)
    row[torch.sort(key, stable=True).indices] = torch.arange(flat.numel(), device=flat.device)
    counts = (key[:, None] == torch.arange(E, device=flat.device)).sum(0)
    return torch.where(flat < 0, -1, row).int().reshape(ids.shape), counts.int()


def prepare(case, seed):
    g, c = _gen(seed), case
    if c["op"] == "norm":
        M, K = c["M"], c["K"]
        s = dict(case=c, x=_rand(g, M, K).to(BF16), res=(_rand(g, M, K) * 2).to(BF16) if c["residual"] else None,
                 w=(1 + 0.1 * _rand(g, K)).to(F32 if c["w32"] else BF16))
        if c["mode"] == "train":
            s["dy"] = (_rand(g, M, K) * 0.1).to(BF16)
            s["dh"] = (_rand(g, M, K) * 0.1).to(BF16) if c["residual"] else None
        return s
    if c["op"] == "route":
        T, E = c["T"], c["E"]
        bias = _popularity(g, E)
        if c["off"]:
            bias[bias.argsort()[:c["off"]]] = -math.inf
        s = dict(case=c, logits=(_rand(g, T, E) * 1.5 + bias).to(BF16 if c["bf16"] else F32), mask=None)
        if c["pad"]:
            s["mask"] = torch.arange(T, device="cuda") < T - int(T * c["pad"])
            s["logits"][T - int(T * c["pad"]):] = math.nan  # what padding holds is of no meaning
        if c["mode"] == "train":
            s["dw"] = _rand(g, T, c["k"])
            s["dloss"] = torch.rand((), generator=g, device="cuda") + 0.5
        return s
    if c["op"] == "exchange":
        T, k, K = c["T"], c["k"], c["K"]
        pos, sizes = _order(_choices(g, T, c["E"], k, c["pad"]), c["E"])
        s = dict(case=c, pos=pos, sizes=sizes)
        if c["mode"] == "fp8":
            s["q"] = (_rand(g, T, K) * 100).clamp(-448, 448).to(E4M3)
            s["s"] = _rand(g, T, K // 128).abs() * 0.01 + 1e-3
            return s
        s["x"] = _rand(g, T, K).to(BF16)
        s["y"] = _rand(g, T * k, K).to(F32 if c["y32"] else BF16)
        s["w"] = torch.where(pos < 0, 0.0, torch.softmax(_rand(g, T, k), 1))
        s["res"] = _rand(g, T, K).to(BF16)
        if c["mode"] == "train":
            s["dout"] = (_rand(g, T, K) * 0.1).to(BF16)
            s["dxs"] = (_rand(g, T * k, K) * 0.1).to(BF16)
        return s
    M, G, K, N = c["M"], c["G"], c["K"], c["N"]
    ids = _choices(g, -(-M // c["topk"]), G, c["topk"], 0.0).reshape(-1)[:M]
    # all 16 values alike: wider than a quantised normal distribution, so sums cancel less
    w4 = torch.randint(-2 ** 31, 2 ** 31, (G, K // 8, N), generator=g, device="cuda", dtype=torch.int32)
    return dict(case=c, x=_rand(g, M, K).to(BF16), w4=w4, s=(_rand(g, G, K // 128, N).abs() + 0.5) * 0.005,
                sizes=_order(ids, G)[1])


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    op, c = state["case"]["op"], state["case"]
    if own:
        return {"norm": _own_norm, "route": _own_route, "exchange": _own_exchange, "w4": _own_w4}[op](state, c)
    return {"norm": _norm, "route": _route, "exchange": _exchange, "w4": _w4}[op](state, c)


def _own_norm(st, c):
    from glaucis_b200 import ops
    if c["mode"] == "quant":
        return ops.rms_norm_quant_1x128(st["x"], st["w"], EPS, residual=st["res"])
    f = ops.rms_norm_fwd(st["x"], st["w"], EPS, residual=st["res"])
    dx, dw = ops.rms_norm_bwd(st["dy"], f.h, st["w"], f.rstd, dh=st["dh"])
    return (f.y, f.h, dx, dw) if c["residual"] else (f.y, dx, dw)


def _own_route(st, c):
    from glaucis_b200 import ops
    r = ops.moe_route_fwd(st["logits"], c["k"], mask=st["mask"], renormalize=c["renorm"])
    out = [r.ids, r.weights, r.counts, r.pos, r.balance_loss]
    if c["mode"] == "train":
        out.append(ops.moe_route_bwd(st["logits"], r, st["dw"], st["dloss"]))
    return out


def _own_exchange(st, c):
    from glaucis_b200 import ops
    if c["mode"] == "fp8":
        return ops.moe_dispatch_quant(st["q"], st["s"], st["pos"], st["sizes"])
    xs = ops.moe_dispatch(st["x"], st["pos"], st["sizes"])
    out = ops.moe_combine(st["y"], st["pos"], st["w"], st["sizes"], residual=st["res"])
    if c["mode"] == "serve":
        return xs, out
    dy, dw = ops.moe_combine_bwd(st["dout"], st["y"], st["pos"], st["w"], st["sizes"])
    return xs, out, dy, dw, ops.moe_dispatch_bwd(st["dxs"], st["pos"])


def _own_w4(st, c):
    from glaucis_b200 import ops
    return ops.gmm_w4_fwd(st["x"], st["w4"], st["s"], st["sizes"], out_dtype=F32 if c["out32"] else BF16)


def _norm(st, c):
    h = st["x"] if st["res"] is None else (st["x"].float() + st["res"].float()).to(BF16)
    hf, w = h.float(), st["w"].float()
    r = 1.0 / torch.sqrt((hf * hf).mean(1, keepdim=True) + EPS)
    y = hf * r * w
    if c["mode"] == "quant":
        b = y.reshape(c["M"], -1, 128)
        s = b.abs().amax(2) / 448.0
        s = torch.where(s == 0, 1.0, s)
        q = (b / s[:, :, None]).to(E4M3).reshape(c["M"], c["K"])
        return (q, s, h) if c["residual"] else (q, s)
    xh, dy = hf * r, st["dy"].float()
    u = dy * w
    dx = r * (u - xh * (u * xh).mean(1, keepdim=True))
    if st["dh"] is not None:
        dx = dx + st["dh"].float()
    out = (y.to(BF16), dx.to(BF16), (dy * xh).sum(0).to(st["w"].dtype))
    return (out[0], h) + out[1:] if c["residual"] else out


def _route(st, c):
    T, E, k = c["T"], c["E"], c["k"]
    z = st["logits"].float()
    live = (z > -math.inf).any(1)
    if st["mask"] is not None:
        live = live & st["mask"]
    z = torch.where(live[:, None], z, 0.0)
    p = (z - z.amax(1, keepdim=True)).exp()
    p = torch.where(live[:, None], p / p.sum(1, keepdim=True), 0.0)
    top = torch.sort(z, dim=1, descending=True, stable=True)
    ok = live[:, None] & (top.values[:, :k] > -math.inf)
    ids = torch.where(ok, top.indices[:, :k], -1)
    w = torch.where(ok, p.gather(1, ids.clamp_min(0)), 0.0)
    total = w.sum(1, keepdim=True)
    total = torch.where(total == 0, 1.0, total)
    if c["renorm"]:
        w = w / total
    pos, counts = _order(ids, E)
    n = live.sum().clamp_min(1).float()
    f = counts.float() / counts.sum().clamp_min(1).float()
    loss = E * (f * (p.sum(0) / n)).sum()
    out = [ids.int(), w, counts, pos, loss]
    if c["mode"] == "train":
        dsel = torch.where(ok, st["dw"], 0.0)
        if c["renorm"]:
            dsel = torch.where(ok, (dsel - (dsel * w).sum(1, keepdim=True)) / total, 0.0)
        dp = (st["dloss"] * E / n * f).repeat(T, 1).scatter_add(1, ids.clamp_min(0), dsel)
        out.append((p * (dp - (p * dp).sum(1, keepdim=True))).to(st["logits"].dtype))
    return out


def _gather(y, pos):
    """float [T, k, K]: row pos of y, zeros where pos is -1."""
    y = torch.cat([y, y.new_zeros(1, y.shape[1])])
    return y[torch.where(pos < 0, y.shape[0] - 1, pos).long()].float()


def _sources(pos, R):
    """int64 [R]: the choice t * k + j of every row in expert order, T * k for a row without one."""
    flat = pos.reshape(-1).long()
    src = torch.full((R + 1,), flat.numel(), dtype=torch.long, device=pos.device)
    src[torch.where(flat < 0, R, flat)] = torch.arange(flat.numel(), device=pos.device)
    return torch.where(torch.arange(R + 1, device=pos.device) == R, flat.numel(), src)[:R]


def _scatter(x, pos, fill=0):
    """[T * k, K]: row t of x at every pos[t, j], `fill` elsewhere."""
    x = torch.cat([x, torch.full_like(x[:1], fill)])
    return x[_sources(pos, pos.numel()) // pos.shape[1]]


def _exchange(st, c):
    T, k, pos = c["T"], c["k"], st["pos"]
    if c["mode"] == "fp8":
        return _scatter(st["q"].view(torch.uint8), pos).view(E4M3), _scatter(st["s"], pos, 1)
    xs = _scatter(st["x"], pos)
    y, w = _gather(st["y"], pos), st["w"]
    out = ((y * w[:, :, None]).sum(1) + st["res"].float()).to(BF16)
    if c["mode"] == "serve":
        return xs, out
    do = st["dout"].float()
    dw = torch.where(pos < 0, 0.0, (y * do[:, None, :]).sum(2))
    src = _sources(pos, T * k)
    wr = torch.cat([w.reshape(-1), w.new_zeros(1)])[src]
    dy = wr[:, None] * torch.cat([do, do.new_zeros(1, c["K"])])[src // k]
    return xs, out, dy.to(st["y"].dtype), dw, _gather(st["dxs"], pos).sum(1).to(BF16)


def _w4(st, c):
    M, G, K, N = c["M"], c["G"], c["K"], c["N"]
    end = st["sizes"].long().cumsum(0)
    g = (torch.arange(M, device="cuda")[:, None] >= end).sum(1)  # group of each row
    at = g.clamp_max(G - 1)
    word = st["w4"][at]
    shift = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    q = ((word[:, :, None, :] >> shift[:, None]) & 15) - 8
    w = q.reshape(M, K // 128, 128, N).float() * st["s"][at][:, :, None, :]
    out = (st["x"].float()[:, None, :] @ w.reshape(M, K, N))[:, 0]
    return torch.where((g < G)[:, None], out, 0.0).to(F32 if c["out32"] else BF16)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "norm":
        n, wb = c["M"] * c["K"], 4 if c["w32"] else 2
        add = 4 if c["residual"] else 0  # the residual in, the sum out
        if c["mode"] == "quant":
            return dict(bytes=n * (2 + add + 1) + n // 128 * 4 + c["K"] * wb, flops=8 * n)
        dh = 2 if c["residual"] else 0
        # forward: x, residual, y, h; backward: dy, dh, h (or x) again, dx
        return dict(bytes=n * (2 + add + 2 + 2 + dh + 2 + 2) + 3 * c["K"] * wb, flops=20 * n)
    if c["op"] == "route":
        n, lb = c["T"] * c["E"], 2 if c["bf16"] else 4
        b = n * lb + 12 * c["T"] * c["k"] + 4 * c["E"]
        if c["mode"] == "train":
            b += 2 * n * lb + 12 * c["T"] * c["k"]
        return dict(bytes=b, flops=(6 if c["mode"] == "serve" else 14) * n)
    if c["op"] == "exchange":
        T, R, K, k = c["T"], c["T"] * c["k"], c["K"], c["k"]
        if c["mode"] == "fp8":
            return dict(bytes=(T + R) * (K + K // 128 * 4) + 4 * R, flops=0)
        yb = 4 if c["y32"] else 2
        b = (T + R) * K * 2 + R * K * yb + 2 * T * K * 2 + 8 * R
        if c["mode"] == "serve":
            return dict(bytes=b, flops=2 * R * K)
        # backward: dout and y in, dy out; the rows' gradients in, the tokens' out
        b += T * K * 2 + 2 * R * K * yb + R * K * 2 + T * K * 2 + 8 * R
        return dict(bytes=b, flops=7 * R * K)
    rows, G, K, N = c["M"], c["G"], c["K"], c["N"]
    # groups that a token reaches are distinct; those of several tokens overlap by popularity
    tokens = -(-rows // c["topk"])
    rank = np.arange(1, G + 1) ** -1.2
    hit = float((1 - (1 - np.minimum(1.0, c["topk"] * rank / rank.sum())) ** tokens).sum())
    hit = min(hit if tokens > 1 else rows, rows, G)
    return dict(bytes=hit * K * N * (0.5 + 4 / 128) + rows * K * 2 + rows * N * (4 if c["out32"] else 2),
                flops=2 * rows * K * N)


# ---------------------------------------------------------------------------
# The same from the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "route": _exact_route, "exchange": _exact_exchange, "w4": _exact_w4}[case["op"]](
        st, case)


def _exact_norm(st, c):
    x, w = st["x"].to(F64), st["w"].to(F64)
    h = x + st["res"].to(F64) if c["residual"] else x
    hr = h.to(BF16).to(F64)  # the stored sum is what the norm takes
    rms = (hr.square().sum(1) / c["K"] + EPS).sqrt()[:, None]
    y = hr / rms * w
    if c["mode"] == "quant":
        scale = torch.stack([b.abs().max(1).values for b in y.split(128, dim=1)], 1) / 448
        scale[scale == 0] = 1
        q = y / scale.repeat_interleave(128, 1)
        return (q, scale, h) if c["residual"] else (q, scale)
    dy = st["dy"].to(F64)
    # d/dh of sum(dy * w * h / rms(h)): the quotient rule
    dx = dy * w / rms - hr * ((dy * w * hr).sum(1, keepdim=True) / c["K"]) / rms ** 3
    if c["residual"]:
        dx = dx + st["dh"].to(F64)
    dw = torch.einsum("mk,mk->k", dy, hr / rms)
    return (y, h, dx, dw) if c["residual"] else (y, dx, dw)


def _exact_route(st, c):
    T, E, k = c["T"], c["E"], c["k"]
    z = st["logits"].double().cpu().numpy()
    live = np.isfinite(z).any(1)
    if st["mask"] is not None:
        live &= st["mask"].cpu().numpy()
    rows = np.flatnonzero(live)
    zl = z[rows]
    e = np.exp(zl - zl.max(1, keepdims=True))
    p = e / e.sum(1, keepdims=True)
    ids = np.full((T, k), -1)
    ids[rows] = np.argsort(-zl, axis=1, kind="stable")[:, :k]
    w = np.zeros((T, k))
    w[rows] = np.take_along_axis(p, ids[rows], 1)
    total = w[rows].sum(1, keepdims=True)
    if c["renorm"]:
        w[rows] /= total
    counts = np.bincount(ids[rows].ravel(), minlength=E)
    flat = ids.ravel()
    pos = np.full(T * k, -1)
    valid = np.flatnonzero(flat >= 0)
    pos[valid[np.argsort(flat[valid], kind="stable")]] = np.arange(valid.size)
    n, f = max(1, rows.size), counts / max(1, counts.sum())
    loss = E * float(f @ p.sum(0)) / n
    out = [ids, w, counts, pos.reshape(T, k), loss]
    if c["mode"] == "train":
        dw = st["dw"].double().cpu().numpy()[rows]
        if c["renorm"]:
            dw = (dw - (dw * w[rows]).sum(1, keepdims=True)) / total
        dp = np.tile(float(st["dloss"]) * E * f / n, (rows.size, 1))
        np.put_along_axis(dp, ids[rows], np.take_along_axis(dp, ids[rows], 1) + dw, 1)
        dz = np.zeros((T, E))
        dz[rows] = p * (dp - (p * dp).sum(1, keepdims=True))
        out.append(dz)
    return [torch.from_numpy(v.astype(np.int32)) if isinstance(v, np.ndarray) and v.dtype.kind == "i"
            else torch.as_tensor(v, dtype=F64) for v in out]


def _exact_exchange(st, c):
    T, k, K, pos = c["T"], c["k"], c["K"], st["pos"].long()
    t, j = torch.nonzero(pos >= 0, as_tuple=True)
    at = pos[t, j]
    if c["mode"] == "fp8":
        q = torch.zeros((T * k, K), dtype=F32, device=pos.device)
        q[at] = st["q"].float()[t]
        s = torch.ones((T * k, K // 128), dtype=F64, device=pos.device)
        s[at] = st["s"].to(F64)[t]
        return q, s
    zeros = torch.zeros((T * k, K), dtype=F64, device=pos.device)
    xs = zeros.index_copy(0, at, st["x"].to(F64)[t])
    part = st["y"].to(F64)[at]
    w = st["w"].to(F64)[t, j][:, None]
    out = st["res"].to(F64).index_add(0, t, part * w)
    if c["mode"] == "serve":
        return xs, out
    do = st["dout"].to(F64)[t]
    dy = zeros.index_copy(0, at, do * w)
    dw = torch.zeros((T, k), dtype=F64, device=pos.device)
    dw[t, j] = (part * do).sum(1)
    dx = torch.zeros((T, K), dtype=F64, device=pos.device).index_add(0, t, st["dxs"].to(F64)[at])
    return xs, out, dy, dw, dx


def _exact_w4(st, c):
    def product(g, x):
        u = st["w4"][g].to(torch.int64) & 0xFFFFFFFF
        q = torch.stack([(u >> (4 * j)) % 16 for j in range(8)], 1).reshape(c["K"], c["N"]).to(F64) - 8
        return x.to(F64) @ (q * st["s"][g].to(F64).repeat_interleave(128, 0))

    rows = torch.split(st["x"], st["sizes"].tolist())
    return torch.cat([product(g, x) for g, x in enumerate(rows) if x.shape[0]])
