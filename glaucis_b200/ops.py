"""Torch-facing ops over the C ABI.  Tensors must live on a CUDA device; every
op launches on the current stream and never falls back to another backend.

Op names and argument meaning mirror the Glaucis kernel templates
(KE/examples/kernels/gmm_fp8_blockwise.py, KE/examples/kernels/chunk_gla.py).
The operators around the grouped matmul (rms_norm*, moe_*, gmm_w4_fwd) have no
counterpart there.
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

FP8 = torch.float8_e4m3fn
TILE = 128


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# The current stream's handle without building a Stream object (3 us a call);
# CUDA is initialised where there is a tensor to launch on.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream() -> int:
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_current_device())


def _need_cuda(*ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("glaucis_b200 ops take CUDA tensors (no CPU path)")
        if not t.is_contiguous():
            raise ValueError("glaucis_b200 ops take contiguous tensors")


# ---------------------------------------------------------------------------
# Block-wise FP8 quantisers
# ---------------------------------------------------------------------------
def _out(t: Optional[torch.Tensor], shape, dtype, device, name: str) -> torch.Tensor:
    """A preallocated contiguous output of the given shape / dtype, or a new one."""
    if t is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")
    return t


def quant_act_1x128(x: torch.Tensor, q: Optional[torch.Tensor] = None,
                    s: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 [M, K] -> (e4m3 [M, K], fp32 scales [M, K/128]); `q` / `s` may be
    given as preallocated outputs.

    Replaces qwix.pallas.quantize(lhs, channelwise_axes=[0], tiled_axes={1: 128},
    absmax, fp32 scale) at KE/examples/kernels/gmm_fp8_blockwise.py:84-91.
    """
    _need_cuda(x)
    if x.dtype != torch.bfloat16 or x.dim() != 2:
        raise ValueError("quant_act_1x128 expects a 2-D bf16 tensor")
    M, K = x.shape
    q = _out(q, (M, K), FP8, x.device, "q")
    s = _out(s, (M, K // TILE), torch.float32, x.device, "s")
    lib = _lib.load()
    _lib.check(lib.gl_quant_act_1x128(x.data_ptr(), M, K, q.data_ptr(), s.data_ptr(), None,
                                      _stream()), "gl_quant_act_1x128")
    return q, s


def quant_w_128x128(w: torch.Tensor, q: Optional[torch.Tensor] = None,
                    s: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 [G, K, N] -> (e4m3 [G, K, N], fp32 scales [G, K/128, N/128]);
    `q` / `s` may be given as preallocated outputs.

    Replaces qwix.pallas.quantize(rhs, channelwise_axes=[0],
    tiled_axes={1: 128, 2: 128}) at KE/examples/kernels/gmm_fp8_blockwise.py:100-107.
    """
    _need_cuda(w)
    if w.dtype != torch.bfloat16 or w.dim() != 3:
        raise ValueError("quant_w_128x128 expects a 3-D bf16 tensor")
    G, K, N = w.shape
    q = _out(q, (G, K, N), FP8, w.device, "q")
    s = _out(s, (G, K // TILE, N // TILE), torch.float32, w.device, "s")
    lib = _lib.load()
    _lib.check(lib.gl_quant_w_128x128(w.data_ptr(), G, K, N, q.data_ptr(), s.data_ptr(), None,
                                      _stream()), "gl_quant_w_128x128")
    return q, s


# ---------------------------------------------------------------------------
# Grouped matmul
# ---------------------------------------------------------------------------
def gmm_fp8_fwd(a_q: torch.Tensor, a_s: torch.Tensor, b_q: torch.Tensor, b_s: torch.Tensor,
                group_sizes: torch.Tensor, out_dtype: torch.dtype = torch.float32,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped matmul on pre-quantised operands (QArray-equivalent inputs).

    Replaces tokamax pallas_mosaic_tpu_kernel.gmm(lhs=QArray, rhs=QArray,
    group_sizes, out_dtype, transpose_rhs=False) at
    KE/examples/kernels/gmm_fp8_blockwise.py:109-119.  Rows at or beyond
    sum(group_sizes) are zero.
    """
    _need_cuda(a_q, a_s, b_q, b_s, group_sizes)
    M, K = a_q.shape
    G, K2, N = b_q.shape
    if K2 != K:
        raise ValueError(f"K mismatch: lhs {K} vs rhs {K2}")
    if group_sizes.dtype != torch.int32 or group_sizes.numel() != G:
        raise ValueError("group_sizes must be int32 [G]")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("out_dtype must be bf16 or fp32")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=a_q.device)
    code = _lib.GL_OUT_F32 if out.dtype == torch.float32 else _lib.GL_OUT_BF16
    lib = _lib.load()
    _lib.check(lib.gl_gmm_fp8_fwd(a_q.data_ptr(), a_s.data_ptr(), b_q.data_ptr(), b_s.data_ptr(),
                                  group_sizes.data_ptr(), G, M, K, N, out.data_ptr(), code, None,
                                  _stream()), "gl_gmm_fp8_fwd")
    return out


def _zero_tail_rows(out: torch.Tensor, group_sizes: torch.Tensor) -> None:
    # Rows past sum(group_sizes) belong to no group: zero them on the device
    # without a host round trip.
    M = out.shape[0]
    total = group_sizes.sum()
    rows = torch.arange(M, device=out.device)
    out.masked_fill_((rows >= total).unsqueeze(1), 0)


def gmm_fp8_blockwise(lhs: torch.Tensor, rhs: torch.Tensor, group_sizes: torch.Tensor,
                      tiling: tuple = (256, 512, 256, 256, 512, 128, 1024, 512, 128),
                      out_dtype: torch.dtype = torch.float32,
                      zero_unassigned_rows: bool = True) -> torch.Tensor:
    """Forward of the Glaucis `gmm_fp8_blockwise(lhs, rhs, group_sizes, tiling)`
    (KE/examples/kernels/gmm_fp8_blockwise.py:53-120): quantise lhs 1x128 and
    rhs 128x128 to e4m3 with fp32 absmax scales, then the grouped matmul with
    per-K-block fp32 promotion.  `tiling` is accepted for signature
    compatibility; the B200 kernel's tiles are fixed (128x256x128).
    """
    del tiling
    if torch.is_grad_enabled() and (lhs.requires_grad or rhs.requires_grad):
        # differentiable path: backward = gmm_fp8_blockwise_bwd
        return _GmmFp8Blockwise.apply(lhs, rhs, group_sizes, out_dtype)
    a_q, a_s = quant_act_1x128(lhs)
    b_q, b_s = quant_w_128x128(rhs)
    out = gmm_fp8_fwd(a_q, a_s, b_q, b_s, group_sizes, out_dtype=out_dtype)
    if zero_unassigned_rows:
        _zero_tail_rows(out, group_sizes)
    return out


# ---------------------------------------------------------------------------
# Grouped matmul backward (KE/examples/kernels/gmm_fp8_blockwise.py:123-169)
# ---------------------------------------------------------------------------
def gmm_fp8_fwd_scatter(a_q: torch.Tensor, a_s: torch.Tensor, b_q: torch.Tensor, b_s: torch.Tensor,
                        group_sizes: torch.Tensor, outs, row_offset: int,
                        out_dtype: torch.dtype = torch.bfloat16) -> None:
    """gmm_fp8_fwd whose output rows go to row `row_offset` + m of every
    buffer in `outs` (tensors on this device, or integer device addresses of
    peer-mapped buffers such as shard.PeerBuffers.ptrs), each holding at
    least row_offset + M rows of N elements of `out_dtype`.  Used to assemble
    an expert-sharded output on every rank inside the matmul's epilogue; the
    caller synchronises the ranks after it."""
    _need_cuda(a_q, a_s, b_q, b_s, group_sizes)
    M, K = a_q.shape
    G, K2, N = b_q.shape
    if K2 != K:
        raise ValueError(f"K mismatch: a {K} vs b {K2}")
    ptrs = [o.data_ptr() if isinstance(o, torch.Tensor) else int(o) for o in outs]
    for o in outs:
        if isinstance(o, torch.Tensor) and (o.dtype != out_dtype or o.dim() != 2 or o.shape[1] != N
                                            or o.shape[0] < row_offset + M or not o.is_contiguous()):
            raise ValueError(f"each output must be a contiguous {out_dtype} [>= row_offset + M, N] tensor")
    import ctypes
    arr = (ctypes.c_void_p * len(ptrs))(*ptrs)
    code = _lib.GL_OUT_F32 if out_dtype == torch.float32 else _lib.GL_OUT_BF16
    _lib.check(_lib.load().gl_gmm_fp8_fwd_scatter(a_q.data_ptr(), a_s.data_ptr(), b_q.data_ptr(),
                                                  b_s.data_ptr(), group_sizes.data_ptr(), G, M, K, N,
                                                  ctypes.cast(arr, ctypes.c_void_p), len(ptrs),
                                                  int(row_offset), code, None, _stream()),
               "gl_gmm_fp8_fwd_scatter")


def quant_col_128x1(x: torch.Tensor, q: Optional[torch.Tensor] = None,
                    s: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 [M, C] (M, C multiples of 128) -> (e4m3 [M, C], fp32 scales
    [M/128, C]): one absmax scale per 128 rows of a column.  Replaces
    qpl.quantize(grad, channelwise_axes=[1], tiled_axes={0: 128}) (:135-141)
    and, untransposed, the lhs_t quantisation of the forward (:92-99)."""
    _need_cuda(x)
    if x.dtype != torch.bfloat16 or x.dim() != 2:
        raise ValueError("quant_col_128x1 expects a 2-D bf16 tensor")
    M, C = x.shape
    q = _out(q, (M, C), FP8, x.device, "q")
    s = _out(s, (M // TILE, C), torch.float32, x.device, "s")
    lib = _lib.load()
    _lib.check(lib.gl_quant_col_128x1(x.data_ptr(), M, C, q.data_ptr(), s.data_ptr(), None,
                                      _stream()), "gl_quant_col_128x1")
    return q, s


def gmm_fp8_dlhs(dq: torch.Tensor, ds: torch.Tensor, b_q: torch.Tensor, b_s: torch.Tensor,
                 group_sizes: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dlhs [M, K] = dout x rhs^T per group from dout quantised 1x128 along N
    (quant_act_1x128 of grad [M, N]) and the forward's weight QArray; replaces
    tokamax gmm(..., transpose_rhs=True) (:143-153).  Rows at or beyond
    sum(group_sizes) are left as they are in `out` (zeroed when allocated)."""
    _need_cuda(dq, ds, b_q, b_s, group_sizes)
    M, N = dq.shape
    G, K, N2 = b_q.shape
    if N2 != N:
        raise ValueError(f"N mismatch: dout {N} vs rhs {N2}")
    if out is None:
        out = torch.zeros((M, K), dtype=out_dtype, device=dq.device)
    code = _lib.GL_OUT_F32 if out.dtype == torch.float32 else _lib.GL_OUT_BF16
    lib = _lib.load()
    _lib.check(lib.gl_gmm_fp8_dlhs(dq.data_ptr(), ds.data_ptr(), b_q.data_ptr(), b_s.data_ptr(),
                                   group_sizes.data_ptr(), G, M, K, N, out.data_ptr(), code, None,
                                   _stream()), "gl_gmm_fp8_dlhs")
    return out


def tgmm_fp8(lq: torch.Tensor, ls: torch.Tensor, dq: torch.Tensor, ds: torch.Tensor,
             group_sizes: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """drhs [G, K, N] = per group lhs^T x dout over the group's rows, both
    quantised by quant_col_128x1; replaces tokamax tgmm (:155-165).  Empty
    groups give zeros."""
    _need_cuda(lq, ls, dq, ds, group_sizes)
    M, K = lq.shape
    N = dq.shape[1]
    G = group_sizes.numel()
    if group_sizes.dtype != torch.int32:
        raise ValueError("group_sizes must be int32")
    if out is None:
        out = torch.empty((G, K, N), dtype=out_dtype, device=lq.device)
    code = _lib.GL_OUT_F32 if out.dtype == torch.float32 else _lib.GL_OUT_BF16
    lib = _lib.load()
    _lib.check(lib.gl_tgmm_fp8(lq.data_ptr(), ls.data_ptr(), dq.data_ptr(), ds.data_ptr(),
                               group_sizes.data_ptr(), G, M, K, N, out.data_ptr(), code, None,
                               _stream()), "gl_tgmm_fp8")
    return out


def gmm_fp8_blockwise_bwd(lhs: torch.Tensor, rhs: torch.Tensor, group_sizes: torch.Tensor,
                          grad: torch.Tensor, rhs_q: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                          ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dlhs, drhs) of `gmm_fp8_blockwise(lhs, rhs, group_sizes)` for the
    output gradient `grad` [M, N] (KE/examples/kernels/gmm_fp8_blockwise.py
    :123-169): dout quantised 1x128 along N for dlhs and 128x1 along M for
    drhs, lhs quantised 128x1 along M, the forward's weight QArray (passed as
    `rhs_q` or recomputed).  dlhs has lhs's dtype, drhs rhs's (bf16)."""
    if grad.dtype != torch.bfloat16:
        grad = grad.to(torch.bfloat16)
    grad = grad.contiguous()
    b_q, b_s = rhs_q if rhs_q is not None else quant_w_128x128(rhs)
    dq1, ds1 = quant_act_1x128(grad)
    dlhs = gmm_fp8_dlhs(dq1, ds1, b_q, b_s, group_sizes, out_dtype=lhs.dtype)
    del dq1, ds1
    lq, ls = quant_col_128x1(lhs)
    dq2, ds2 = quant_col_128x1(grad)
    drhs = tgmm_fp8(lq, ls, dq2, ds2, group_sizes, out_dtype=rhs.dtype)
    return dlhs, drhs


class _GmmFp8Blockwise(torch.autograd.Function):
    """custom-VJP pair of the template (gmm_fp8_blockwise.py:71-78)."""

    @staticmethod
    def forward(ctx, lhs, rhs, group_sizes, out_dtype):
        a_q, a_s = quant_act_1x128(lhs)
        b_q, b_s = quant_w_128x128(rhs)
        out = gmm_fp8_fwd(a_q, a_s, b_q, b_s, group_sizes, out_dtype=out_dtype)
        _zero_tail_rows(out, group_sizes)
        ctx.save_for_backward(lhs, rhs, group_sizes, b_q, b_s)
        return out

    @staticmethod
    def backward(ctx, grad):
        lhs, rhs, group_sizes, b_q, b_s = ctx.saved_tensors
        dlhs, drhs = gmm_fp8_blockwise_bwd(lhs, rhs, group_sizes, grad, rhs_q=(b_q, b_s))
        return dlhs, drhs, None, None


_SIDE_STREAMS = {}


def _side_streams(device: torch.device):
    """Three per-device streams (copy-in, compute, copy-out) for the host op."""
    key = device.index if device.index is not None else torch.cuda.current_device()
    if key not in _SIDE_STREAMS:
        with torch.cuda.device(key):
            _SIDE_STREAMS[key] = (torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream())
    return _SIDE_STREAMS[key]


def _plan_chunks(sizes, chunks: int, min_rows: int = 1024):
    """Row ranges [r0, r1) of about equal size over the assigned rows, each
    with the index of its first group and its per-group row counts (a group
    may be split between consecutive chunks)."""
    import numpy as np
    sizes = np.asarray(sizes, dtype=np.int64)
    off = np.concatenate([[0], np.cumsum(sizes)])
    total = int(off[-1])
    n = max(1, min(chunks, total // min_rows if total >= min_rows else 1))
    bounds = [total * i // n for i in range(n + 1)]
    plan = []
    for r0, r1 in zip(bounds[:-1], bounds[1:]):
        if r1 <= r0:
            continue
        g_a = int(np.searchsorted(off, r0, side="right") - 1)
        g_b = int(np.searchsorted(off, r1, side="left") - 1)
        g_a = max(g_a, 0)
        sub = [max(0, min(int(off[g + 1]), r1) - max(int(off[g]), r0)) for g in range(g_a, g_b + 1)]
        plan.append((r0, r1, g_a, sub))
    return plan, total


def gmm_fp8_blockwise_host(lhs: torch.Tensor, rhs: torch.Tensor, group_sizes: torch.Tensor,
                           out: Optional[torch.Tensor] = None,
                           out_dtype: torch.dtype = torch.bfloat16,
                           chunks: int = 16, min_chunk_rows: int = 1024) -> torch.Tensor:
    """`gmm_fp8_blockwise` for activations that arrive in host memory (the
    serving case): `lhs` bf16 [M, K] in pinned host memory, `rhs` bf16
    [G, K, N] on the GPU (the weights), `group_sizes` int32 [G] (host or
    device); returns `out` [M, N] in pinned host memory (allocated when not
    given).  The activation rows go to the device in `chunks` row ranges on a
    copy stream (ranges of at least `min_chunk_rows` rows) while the ranges
    already there are quantised and multiplied on
    a compute stream, and finished output rows go back on a third stream, so
    the PCIe transfers overlap the kernels.  The work is ordered after the
    current stream and the current stream waits for all of it: the result is
    valid once the current stream has been synchronised.  Same numbers as
    `gmm_fp8_blockwise` (row ranges are computed by the same kernel).
    """
    if lhs.is_cuda or not lhs.is_pinned():
        raise ValueError("lhs must be a pinned host tensor")
    _need_cuda(rhs)
    if lhs.dtype != torch.bfloat16 or rhs.dtype != torch.bfloat16 or lhs.dim() != 2 or rhs.dim() != 3:
        raise ValueError("lhs bf16 [M, K] and rhs bf16 [G, K, N] expected")
    M, K = lhs.shape
    G, K2, N = rhs.shape
    if K2 != K:
        raise ValueError(f"K mismatch: lhs {K} vs rhs {K2}")
    if group_sizes.dtype != torch.int32 or group_sizes.numel() != G:
        raise ValueError("group_sizes must be int32 [G]")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, pin_memory=True)
    elif out.is_cuda or not out.is_pinned() or tuple(out.shape) != (M, N) or out.dtype != out_dtype:
        raise ValueError("out must be a pinned host tensor [M, N] of out_dtype")
    sizes = group_sizes.cpu().numpy()
    if (sizes < 0).any() or int(sizes.sum()) > M:
        raise ValueError("group_sizes must be non-negative with sum <= M")
    plan, total = _plan_chunks(sizes, chunks, min_chunk_rows)
    if total < M:
        out[total:].zero_()  # rows that belong to no group
    if total == 0:
        return out
    dev = rhs.device
    s_in, s_c, s_out = _side_streams(dev)
    cur = torch.cuda.current_stream(dev)
    start = cur.record_event()
    for st in (s_in, s_c, s_out):
        st.wait_event(start)
    tab = torch.zeros((len(plan), G), dtype=torch.int32, pin_memory=True)
    for c, (_, _, _, sub) in enumerate(plan):
        tab[c, :len(sub)] = torch.tensor(sub, dtype=torch.int32)
    lhs_d = torch.empty((M, K), dtype=torch.bfloat16, device=dev)
    a_q = torch.empty((M, K), dtype=FP8, device=dev)
    a_s = torch.empty((M, K // TILE), dtype=torch.float32, device=dev)
    out_d = torch.empty((M, N), dtype=out_dtype, device=dev)
    with torch.cuda.stream(s_in):
        tab_d = tab.to(dev, non_blocking=True)
    tab_ready = s_in.record_event()
    with torch.cuda.stream(s_c):
        b_q, b_s = quant_w_128x128(rhs)
        s_c.wait_event(tab_ready)
    for c, (r0, r1, g_a, sub) in enumerate(plan):
        g_b = g_a + len(sub)
        with torch.cuda.stream(s_in):
            lhs_d[r0:r1].copy_(lhs[r0:r1], non_blocking=True)
            landed = s_in.record_event()
        with torch.cuda.stream(s_c):
            s_c.wait_event(landed)
            quant_act_1x128(lhs_d[r0:r1], a_q[r0:r1], a_s[r0:r1])
            gmm_fp8_fwd(a_q[r0:r1], a_s[r0:r1], b_q[g_a:g_b], b_s[g_a:g_b], tab_d[c, :len(sub)],
                        out=out_d[r0:r1])
            done = s_c.record_event()
        with torch.cuda.stream(s_out):
            s_out.wait_event(done)
            out[r0:r1].copy_(out_d[r0:r1], non_blocking=True)
    # keep the device buffers alive for the side streams, then join them
    for t in (lhs_d, a_q, a_s, out_d, tab_d, b_q, b_s):
        for st in (s_in, s_c, s_out):
            t.record_stream(st)
    for st in (s_in, s_c, s_out):
        cur.wait_stream(st)
    return out


# ---------------------------------------------------------------------------
# Chunked GLA forward
# ---------------------------------------------------------------------------
class GLAForward(tuple):
    """Result of chunk_gla_fwd, unpackable as the reference's
    (g_cumsum, A, h, o).  The fused kernel keeps g_cumsum and A on chip, so
    those entries are None unless asked for with output_intermediates=True
    (then fp32 [B, T, H, K] and fp32 [B, T, H, 64], from a separate kernel);
    h (the bf16 state before every chunk, [B, T/64, H, K, V]) is returned
    when asked for with output_states=True, else None; the final state is
    `.ht`."""

    def __new__(cls, o: torch.Tensor, ht: Optional[torch.Tensor], h: Optional[torch.Tensor] = None,
                g_cumsum: Optional[torch.Tensor] = None, A: Optional[torch.Tensor] = None):
        self = tuple.__new__(cls, (g_cumsum, A, h, o))
        self.ht = ht
        return self

    @property
    def g_cumsum(self) -> Optional[torch.Tensor]:
        return self[0]

    @property
    def A(self) -> Optional[torch.Tensor]:
        return self[1]

    @property
    def o(self) -> torch.Tensor:
        return self[3]

    @property
    def h(self) -> Optional[torch.Tensor]:
        return self[2]


def _gla_check(q, k, v, g_gamma, g, h0):
    _need_cuda(q, k, v, g_gamma, g, h0)
    B, T, H, K = q.shape
    V = v.shape[-1]
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be bf16")
    if g is not None and (g.dtype != torch.float32 or tuple(g.shape) != (B, T, H, K)):
        raise ValueError("g must be fp32 [B, T, H, K]")
    if g_gamma is not None and (g_gamma.dtype != torch.float32 or g_gamma.numel() != H):
        raise ValueError("g_gamma must be fp32 [H]")
    if h0 is not None and (h0.dtype != torch.float32 or tuple(h0.shape) != (B, H, K, V)):
        raise ValueError("h0 must be fp32 [B, H, K, V]")
    return B, T, H, K, V


def chunk_gla_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  g_gamma: Optional[torch.Tensor], scale: float, chunk_size: int = 64, *,
                  g: Optional[torch.Tensor] = None, h0: Optional[torch.Tensor] = None,
                  output_final_state: bool = False, output_states: bool = False,
                  output_intermediates: bool = False, exact_intra: bool = True,
                  o: Optional[torch.Tensor] = None,
                  ht: Optional[torch.Tensor] = None,
                  h: Optional[torch.Tensor] = None) -> GLAForward:
    """Chunked GLA forward (KE/examples/kernels/chunk_gla.py:258-273), fused
    into one kernel.  Either the per-head constant gate `g_gamma` [H] (the
    reference template's mode) or the per-key log-gate `g` [B, T, H, K] (raw,
    chunk-local cumsum taken in-kernel; semantics of
    KE/upstream/fused_chunk_simple_gla/common_chunk_h.py:330-334) is used.
    output_states=True also returns the per-chunk states h (bf16), the
    residual of the backward.  output_intermediates=True also returns
    g_cumsum (fp32 [B, T, H, K]) and the unmasked intra-chunk A (fp32
    [B, T, H, 64]) as the reference's first two outputs, computed by a
    separate fp32 kernel (one more pass over q, k and g).
    exact_intra=True (the default) feeds tril(A) to the intra-chunk product
    as a bf16 hi + lo pair (A to ~2^-17 relative, the fp32 A of the
    template's output kernel, chunk_gla.py:208-212); exact_intra=False
    rounds it to bf16 once (the operand precision of the reference jnp
    oracle's einsum at TPU default precision, chunk_gla_ref.py:96-97),
    about 10 % faster.  o, ht and h may be given
    preallocated.
    """
    B, T, H, K, V = _gla_check(q, k, v, g_gamma, g, h0)
    if o is None:
        o = torch.empty((B, T, H, V), dtype=torch.bfloat16, device=q.device)
    if output_final_state and ht is None:
        ht = torch.empty((B, H, K, V), dtype=torch.float32, device=q.device)
    lib = _lib.load()
    # Few (batch, head) pairs: the library splits the sequence and needs a
    # workspace for the per-segment states (0 bytes otherwise).
    ws_bytes = lib.gl_chunk_gla_fwd_workspace_bytes(B, T, H, K, V, chunk_size)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    if output_states:
        h = _out(h, (B, T // chunk_size, H, K, V), torch.bfloat16, q.device, "h")
    flags = 0 if exact_intra else _lib.GL_GLA_BF16_INTRA
    _lib.check(lib.gl_chunk_gla_fwd_ex(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(g),
                                       _ptr(g_gamma), _ptr(h0), float(scale), B, T, H, K, V,
                                       chunk_size, o.data_ptr(), _ptr(ht),
                                       h.data_ptr() if output_states else None, _ptr(ws), ws_bytes,
                                       flags, None, _stream()),
               "gl_chunk_gla_fwd_states" if output_states else "gl_chunk_gla_fwd")
    g_cumsum = A = None
    if output_intermediates:
        g_cumsum = torch.empty((B, T, H, K), dtype=torch.float32, device=q.device)
        A = torch.empty((B, T, H, chunk_size), dtype=torch.float32, device=q.device)
        _lib.check(lib.gl_chunk_gla_fwd_intermediates(q.data_ptr(), k.data_ptr(), _ptr(g),
                                                      _ptr(g_gamma), float(scale), B, T, H, K,
                                                      chunk_size, g_cumsum.data_ptr(), A.data_ptr(),
                                                      None, _stream()),
                   "gl_chunk_gla_fwd_intermediates")
    return GLAForward(o, ht if output_final_state else None, h, g_cumsum, A)


def chunk_gla_fwd_scatter(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          g_gamma: Optional[torch.Tensor], scale: float, chunk_size: int = 64, *,
                          outs, g: Optional[torch.Tensor] = None, h0: Optional[torch.Tensor] = None,
                          ht: Optional[torch.Tensor] = None, exact_intra: bool = True) -> None:
    """chunk_gla_fwd whose output o is stored into every buffer of `outs`
    (tensors on this device, or integer device addresses of peer-mapped
    buffers such as shard.PeerBuffers.ptrs plus an offset), each holding o's
    layout [B, T, H, V] bf16.  Used to assemble a head-sharded forward on
    every rank inside the kernel; the caller synchronises the ranks after it.
    ht (fp32 [B, H, K, V]) receives the final state when given."""
    B, T, H, K, V = _gla_check(q, k, v, g_gamma, g, h0)
    ptrs = [o.data_ptr() if isinstance(o, torch.Tensor) else int(o) for o in outs]
    for o in outs:
        if isinstance(o, torch.Tensor) and (o.dtype != torch.bfloat16 or tuple(o.shape) != (B, T, H, V)
                                            or not o.is_contiguous()):
            raise ValueError("each output must be a contiguous bf16 [B, T, H, V] tensor")
    if ht is not None and (ht.dtype != torch.float32 or tuple(ht.shape) != (B, H, K, V)):
        raise ValueError("ht must be fp32 [B, H, K, V]")
    lib = _lib.load()
    ws_bytes = lib.gl_chunk_gla_fwd_workspace_bytes(B, T, H, K, V, chunk_size)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    import ctypes
    arr = (ctypes.c_void_p * len(ptrs))(*ptrs)
    flags = 0 if exact_intra else _lib.GL_GLA_BF16_INTRA
    _lib.check(lib.gl_chunk_gla_fwd_scatter(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(g),
                                            _ptr(g_gamma), _ptr(h0), float(scale), B, T, H, K, V,
                                            chunk_size, ctypes.cast(arr, ctypes.c_void_p), len(ptrs),
                                            _ptr(ht), _ptr(ws), ws_bytes, flags, None, _stream()),
               "gl_chunk_gla_fwd_scatter")


def chunk_gla_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, do: torch.Tensor,
                  h: torch.Tensor, g_gamma: Optional[torch.Tensor], scale: float,
                  chunk_size: int = 64, *, g: Optional[torch.Tensor] = None,
                  dht: Optional[torch.Tensor] = None, output_dh0: bool = False,
                  dq: Optional[torch.Tensor] = None, dk: Optional[torch.Tensor] = None,
                  dv: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None
                  ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Backward of chunk_gla_fwd: (dq, dk, dv, dh0) for the output gradient
    `do` (and the final-state gradient `dht`), from the forward's per-chunk
    states `h` (chunk_gla_fwd(..., output_states=True).h).  Replaces _bwd of
    KE/examples/kernels/chunk_gla.py:446-453 (reverse dh scan :281-305, fused
    dq/dk/dv :313-426); the gate gets no gradient, as there.  dq, dk, dv and
    the uint8 `workspace` (chunk_gla_bwd_workspace_bytes) may be given
    preallocated."""
    B, T, H, K, V = _gla_check(q, k, v, g_gamma, g, dht)
    _need_cuda(do, h)
    if do.dtype != torch.bfloat16 or tuple(do.shape) != (B, T, H, V):
        raise ValueError("do must be bf16 [B, T, H, V]")
    if h.dtype != torch.bfloat16 or tuple(h.shape) != (B, T // chunk_size, H, K, V):
        raise ValueError("h must be bf16 [B, T/chunk, H, K, V]")
    lib = _lib.load()
    dq = _out(dq, q.shape, torch.bfloat16, q.device, "dq")
    dk = _out(dk, k.shape, torch.bfloat16, q.device, "dk")
    dv = _out(dv, v.shape, torch.bfloat16, q.device, "dv")
    dh0 = torch.empty((B, H, K, V), dtype=torch.float32, device=q.device) if output_dh0 else None
    ws_bytes = lib.gl_chunk_gla_bwd_workspace_bytes(B, T, H, K, V, chunk_size)
    if ws_bytes == 0:
        raise ValueError("gl_chunk_gla_bwd: unsupported shape")
    if workspace is None:
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    elif workspace.dtype != torch.uint8 or workspace.numel() < ws_bytes or not workspace.is_cuda:
        raise ValueError(f"workspace must be a CUDA uint8 tensor of at least {ws_bytes} bytes")
    ws = workspace
    _lib.check(lib.gl_chunk_gla_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(g), _ptr(g_gamma),
                                    h.data_ptr(), do.data_ptr(), _ptr(dht), float(scale), B, T, H, K,
                                    V, chunk_size, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                    _ptr(dh0), ws.data_ptr(), ws.numel(), None, _stream()),
               "gl_chunk_gla_bwd")
    return dq, dk, dv, dh0


def chunk_gla_bwd_workspace_bytes(B: int, T: int, H: int, K: int = 128, V: int = 128,
                                  chunk_size: int = 64) -> int:
    """Device workspace chunk_gla_bwd needs for this shape on the current device."""
    return int(_lib.load().gl_chunk_gla_bwd_workspace_bytes(B, T, H, K, V, chunk_size))


class _ChunkGLA(torch.autograd.Function):
    """custom-VJP pair of the template (chunk_gla.py:434-456): the forward
    keeps q, k, v, the gate and the per-chunk states; the backward returns
    dq, dk, dv (and dh0 when h0 is given)."""

    @staticmethod
    def forward(ctx, q, k, v, g_gamma, g, h0, scale, chunk_size, exact_intra):
        res = chunk_gla_fwd(q, k, v, g_gamma, scale, chunk_size, g=g, h0=h0, output_states=True,
                            exact_intra=exact_intra)
        ctx.save_for_backward(q, k, v, g_gamma, g, res.h)
        ctx.scale, ctx.chunk_size, ctx.has_h0 = scale, chunk_size, h0 is not None
        return res.o

    @staticmethod
    def backward(ctx, do):
        q, k, v, g_gamma, g, h = ctx.saved_tensors
        dq, dk, dv, dh0 = chunk_gla_bwd(q, k, v, do.to(torch.bfloat16).contiguous(), h, g_gamma,
                                        ctx.scale, ctx.chunk_size, g=g, output_dh0=ctx.has_h0)
        return dq, dk, dv, None, None, dh0, None, None, None


def chunk_gla(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g_gamma: Optional[torch.Tensor],
              scale: float, chunk_size: int = 64, *, g: Optional[torch.Tensor] = None,
              h0: Optional[torch.Tensor] = None, exact_intra: bool = True) -> torch.Tensor:
    """`chunk_gla(q, k, v, g_gamma, scale, chunk_size)`
    (KE/examples/kernels/chunk_gla.py:434-456): returns o (bf16),
    differentiable in q, k, v (and h0) when any of them requires grad.
    exact_intra as in chunk_gla_fwd."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, h0)):
        return _ChunkGLA.apply(q, k, v, g_gamma, g, h0, scale, chunk_size, exact_intra)
    return chunk_gla_fwd(q, k, v, g_gamma, scale, chunk_size, g=g, h0=h0, exact_intra=exact_intra).o


# ---------------------------------------------------------------------------
# RMS norm with the residual's addition
# ---------------------------------------------------------------------------
_NO_GUARD = contextlib.nullcontext()


def _same_device(first: torch.Tensor, *rest: Optional[torch.Tensor]):
    """Checks that every tensor is a contiguous one on `first`'s CUDA device;
    returns a context in which that device is the current one."""
    dev = first.get_device()
    if dev < 0 or not first.is_contiguous():
        _need_cuda(first)
    for t in rest:
        if t is not None and (t.get_device() != dev or not t.is_contiguous()):
            _need_cuda(t)
            raise ValueError(f"all tensors of a call must be on one device, got {first.device} and {t.device}")
    return _NO_GUARD if dev == _current_device() else torch.cuda.device(dev)


def _new(like: torch.Tensor, t: Optional[torch.Tensor], shape, dtype: torch.dtype, name: str) -> torch.Tensor:
    """_out on `like`'s device."""
    if t is not None:
        return _out(t, shape, dtype, like.device, name)
    return torch.empty(*shape, dtype=dtype, device=like.device)


def _new_like(like: torch.Tensor, t: Optional[torch.Tensor], dtype: torch.dtype, name: str) -> torch.Tensor:
    """_out of `like`'s shape on its device."""
    if t is not None:
        return _out(t, like.shape, dtype, like.device, name)
    return torch.empty_like(like, dtype=dtype)


def _records(name: str, *ts: Optional[torch.Tensor]) -> bool:
    """Whether autograd records this call of `name`.  A tensor that carries a
    forward-mode tangent is refused: no operator here has one for its outputs."""
    if getattr(forward_ad, "_current_level", 0) >= 0:  # inside a dual_level
        for t in ts:
            if t is not None and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no forward-mode derivative")
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


class _NoGradient(torch.autograd.Function):
    """A call without a backward inside a recorded computation: its gradient is
    an error when it is asked for, not missing."""
    @staticmethod
    def forward(ctx, name, call, args, *inputs):
        ctx.name = name
        return call(*args)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no gradient: detach its inputs or call it under torch.no_grad()")


def _without_gradient(name: str, call, args, outs, *inputs: Optional[torch.Tensor]):
    """call(*args), recorded as _NoGradient of the inputs."""
    if any(o is not None for o in outs):
        raise RuntimeError(f"{name} has no gradient and takes preallocated outputs under torch.no_grad() only")
    return _NoGradient.apply(name, call, args, *inputs)


class RMSNormForward(NamedTuple):
    """Result of rms_norm_fwd.  y (bf16) and q, s (e4m3 and its 1x128 scales)
    are None unless asked for; h is the stored sum (x itself without a
    residual); rstd (fp32 [M]) is the residual of the backward."""
    y: Optional[torch.Tensor]
    h: torch.Tensor
    q: Optional[torch.Tensor]
    s: Optional[torch.Tensor]
    rstd: Optional[torch.Tensor]


def _rms_check(x, weight, residual):
    shape = x.shape
    if x.dtype != torch.bfloat16 or len(shape) != 2:
        raise ValueError("x must be a 2-D bf16 tensor")
    M, K = shape
    if weight.dtype not in (torch.bfloat16, torch.float32) or weight.shape != shape[1:]:
        raise ValueError("weight must be bf16 or fp32 [K]")
    if residual is not None and (residual.dtype != torch.bfloat16 or residual.shape != shape):
        raise ValueError("residual must be bf16 of x's shape")
    return M, K


def _rms_norm(x, weight, eps, residual, h, y, q, s, rstd):
    """The launch itself: y, q and s, rstd are written where given."""
    M, K = x.shape
    _lib.check(_lib.load().gl_rms_norm_fwd(
        x.data_ptr(), _ptr(residual), weight.data_ptr(), weight.dtype == torch.float32, eps, M, K,
        h.data_ptr() if residual is not None else None, _ptr(y), _ptr(q), _ptr(s), _ptr(rstd), None,
        _stream()), "gl_rms_norm_fwd")


def rms_norm_quant_1x128(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                         residual: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
                         s: Optional[torch.Tensor] = None, h: Optional[torch.Tensor] = None
                         ) -> Tuple[torch.Tensor, ...]:
    """RMS norm of x (+ residual) straight into the operand of gmm_fp8_fwd: x,
    residual bf16 [M, K], weight bf16 or fp32 [K] -> (e4m3 [M, K], fp32 scales
    [M, K/128]), and with a residual also h = bf16(x + residual), the stream
    that goes on.  K a multiple of 128, at most 16384.

    The layout and scales are quant_act_1x128's; the norm enters them in 32
    bits, so the pair is rounded once.  q, s and h may be given preallocated;
    h may be `x` or `residual` itself.  It has no gradient (rms_norm has):
    asking for one of its outputs is an error.
    """
    if _records("rms_norm_quant_1x128", x, weight, residual):
        return _without_gradient("rms_norm_quant_1x128", _rms_norm_quant_1x128, (x, weight, eps, residual, q, s, h),
                                 (q, s, h), x, weight, residual)
    return _rms_norm_quant_1x128(x, weight, eps, residual, q, s, h)


def _rms_norm_quant_1x128(x, weight, eps, residual, q, s, h):
    with _same_device(x, weight, residual):
        M, K = _rms_check(x, weight, residual)
        if h is not None and residual is None:
            raise ValueError("h goes with a residual")
        q = _new_like(x, q, FP8, "q")
        s = _new(x, s, (M, K // TILE), torch.float32, "s")
        if residual is not None:
            h = _new_like(x, h, torch.bfloat16, "h")
        _rms_norm(x, weight, eps, residual, h, None, q, s, None)
    return (q, s) if residual is None else (q, s, h)


def rms_norm_fwd(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                 residual: Optional[torch.Tensor] = None, output_quant: bool = False,
                 y: Optional[torch.Tensor] = None, h: Optional[torch.Tensor] = None) -> RMSNormForward:
    """Training forward of the RMS norm: h = bf16(x + residual) (x without
    one), y = h / sqrt(mean(h^2) + eps) * weight in bf16, and what rms_norm_bwd
    needs.  output_quant=True also returns y's e4m3 pair (rms_norm_quant_1x128)
    from the same pass.  K a multiple of 8 (128 with output_quant), at most
    16384; y and h may be given preallocated."""
    with _same_device(x, weight, residual):
        M, K = _rms_check(x, weight, residual)
        if h is not None and residual is None:
            raise ValueError("h goes with a residual")
        y = _new_like(x, y, torch.bfloat16, "y")
        h = _new_like(x, h, torch.bfloat16, "h") if residual is not None else x
        q = s = None
        if output_quant:
            q = torch.empty_like(x, dtype=FP8)
            s = torch.empty(M, K // TILE, dtype=torch.float32, device=x.device)
        rstd = x.new_empty(M, dtype=torch.float32)
        _rms_norm(x, weight, eps, residual, h, y, q, s, rstd)
    return RMSNormForward(y, h, q, s, rstd)


def rms_norm_bwd(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor, *,
                 dh: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dx, dweight) for the gradients dy of y and dh of h (bf16 [M, K]), from
    the forward's h and rstd.  dx is the gradient of x and of the residual;
    dweight has weight's type and is summed in fp32 in a fixed order."""
    with _same_device(h, dy, weight, rstd, dh):
        M, K = _rms_check(h, weight, dh)
        if dy.dtype != torch.bfloat16 or dy.shape != h.shape:
            raise ValueError("dy must be bf16 of h's shape")
        if rstd.dtype != torch.float32 or tuple(rstd.shape) != (M,):
            raise ValueError("rstd must be fp32 [M]")
        lib = _lib.load()
        dx = torch.empty_like(h)
        dw = torch.empty_like(weight)
        ws_bytes = lib.gl_rms_norm_bwd_workspace_bytes(M, K)
        ws = h.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
        _lib.check(lib.gl_rms_norm_bwd(dy.data_ptr(), _ptr(dh), h.data_ptr(), weight.data_ptr(),
                                       weight.dtype == torch.float32, rstd.data_ptr(), M, K,
                                       dx.data_ptr(), dw.data_ptr(), _ptr(ws), ws_bytes, None,
                                       _stream()), "gl_rms_norm_bwd")
    return dx, dw


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        f = rms_norm_fwd(x, weight, eps, residual=residual)
        ctx.save_for_backward(f.h, weight, f.rstd)
        ctx.set_materialize_grads(False)
        return f.y if residual is None else (f.y, f.h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        if dh is not None:
            dh = dh.to(torch.bfloat16).contiguous()
        if dy is None:  # only the sum was used
            return dh, None, None, dh
        dx, dw = rms_norm_bwd(dy.to(torch.bfloat16).contiguous(), h, weight, rstd, dh=dh)
        has_res = ctx.needs_input_grad[3]
        return dx, dw, None, dx if has_res else None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
             residual: Optional[torch.Tensor] = None):
    """RMS norm in bf16, differentiable in x, weight and residual: y, or with a
    residual (y, h), h = bf16(x + residual) being the stream that goes on."""
    if _records("rms_norm", x, weight, residual):
        return _RMSNorm.apply(x, weight, eps, residual)
    f = rms_norm_fwd(x, weight, eps, residual=residual)
    return f.y if residual is None else (f.y, f.h)


# ---------------------------------------------------------------------------
# Router: top-k, group sizes, rows in expert order, balance loss
# ---------------------------------------------------------------------------
class MoERouting(NamedTuple):
    """Result of moe_route.  ids (int32 [T, topk]) are the chosen experts in
    falling order of their logits, weights (fp32) their softmax, counts (int32
    [E]) the group_sizes of the grouped matmul, pos (int32 [T, topk]) the row
    of every choice in expert order; slots without an expert have ids and pos
    -1 and weight 0.  routed, mask and renormalize are kept for the backward."""
    ids: torch.Tensor
    weights: torch.Tensor
    counts: torch.Tensor
    pos: torch.Tensor
    balance_loss: torch.Tensor
    routed: torch.Tensor
    mask: Optional[torch.Tensor]
    renormalize: bool


def _route_check(logits, mask):
    if logits.dtype not in (torch.bfloat16, torch.float32) or logits.dim() != 2:
        raise ValueError("logits must be a 2-D bf16 or fp32 tensor")
    T, E = logits.shape
    if mask is not None and (mask.dtype != torch.bool or tuple(mask.shape) != (T,)):
        raise ValueError("mask must be bool [T]")
    return T, E


def moe_route_fwd(logits: torch.Tensor, topk: int, *, mask: Optional[torch.Tensor] = None,
                  renormalize: bool = True) -> MoERouting:
    """Routes every token (logits [T, E], bf16 or fp32) to its topk experts:
    softmax, the largest logits with ties to the lowest expert, their weights
    (over their sum with renormalize), the experts' counts, the rows in expert
    order, and the balance loss E * sum_e f_e P_e (f_e: share of the choices,
    P_e: mean probability), which is 1 for an even split.

    A logit of -inf takes its expert out for that token; tokens with mask
    False, or with no logit above -inf, are not routed and are in no sum.  A
    NaN is never chosen and makes its token's weights and the loss NaN.
    E <= 1024, topk <= 32."""
    with _same_device(logits, mask):
        T, E = _route_check(logits, mask)
        ids = torch.empty(T, topk, dtype=torch.int32, device=logits.device)
        pos = torch.empty_like(ids)
        weights = torch.empty_like(ids, dtype=torch.float32)
        counts = logits.new_empty(E, dtype=torch.int32)
        loss = logits.new_empty((), dtype=torch.float32)
        routed = torch.empty_like(loss)
        lib = _lib.load()
        ws_bytes = lib.gl_moe_route_workspace_bytes(T, E)
        ws = logits.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
        _lib.check(lib.gl_moe_route_fwd(logits.data_ptr(), logits.dtype == torch.float32, _ptr(mask), T, E,
                                        topk, renormalize, ids.data_ptr(), weights.data_ptr(),
                                        counts.data_ptr(), pos.data_ptr(), loss.data_ptr(),
                                        routed.data_ptr(), _ptr(ws), ws_bytes, None, _stream()),
                   "gl_moe_route_fwd")
    return MoERouting(ids, weights, counts, pos, loss, routed, mask, renormalize)


def moe_route_bwd(logits: torch.Tensor, routing: MoERouting, dweights: Optional[torch.Tensor],
                  dloss: Optional[torch.Tensor]) -> torch.Tensor:
    """dlogits (of logits' type) for the gradients of routing.weights (fp32
    [T, topk]) and of the balance loss (fp32, one element; either may be None).
    The choices and counts are constants of the differentiation."""
    r = routing
    with _same_device(logits, r.ids, r.weights, r.counts, r.routed, r.mask, dweights, dloss):
        T, E = _route_check(logits, r.mask)
        topk = r.ids.shape[1]
        if tuple(r.ids.shape) != (T, topk) or r.weights.shape != r.ids.shape or r.counts.numel() != E \
                or r.routed.numel() != 1:
            raise ValueError("routing does not belong to these logits")
        if r.ids.dtype != torch.int32 or r.counts.dtype != torch.int32 or r.weights.dtype != torch.float32 \
                or r.routed.dtype != torch.float32:
            raise ValueError("routing's tensors must have the types that belong to moe_route_fwd's")
        if dweights is not None and (dweights.dtype != torch.float32 or dweights.shape != r.ids.shape):
            raise ValueError("dweights must be fp32 [T, topk]")
        if dloss is not None and (dloss.dtype != torch.float32 or dloss.numel() != 1):
            raise ValueError("dloss must be fp32 with one element")
        dlogits = torch.empty_like(logits)
        _lib.check(_lib.load().gl_moe_route_bwd(
            logits.data_ptr(), logits.dtype == torch.float32, _ptr(r.mask), r.ids.data_ptr(),
            r.weights.data_ptr(), r.counts.data_ptr(), r.routed.data_ptr(), _ptr(dweights), _ptr(dloss),
            T, E, topk, r.renormalize, dlogits.data_ptr(), None, _stream()), "gl_moe_route_bwd")
    return dlogits


class _MoERoute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, mask, renormalize):
        r = moe_route_fwd(logits, topk, mask=mask, renormalize=renormalize)
        ctx.save_for_backward(logits, r.ids, r.weights, r.counts, r.routed, mask)
        ctx.renormalize = renormalize
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(r.ids, r.counts, r.pos, r.routed)
        return r.ids, r.weights, r.counts, r.pos, r.balance_loss, r.routed

    @staticmethod
    @once_differentiable
    def backward(ctx, _ids, dweights, _counts, _pos, dloss, _routed):
        if dweights is None and dloss is None:
            return None, None, None, None
        logits, ids, weights, counts, routed, mask = ctx.saved_tensors
        r = MoERouting(ids, weights, counts, None, None, routed, mask, ctx.renormalize)
        dweights = dweights.float().contiguous() if dweights is not None else None
        dloss = dloss.float().contiguous() if dloss is not None else None
        return moe_route_bwd(logits, r, dweights, dloss), None, None, None


def moe_route(logits: torch.Tensor, topk: int, *, mask: Optional[torch.Tensor] = None,
              renormalize: bool = True) -> MoERouting:
    """moe_route_fwd, its weights and balance loss differentiable in logits."""
    if _records("moe_route", logits):
        out = _MoERoute.apply(logits, topk, mask, renormalize)
        return MoERouting(*out, mask, renormalize)
    return moe_route_fwd(logits, topk, mask=mask, renormalize=renormalize)


# ---------------------------------------------------------------------------
# Rows into expert order and back
# ---------------------------------------------------------------------------
def _pos_check(pos, group_sizes=None):
    if pos.dtype != torch.int32 or pos.dim() != 2:
        raise ValueError("pos must be int32 [T, topk]")
    if group_sizes is not None and (group_sizes.dtype != torch.int32 or group_sizes.dim() != 1):
        raise ValueError("group_sizes must be int32 [G]")
    return pos.shape


def _dispatch(x, s, pos, group_sizes, rows, out, out_s):
    T, topk = pos.shape
    scales = 0 if s is None else s.shape[1]
    _lib.check(_lib.load().gl_moe_dispatch(x.data_ptr(), x.shape[1] * x.element_size(), _ptr(s), scales,
                                           pos.data_ptr(), group_sizes.data_ptr(), group_sizes.numel(), T,
                                           topk, rows, out.data_ptr(), _ptr(out_s), None, _stream()),
               "gl_moe_dispatch")


def moe_dispatch_fwd(x: torch.Tensor, pos: torch.Tensor, group_sizes: torch.Tensor,
                     rows: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The forward of moe_dispatch, with `out` optionally preallocated."""
    with _same_device(x, pos, group_sizes):
        T, topk = _pos_check(pos, group_sizes)
        if x.dtype not in (torch.bfloat16, torch.float32) or x.dim() != 2 or x.shape[0] != T:
            raise ValueError("x must be bf16 or fp32 [T, K]")
        rows = T * topk if rows is None else int(rows)
        out = _new(x, out, (rows, x.shape[1]), x.dtype, "out")
        _dispatch(x, None, pos, group_sizes, rows, out, None)
    return out


def moe_dispatch_quant(q: torch.Tensor, s: torch.Tensor, pos: torch.Tensor, group_sizes: torch.Tensor,
                       rows: Optional[int] = None, out: Optional[torch.Tensor] = None,
                       out_s: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """moe_dispatch of quantised rows: q e4m3 [T, K] and s fp32 [T, K/128]
    (quant_act_1x128 or rms_norm_quant_1x128 of the tokens) -> the operands of
    gmm_fp8_fwd, quantised once per token instead of once per choice.  Rows
    past sum(group_sizes) are zeros with scale 1.  It has no gradient: asking
    for one of its outputs is an error."""
    if _records("moe_dispatch_quant", q, s):
        return _without_gradient("moe_dispatch_quant", _moe_dispatch_quant,
                                 (q, s, pos, group_sizes, rows, out, out_s), (out, out_s), q, s)
    return _moe_dispatch_quant(q, s, pos, group_sizes, rows, out, out_s)


def _moe_dispatch_quant(q, s, pos, group_sizes, rows, out, out_s):
    with _same_device(q, s, pos, group_sizes):
        T, topk = _pos_check(pos, group_sizes)
        if q.dtype != FP8 or q.dim() != 2 or q.shape[0] != T:
            raise ValueError("q must be e4m3 [T, K]")
        if s.dtype != torch.float32 or tuple(s.shape) != (T, q.shape[1] // TILE) or q.shape[1] % TILE:
            raise ValueError("s must be fp32 [T, K/128], K a multiple of 128")
        rows = T * topk if rows is None else int(rows)
        out = _new(q, out, (rows, q.shape[1]), FP8, "out")
        out_s = _new(q, out_s, (rows, s.shape[1]), torch.float32, "out_s")
        _dispatch(q, s, pos, group_sizes, rows, out, out_s)
    return out, out_s


def _combine(y, pos, weights, residual, out):
    T, topk = pos.shape
    rows, K = y.shape
    _lib.check(_lib.load().gl_moe_combine(y.data_ptr(), y.dtype == torch.float32, pos.data_ptr(),
                                          _ptr(weights), _ptr(residual), T, topk, K, rows, out.data_ptr(),
                                          None, _stream()), "gl_moe_combine")


def moe_dispatch_bwd(dout: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """Gradient bf16 [T, K] of moe_dispatch's x for dout [rows, K] (bf16 or
    fp32): the sum of a token's rows, in fp32."""
    with _same_device(dout, pos):
        T, _ = _pos_check(pos)
        if dout.dtype not in (torch.bfloat16, torch.float32) or dout.dim() != 2:
            raise ValueError("dout must be bf16 or fp32 [rows, K]")
        dx = torch.empty(T, dout.shape[1], dtype=torch.bfloat16, device=dout.device)
        _combine(dout, pos, None, None, dx)
    return dx


class _MoEDispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, group_sizes, rows):
        ctx.save_for_backward(pos)
        return moe_dispatch_fwd(x, pos, group_sizes, rows)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        return moe_dispatch_bwd(dout.to(torch.bfloat16).contiguous(), ctx.saved_tensors[0]), None, None, None


def moe_dispatch(x: torch.Tensor, pos: torch.Tensor, group_sizes: torch.Tensor,
                 rows: Optional[int] = None) -> torch.Tensor:
    """Rows of the tokens in expert order: out[pos[t, j]] = x[t] (bf16 [T, K])
    for the pos and counts of moe_route (rows 0 to sum(group_sizes) - 1, each of
    one choice; a negative one is skipped); the lhs of gmm_fp8_blockwise with group_sizes =
    counts.  `rows` (default T * topk) is the number of output rows; those past
    sum(group_sizes) are zero.  Differentiable in x (bf16)."""
    if _records("moe_dispatch", x):
        if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] > 16384:
            raise ValueError("the differentiable moe_dispatch takes bf16 [T, K], K at most 16384")
        return _MoEDispatch.apply(x, pos, group_sizes, rows)
    return moe_dispatch_fwd(x, pos, group_sizes, rows)


def _combine_check(y, pos, weights):
    T, topk = _pos_check(pos)
    if y.dtype not in (torch.bfloat16, torch.float32) or y.dim() != 2:
        raise ValueError("y must be bf16 or fp32 [rows, K]")
    if weights.dtype != torch.float32 or weights.shape != pos.shape:
        raise ValueError("weights must be fp32 [T, topk]")
    return T, topk


def moe_combine_fwd(y: torch.Tensor, pos: torch.Tensor, weights: torch.Tensor, *,
                    residual: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The forward of moe_combine, with `out` optionally preallocated (it may
    be `residual` itself)."""
    with _same_device(y, pos, weights, residual):
        T, _ = _combine_check(y, pos, weights)
        if residual is not None and (residual.dtype != torch.bfloat16
                                     or tuple(residual.shape) != (T, y.shape[1])):
            raise ValueError("residual must be bf16 [T, K]")
        out = _new(y, out, (T, y.shape[1]), torch.bfloat16, "out")
        _combine(y, pos, weights, residual, out)
    return out


def moe_combine_bwd(dout: torch.Tensor, y: torch.Tensor, pos: torch.Tensor, weights: torch.Tensor,
                    group_sizes: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dy, dweights) of moe_combine for dout (bf16 [T, K]): dy has y's type,
    its rows past sum(group_sizes) are zero; the residual's gradient is dout."""
    with _same_device(y, dout, pos, weights, group_sizes):
        T, topk = _combine_check(y, pos, weights)
        _pos_check(pos, group_sizes)
        rows, K = y.shape
        if dout.dtype != torch.bfloat16 or tuple(dout.shape) != (T, K):
            raise ValueError("dout must be bf16 [T, K]")
        dy = torch.empty_like(y)
        dw = torch.empty_like(weights)
        _lib.check(_lib.load().gl_moe_combine_bwd(
            dout.data_ptr(), y.data_ptr(), y.dtype == torch.float32, pos.data_ptr(), weights.data_ptr(),
            group_sizes.data_ptr(), group_sizes.numel(), T, topk, K, rows, dy.data_ptr(), dw.data_ptr(),
            None, _stream()), "gl_moe_combine_bwd")
    return dy, dw


class _MoECombine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, pos, weights, group_sizes, residual):
        ctx.save_for_backward(y, pos, weights, group_sizes)
        return moe_combine_fwd(y, pos, weights, residual=residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        y, pos, weights, group_sizes = ctx.saved_tensors
        dout = dout.to(torch.bfloat16).contiguous()
        dy = dw = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[2]:
            dy, dw = moe_combine_bwd(dout, y, pos, weights, group_sizes)
        return dy, None, dw, None, dout if ctx.needs_input_grad[4] else None


def moe_combine(y: torch.Tensor, pos: torch.Tensor, weights: torch.Tensor, group_sizes: torch.Tensor, *,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The experts' rows back to their tokens: out[t] = residual[t] + sum_j
    weights[t, j] * y[pos[t, j]] (y bf16 or fp32 [rows, K], out bf16), summed in
    fp32 and rounded once; for pos, weights and counts (group_sizes) of
    moe_route.  Differentiable in y, weights and residual."""
    if _records("moe_combine", y, weights, residual):
        # what the backward alone reads
        _same_device(y, group_sizes)
        _pos_check(pos, group_sizes)
        if not 1 <= group_sizes.numel() <= 1024:
            raise ValueError("the differentiable moe_combine takes group_sizes of 1 to 1024 groups")
        return _MoECombine.apply(y, pos, weights, group_sizes, residual)
    return moe_combine_fwd(y, pos, weights, residual=residual)


# ---------------------------------------------------------------------------
# Grouped products with 4-bit weights, for few rows
# ---------------------------------------------------------------------------
def quant_w4_128x1(w: torch.Tensor, w4: Optional[torch.Tensor] = None,
                   s: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 [G, K, N] -> (int32 [G, K/8, N], fp32 scales [G, K/128, N]): 4-bit
    weights, eight along K in a word (nibble j of word [g, i, n] is q[g, 8i + j,
    n] + 8, q in -7..7), one absmax scale per 128 weights of a column.  K a
    multiple of 128, N of 32; `w4` / `s` may be given as preallocated outputs."""
    with _same_device(w):
        if w.dtype != torch.bfloat16 or w.dim() != 3:
            raise ValueError("quant_w4_128x1 expects a 3-D bf16 tensor")
        G, K, N = w.shape
        w4 = _new(w, w4, (G, K // 8, N), torch.int32, "w4")
        s = _new(w, s, (G, K // TILE, N), torch.float32, "s")
        _lib.check(_lib.load().gl_quant_w4_128x1(w.data_ptr(), G, K, N, w4.data_ptr(), s.data_ptr(), None,
                                                 _stream()), "gl_quant_w4_128x1")
    return w4, s


def gmm_w4_fwd(x: torch.Tensor, w4: torch.Tensor, s: torch.Tensor, group_sizes: torch.Tensor,
               out_dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped matmul of few rows with 4-bit weights: x bf16 [M, K] (rows in
    group order), w4 and s as quant_w4_128x1 gives them, group_sizes int32 [G]
    -> [M, N].  The decoding counterpart of gmm_fp8_fwd: reads half a byte a
    weight of the groups that have rows, and x in bf16.  It has no gradient:
    asking for one of its output is an error.  Rows at or beyond sum(group_sizes) are left as they are in
    `out` (zeroed when allocated)."""
    if _records("gmm_w4_fwd", x, s):
        return _without_gradient("gmm_w4_fwd", _gmm_w4, (x, w4, s, group_sizes, out_dtype, out), (out,), x, s)
    return _gmm_w4(x, w4, s, group_sizes, out_dtype, out)


def _gmm_w4(x, w4, s, group_sizes, out_dtype, out):
    with _same_device(x, w4, s, group_sizes, out):
        if x.dtype != torch.bfloat16 or x.dim() != 2:
            raise ValueError("x must be a 2-D bf16 tensor")
        M, K = x.shape
        if w4.dtype != torch.int32 or w4.dim() != 3 or w4.shape[1] * 8 != K:
            raise ValueError("w4 must be int32 [G, K/8, N]")
        G, _, N = w4.shape
        if s.dtype != torch.float32 or tuple(s.shape) != (G, K // TILE, N):
            raise ValueError("s must be fp32 [G, K/128, N]")
        if group_sizes.dtype != torch.int32 or group_sizes.numel() != G:
            raise ValueError("group_sizes must be int32 [G]")
        if out is None and out_dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("out_dtype must be bf16 or fp32")
        if out is not None and (out.dtype not in (torch.bfloat16, torch.float32)
                                or tuple(out.shape) != (M, N)):
            raise ValueError("out must be a contiguous bf16 or fp32 [M, N] tensor")
        flags = _lib.GL_W4_ZERO_TAIL if out is None else 0
        if out is None:
            out = torch.empty(M, N, dtype=out_dtype, device=x.device)
        code = _lib.GL_OUT_F32 if out.dtype == torch.float32 else _lib.GL_OUT_BF16
        lib = _lib.load()
        ws_bytes = lib.gl_gmm_w4_workspace_bytes(M, K)
        ws = x.new_empty(ws_bytes, dtype=torch.uint8)
        _lib.check(lib.gl_gmm_w4_fwd(x.data_ptr(), w4.data_ptr(), s.data_ptr(), group_sizes.data_ptr(), G,
                                     M, K, N, out.data_ptr(), code, flags, ws.data_ptr(), ws_bytes, None,
                                     _stream()), "gl_gmm_w4_fwd")
    return out


def device_status() -> int:
    """Synchronises the current stream and returns (and clears) the library's
    device error word: 0 when no kernel reported a problem."""
    return _lib.device_status(_stream())
