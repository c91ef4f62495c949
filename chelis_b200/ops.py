"""Host-side calls of the CUDA backend on torch-owned device memory.

torch provides device memory and streams only; every computation is one of
libchelis_cuda.so's kernels, reached through the C ABI (chelis_b200.lib).
Each wrapper enqueues on torch's current CUDA stream and returns torch
tensors.  Names and argument meanings follow the reference's operations
(matmul, layer_norm, softmax, dropout, sum, max_reduce, count, cumsum).
"""
from __future__ import annotations

import array
import contextlib
import ctypes
import operator
import struct
from typing import NamedTuple

import torch

from . import lib as L

_initialised: set[int] = set()


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# the handle of a device's current stream; torch.cuda.current_stream makes a
# Stream object around it, a microsecond more at every call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _prepare(*tensors: torch.Tensor) -> None:
    last = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("chelis_b200 ops take CUDA tensors (device memory)")
        if not t.is_contiguous():
            raise ValueError("chelis_b200 ops take contiguous tensors")
        last = t
    dev = torch.cuda.current_device() if last is None else last.device.index
    if dev not in _initialised:
        L.call("chelis_cuda_init", dev)
        _initialised.add(dev)
    L.load().chelis_cuda_set_stream(_raw_stream(dev))


@contextlib.contextmanager
def gemm_mode(mode: int):
    lib = L.load()
    old = lib.chelis_cuda_get_gemm_mode()
    L.call("chelis_cuda_set_gemm_mode", mode)
    try:
        yield
    finally:
        L.call("chelis_cuda_set_gemm_mode", old)


@contextlib.contextmanager
def dgemm_kernel(kernel: int):
    """f64 GEMM kernel (L.DGEMM_AUTO / _DMMA / _FFMA) for this thread only."""
    L.call("chelis_cuda_set_thread_modes", -1, -1, kernel)
    try:
        yield
    finally:
        L.call("chelis_cuda_set_thread_modes", -1, -1, -1)


@contextlib.contextmanager
def gemm_pairs(enable: bool):
    """3xTF32 main kernel on CTA pairs (256 x 256 tiles, the default) or on
    single CTAs (128 x 256 tiles)."""
    lib = L.load()
    old = lib.chelis_cuda_get_gemm_pairs()
    L.call("chelis_cuda_set_gemm_pairs", int(enable))
    try:
        yield
    finally:
        L.call("chelis_cuda_set_gemm_pairs", old)


@contextlib.contextmanager
def fused_jit(enable: bool):
    """FusedElem elementwise groups through per-chain compiled kernels (the
    default) or the ahead-of-time interpreter; the same bits either way."""
    lib = L.load()
    old = lib.chelis_cuda_get_fused_jit()
    L.call("chelis_cuda_set_fused_jit", int(enable))
    try:
        yield
    finally:
        L.call("chelis_cuda_set_fused_jit", old)


@contextlib.contextmanager
def rows_mode(mode: int):
    lib = L.load()
    old = lib.chelis_cuda_get_rows_mode()
    L.call("chelis_cuda_set_rows_mode", mode)
    try:
        yield
    finally:
        L.call("chelis_cuda_set_rows_mode", old)


def device_status() -> None:
    """Raise if a bounded device wait gave up since the last check."""
    L.call("chelis_cuda_device_status")


def launch_count() -> int:
    return int(L.load().chelis_cuda_launch_count())


# ---------------------------------------------------------------- matmul

def matmul(a: torch.Tensor, b: torch.Tensor, trans_a: bool = False, trans_b: bool = False,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """op(A).op(B) for f32 (3xTF32 tensor cores, or the exact tree mode) or f64
    (DMMA); rank-3 operands are a strided batch."""
    if a.dtype != b.dtype or a.dtype not in (torch.float32, torch.float64):
        raise ValueError("matmul takes two f32 or two f64 tensors")
    batched = a.dim() == 3
    if batched != (b.dim() == 3) or a.dim() not in (2, 3):
        raise ValueError("matmul takes rank-2 or rank-3 operands of equal rank")
    _prepare(a, b, out)
    ar, ac = a.shape[-2:]
    br, bc = b.shape[-2:]
    m, k = (ac, ar) if trans_a else (ar, ac)
    k2, n = (bc, br) if trans_b else (br, bc)
    if k != k2:
        raise ValueError(f"contraction extents differ: {k} vs {k2}")
    batch = a.shape[0] if batched else 1
    shape = (batch, m, n) if batched else (m, n)
    if out is None:
        out = torch.empty(shape, dtype=a.dtype, device=a.device)
    name = "chelis_cuda_sgemm" if a.dtype == torch.float32 else "chelis_cuda_dgemm"
    L.call(name, int(trans_a), int(trans_b), m, n, k, a.data_ptr(), ac, ar * ac,
           b.data_ptr(), bc, br * bc, out.data_ptr(), n, m * n, batch)
    return out


def matmul_host(a: torch.Tensor, b: torch.Tensor, trans_a: bool = False, trans_b: bool = False,
                out: torch.Tensor | None = None, device: int | None = None) -> torch.Tensor:
    """op(A).op(B) for host (CPU) tensors through chelis_cuda_[sd]gemm_host:
    uploads, GEMM panels and read-back overlap on the GPU's copy engines.
    Returns once the result is in `out` (pinned output memory is allocated
    when `out` is None and `a` is pinned)."""
    if a.device.type != "cpu" or b.device.type != "cpu":
        raise ValueError("matmul_host takes host tensors")
    if a.dtype != b.dtype or a.dtype not in (torch.float32, torch.float64):
        raise ValueError("matmul_host takes two f32 or two f64 tensors")
    if not (a.is_contiguous() and b.is_contiguous()):
        raise ValueError("matmul_host takes contiguous tensors")
    batched = a.dim() == 3
    if batched != (b.dim() == 3) or a.dim() not in (2, 3):
        raise ValueError("matmul_host takes rank-2 or rank-3 operands of equal rank")
    dev = torch.device("cuda", torch.cuda.current_device() if device is None else device)
    with torch.cuda.device(dev):
        _prepare()
        ar, ac = a.shape[-2:]
        br, bc = b.shape[-2:]
        m, k = (ac, ar) if trans_a else (ar, ac)
        k2, n = (bc, br) if trans_b else (br, bc)
        if k != k2:
            raise ValueError(f"contraction extents differ: {k} vs {k2}")
        batch = a.shape[0] if batched else 1
        shape = (batch, m, n) if batched else (m, n)
        if out is None:
            out = torch.empty(shape, dtype=a.dtype, pin_memory=a.is_pinned())
        elif out.device.type != "cpu" or not out.is_contiguous() or tuple(out.shape) != shape:
            raise ValueError("out must be a contiguous host tensor of the product's shape")
        name = "chelis_cuda_sgemm_host" if a.dtype == torch.float32 else "chelis_cuda_dgemm_host"
        L.call(name, int(trans_a), int(trans_b), m, n, k, a.data_ptr(), ac, ar * ac,
               b.data_ptr(), bc, br * bc, out.data_ptr(), n, m * n, batch)
        torch.cuda.current_stream(dev).synchronize()
    return out


def attention_causal(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                     with_lse: bool = False):
    """softmax(where(causal, (q.k^T)*scale, -inf)).v for f32 [..., seq, dh]
    heads (flattened to [bh, seq, dh]); head dims 32 and 64."""
    if not (q.dtype == k.dtype == v.dtype == torch.float32) or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("attention_causal takes three f32 tensors of one shape")
    _prepare(q, k, v)
    seq, dh = q.shape[-2:]
    bh = q.numel() // (seq * dh) if q.numel() else 0
    o = torch.empty_like(q)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if with_lse else None
    L.call("chelis_cuda_attention_causal_fwd", bh, seq, dh, float(scale), q.data_ptr(),
           k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr() if with_lse else None)
    return (o, lse) if with_lse else o


def attention_causal_bwd(q, k, v, o, lse, dout, scale: float):
    """(dq, dk, dv) of attention_causal given its output o and lse."""
    _prepare(q, k, v, o, lse, dout)
    seq, dh = q.shape[-2:]
    bh = q.numel() // (seq * dh) if q.numel() else 0
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    L.call("chelis_cuda_attention_causal_bwd", bh, seq, dh, float(scale), q.data_ptr(),
           k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), dout.data_ptr(),
           dq.data_ptr(), dk.data_ptr(), dv.data_ptr())
    return dq, dk, dv


# ---------------------------------------------------------------- rows

def row_sum(x: torch.Tensor) -> torch.Tensor:
    _prepare(x)
    out = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    L.call("chelis_cuda_row_sum_f32", x.data_ptr(), x.shape[0], x.shape[1], out.data_ptr())
    return out


def col_sum(x: torch.Tensor) -> torch.Tensor:
    _prepare(x)
    out = torch.empty(x.shape[1], dtype=torch.float32, device=x.device)
    L.call("chelis_cuda_col_sum_f32", x.data_ptr(), x.shape[0], x.shape[1], out.data_ptr())
    return out


def row_max(x: torch.Tensor) -> torch.Tensor:
    _prepare(x)
    out = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    L.call("chelis_cuda_row_max_f32", x.data_ptr(), x.shape[0], x.shape[1], out.data_ptr())
    return out


def count(x: torch.Tensor) -> int:
    _prepare(x)
    out = torch.empty(1, dtype=torch.int64, device=x.device)
    L.call("chelis_cuda_count_bool", x.data_ptr(), x.numel(), out.data_ptr())
    return int(out.item())


def dropout(x: torch.Tensor, key: int, rate: float, index_base: int = 0) -> torch.Tensor:
    _prepare(x)
    y = torch.empty_like(x)
    L.call("chelis_cuda_dropout_f32", x.data_ptr(), y.data_ptr(), x.numel(), key, rate, index_base)
    return y


def dropout_mask(n: int, key: int, rate: float, index_base: int = 0,
                 device: torch.device | None = None) -> torch.Tensor:
    keep = torch.empty(n, dtype=torch.uint8, device=device or "cuda")
    _prepare(keep)
    L.call("chelis_cuda_dropout_mask", keep.data_ptr(), n, key, rate, index_base)
    return keep


def layer_norm(x, gamma, beta, eps: float) -> torch.Tensor:
    _prepare(x, gamma, beta)
    y = torch.empty_like(x)
    L.call("chelis_cuda_layer_norm_f32", x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), eps,
           y.data_ptr(), x.shape[0], x.shape[1])
    return y


def softmax_rows(x) -> torch.Tensor:
    _prepare(x)
    y = torch.empty_like(x)
    L.call("chelis_cuda_softmax_rows_f32", x.data_ptr(), y.data_ptr(), x.shape[0], x.shape[1])
    return y


def softmax_rows_bwd(y, g) -> torch.Tensor:
    _prepare(y, g)
    dx = torch.empty_like(y)
    L.call("chelis_cuda_softmax_rows_bwd_f32", y.data_ptr(), g.data_ptr(), dx.data_ptr(),
           y.shape[0], y.shape[1])
    return dx


def chain_fwd(x, gamma, beta, eps: float, key: int, rate: float, index_base: int = 0,
              want_stats: bool = False):
    _prepare(x, gamma, beta)
    rows, hidden = x.shape
    rowsum = torch.empty(rows, dtype=torch.float32, device=x.device)
    stats = torch.empty((rows, 4), dtype=torch.float32, device=x.device) if want_stats else None
    L.call("chelis_cuda_chain_fwd", x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), eps, key,
           rate, rows, hidden, index_base, rowsum.data_ptr(), _ptr(stats))
    return (rowsum, stats) if want_stats else rowsum


def chain_bwd(x, gamma, beta, eps: float, key: int, rate: float, index_base: int = 0,
              stats: torch.Tensor | None = None):
    _prepare(x, gamma, beta, stats)
    rows, hidden = x.shape
    dx = torch.empty_like(x)
    dg = torch.empty(hidden, dtype=torch.float32, device=x.device)
    db = torch.empty(hidden, dtype=torch.float32, device=x.device)
    L.call("chelis_cuda_chain_bwd", x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), eps, key,
           rate, rows, hidden, index_base, _ptr(stats), dx.data_ptr(), dg.data_ptr(),
           db.data_ptr())
    return dx, dg, db


def chain_fwd_save(x, gamma, beta, eps: float, key: int, rate: float, index_base: int = 0):
    """Forward that also returns the saved state (statistics + keep bits)."""
    _prepare(x, gamma, beta)
    rows, hidden = x.shape
    nbytes = int(L.load().chelis_cuda_chain_saved_bytes(rows, hidden))
    if nbytes < 0:
        raise ValueError("unsupported chain shape")
    saved = torch.empty(max(nbytes, 16) // 4, dtype=torch.float32, device=x.device)
    rowsum = torch.empty(rows, dtype=torch.float32, device=x.device)
    L.call("chelis_cuda_chain_fwd_save", x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), eps, key,
           rate, rows, hidden, index_base, rowsum.data_ptr(), saved.data_ptr())
    return rowsum, saved


def chain_bwd_saved(x, gamma, beta, eps: float, rate: float, saved: torch.Tensor):
    _prepare(x, gamma, beta, saved)
    rows, hidden = x.shape
    dx = torch.empty_like(x)
    dg = torch.empty(hidden, dtype=torch.float32, device=x.device)
    db = torch.empty(hidden, dtype=torch.float32, device=x.device)
    L.call("chelis_cuda_chain_bwd_saved", x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), eps,
           rate, rows, hidden, saved.data_ptr(), dx.data_ptr(), dg.data_ptr(), db.data_ptr())
    return dx, dg, db


def cumsum(x: torch.Tensor, reverse: bool = False) -> torch.Tensor:
    _prepare(x)
    y = torch.empty_like(x)
    name = "chelis_cuda_cumsum_f64" if x.dtype == torch.float64 else "chelis_cuda_cumsum_f32"
    L.call(name, x.data_ptr(), y.data_ptr(), x.shape[0], x.shape[1], int(reverse))
    return y


# ---------------------------------------------------------------- programs

def portfolio(r: torch.Tensor, w: torch.Tensor):
    _prepare(r, w)
    count_, t, a = r.shape
    sigma = torch.empty((count_, a, a), dtype=torch.float64, device=r.device)
    risk = torch.empty(count_, dtype=torch.float64, device=r.device)
    cum = torch.empty((count_, t), dtype=torch.float64, device=r.device)
    L.call("chelis_cuda_portfolio_f64", r.data_ptr(), w.data_ptr(), count_, t, a,
           sigma.data_ptr(), risk.data_ptr(), cum.data_ptr())
    return sigma, risk, cum


BLOCK_WEIGHTS = ("w_qkv", "w_o", "w_1", "w_2", "ln1_gamma", "ln1_beta", "ln2_gamma", "ln2_beta")


def block_step(x, weights: dict, heads: int, eps: float = 1e-5, dy=None, workspace=None,
               out: dict | None = None, reduce_grads: bool = False):
    """Transformer block forward (+ vector-Jacobian product when dy is given).
    Returns a dict with y and, with dy, dx and d<weight> for every weight.
    reduce_grads: one rank of a data-parallel step (chelis_cuda_block_step_dp):
    every weight gradient is summed across the ranks of the library's
    communicator while the reverse pass runs."""
    import ctypes
    _prepare(x, dy, *[weights[k] for k in BLOCK_WEIGHTS])
    batch, seq, d = x.shape
    dff = weights["w_1"].shape[1]
    o = out if out is not None else {}
    if "y" not in o:
        o["y"] = torch.empty_like(x)
    if dy is not None:
        if "dx" not in o:
            o["dx"] = torch.empty_like(x)
        for k in BLOCK_WEIGHTS:
            if "d" + k not in o:
                o["d" + k] = torch.empty_like(weights[k])
    p = L.BlockParams()
    p.batch, p.seq, p.d_model, p.heads, p.d_ff, p.eps = batch, seq, d, heads, dff, eps
    p.x = x.data_ptr()
    p.dy = dy.data_ptr() if dy is not None else None
    for k in BLOCK_WEIGHTS:
        setattr(p, k, weights[k].data_ptr())
    p.y = o["y"].data_ptr()
    if dy is not None:
        p.dx = o["dx"].data_ptr()
        for k in BLOCK_WEIGHTS:
            setattr(p, "d" + k if k.startswith("w") else "d" + k, o["d" + k].data_ptr())
    L.call("chelis_cuda_block_step_dp" if reduce_grads else "chelis_cuda_block_step",
           ctypes.byref(p), None if workspace is None else workspace.data_ptr())
    return o


def block_workspace(x, weights: dict, heads: int) -> torch.Tensor:
    import ctypes
    batch, seq, d = x.shape
    p = L.BlockParams()
    p.batch, p.seq, p.d_model, p.heads, p.d_ff = batch, seq, d, heads, weights["w_1"].shape[1]
    nbytes = int(L.load().chelis_cuda_block_workspace_bytes(ctypes.byref(p)))
    if nbytes < 0:
        raise ValueError("transformer block shape not admitted")
    return torch.empty(nbytes // 4 + 64, dtype=torch.float32, device=x.device)


def mlp_step(x, labels, w1, b1, w2, b2):
    _prepare(x, labels, w1, b1, w2, b2)
    batch, din = x.shape
    dh = w1.shape[1]
    dout = w2.shape[1]
    dev = x.device
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    dw1 = torch.empty_like(w1)
    db1 = torch.empty_like(b1)
    dw2 = torch.empty_like(w2)
    db2 = torch.empty_like(b2)
    L.call("chelis_cuda_mlp_step", x.data_ptr(), labels.data_ptr(), w1.data_ptr(),
           b1.data_ptr(), w2.data_ptr(), b2.data_ptr(), batch, din, dh, dout, loss.data_ptr(),
           dw1.data_ptr(), db1.data_ptr(), dw2.data_ptr(), db2.data_ptr())
    return loss, dw1, db1, dw2, db2


def _fused_args(steps, inputs, shape):
    from . import fused as F
    if not steps:
        raise ValueError("a fused group has at least one step")
    dtypes = {t.dtype for t in inputs}
    if len(dtypes) > 1:
        raise ValueError("fused group inputs share one dtype")
    dtype = dtypes.pop() if dtypes else torch.float32
    if dtype not in (torch.float32, torch.float64):
        raise ValueError("fused groups compute in f32 or f64")
    for t in inputs:
        if not t.is_cuda:
            raise ValueError("chelis_b200 ops take CUDA tensors (device memory)")
    shape = tuple(torch.broadcast_shapes(*(t.shape for t in inputs))) if shape is None else tuple(shape)
    rank = len(shape)
    strides = []
    for t in inputs:
        strides.extend(t.expand(shape).stride() if rank else ())
    c_i64 = ctypes.c_int64
    arrays = dict(
        steps=F.encode(steps),
        ptrs=(ctypes.c_void_p * max(len(inputs), 1))(*[t.data_ptr() for t in inputs]),
        strides=(c_i64 * max(len(strides), 1))(*strides),
        shape=(c_i64 * max(rank, 1))(*shape),
    )
    dt = L.DTYPE_F32 if dtype == torch.float32 else L.DTYPE_F64
    return dt, dtype, shape, arrays


def fused_elementwise(steps, inputs, shape=None) -> torch.Tensor:
    """Evaluate a FusedElem chain (a list of chelis_b200.fused.FusedStep)
    over `inputs` broadcast to `shape` (default: their broadcast shape)."""
    dt, dtype, shape, a = _fused_args(steps, inputs, shape)
    device = inputs[0].device if inputs else torch.device("cuda", torch.cuda.current_device())
    out = torch.empty(shape, dtype=dtype, device=device)
    _prepare(out)
    L.call("chelis_cuda_fused_elementwise", dt, a["steps"], len(steps), a["ptrs"], a["strides"],
           len(inputs), a["shape"], len(shape), out.data_ptr())
    return out


def fused_reduce(steps, inputs, axis: int, kind: str = "sum", shape=None) -> torch.Tensor:
    """The chain reduced along `axis` ("sum" or "max", emit_fused_reduce):
    the result has the iteration shape without `axis`."""
    from . import fused as F
    dt, dtype, shape, a = _fused_args(steps, inputs, shape)
    if not shape:
        raise ValueError("fused_reduce needs rank >= 1")
    axis = axis % len(shape)
    device = inputs[0].device if inputs else torch.device("cuda", torch.cuda.current_device())
    out = torch.empty(shape[:axis] + shape[axis + 1:], dtype=dtype, device=device)
    _prepare(out)
    L.call("chelis_cuda_fused_reduce", dt, a["steps"], len(steps), a["ptrs"], a["strides"],
           len(inputs), a["shape"], len(shape), axis, F.REDUCE_KIND[kind], out.data_ptr())
    return out


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return L.DTYPE_F32
    if t.dtype == torch.float64:
        return L.DTYPE_F64
    raise ValueError("f32 or f64 tensors")


def relu(x: torch.Tensor) -> torch.Tensor:
    _prepare(x)
    y = torch.empty_like(x)
    L.call("chelis_cuda_relu", _dt(x), x.data_ptr(), y.data_ptr(), x.numel())
    return y


def relu_adjoint(x: torch.Tensor, g: torch.Tensor) -> torch.Tensor:
    _prepare(x, g)
    dx = torch.empty_like(g)
    L.call("chelis_cuda_relu_adjoint", _dt(x), x.data_ptr(), g.data_ptr(), dx.data_ptr(), x.numel())
    return dx


def gelu(x: torch.Tensor) -> torch.Tensor:
    _prepare(x)
    y = torch.empty_like(x)
    L.call("chelis_cuda_gelu_f32", x.data_ptr(), y.data_ptr(), x.numel())
    return y


def gelu_adjoint(x: torch.Tensor, g: torch.Tensor) -> torch.Tensor:
    _prepare(x, g)
    dx = torch.empty_like(g)
    L.call("chelis_cuda_gelu_adjoint_f32", x.data_ptr(), g.data_ptr(), dx.data_ptr(), x.numel())
    return dx


def layer_norm_bwd(x, gamma, eps: float, dy):
    _prepare(x, gamma, dy)
    rows, hidden = x.shape
    dx = torch.empty_like(x)
    dg = torch.empty(hidden, dtype=torch.float32, device=x.device)
    db = torch.empty(hidden, dtype=torch.float32, device=x.device)
    L.call("chelis_cuda_layer_norm_bwd_f32", x.data_ptr(), gamma.data_ptr(), eps, dy.data_ptr(),
           rows, hidden, dx.data_ptr(), dg.data_ptr(), db.data_ptr())
    return dx, dg, db


def cross_entropy(logits, labels, want_grad: bool = True):
    """Mean cross-entropy of row softmax at int64 labels; returns (loss, dlogits)."""
    _prepare(logits, labels)
    rows, classes = logits.shape
    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    dz = torch.empty_like(logits) if want_grad else None
    L.call("chelis_cuda_cross_entropy_f32", logits.data_ptr(), labels.data_ptr(), rows, classes,
           loss.data_ptr(), _ptr(dz))
    return loss, dz


# ---------------------------------------------------------------- routed feed-forward

_ACT = {torch.float32: L.DTYPE_F32, torch.bfloat16: L.DTYPE_BF16, torch.float16: L.DTYPE_F16}
_FLOAT8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_FORMAT = {torch.float8_e4m3fn: L.FORMAT_E4M3, torch.float8_e5m2: L.FORMAT_E5M2}


class ExpertOrder(NamedTuple):
    """The (token, slot) pairs sorted by expert (expert_sort), all int32."""
    offsets: torch.Tensor   # [experts + 1]: expert e's rows are offsets[e] .. offsets[e + 1]
    position: torch.Tensor  # [tokens, k]: each pair's row, -1 for a pair with none
    source: torch.Tensor    # [tokens * k]: each row's pair, -1 for a row that no pair takes


class Blocks8(NamedTuple):
    """A matrix in 8-bit floating point with a scale for each block of 128.
    Its numbers are data times the scale of their block."""
    data: torch.Tensor    # float8_e4m3fn or float8_e5m2, [..., rows, cols rounded up to 16]
    scales: torch.Tensor  # f32; rows: [ceil(cols / 128), rows]; tiles: [..., ceil(rows / 128), ceil(cols / 128)]
    cols: int             # numbers in a row; the bytes past them are zero
    blocks: str           # "rows" (1 x 128) or "tiles" (128 x 128)


def _act(name: str, t: torch.Tensor) -> int:
    if t.dtype not in _ACT:
        raise ValueError(f"{name} takes f32, bf16 or f16 tensors")
    return _ACT[t.dtype]


def _check_i32(name: str, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype != torch.int32:
            raise ValueError(f"{name} takes int32 indices")


def _check_order(name: str, order: ExpertOrder) -> None:
    offsets, position, source = order
    _check_i32(name, offsets, position, source)
    if not (position.dim() == 2 and offsets.dim() == 1 and offsets.numel() >= 2
            and source.dim() == 1 and source.numel() == position.numel()):
        raise ValueError(f"{name} takes expert_sort's order")


def _routed(order: ExpertOrder) -> int:
    """The device address of the number of rows that a pair takes."""
    return order.offsets.data_ptr() + 4 * (order.offsets.numel() - 1)


def expert_route(logits: torch.Tensor, k: int, renormalize: bool = True):
    """The router: (weights f32 [tokens, k], experts int32 [tokens, k]), the k
    largest of the softmax of logits [tokens, experts], with renormalize over
    the chosen alone.  Ties go to the lowest index; an expert at -inf is never
    chosen (id -1, weight 0 where fewer than k are left)."""
    dt = _act("expert_route", logits)
    if logits.dim() != 2:
        raise ValueError("expert_route takes logits [tokens, experts]")
    _prepare(logits)
    tokens, experts = logits.shape
    slots, dev = max(k, 0), logits.device
    weights = torch.empty(tokens, slots, dtype=torch.float32, device=dev)
    ids = torch.empty(tokens, slots, dtype=torch.int32, device=dev)
    L.call("chelis_cuda_expert_route", dt, logits.data_ptr(), tokens, experts, k, int(renormalize),
           weights.data_ptr(), ids.data_ptr())
    return weights, ids


def expert_route_bwd(logits: torch.Tensor, experts: torch.Tensor, dweights: torch.Tensor,
                     renormalize: bool = True) -> torch.Tensor:
    """dlogits of expert_route, given the experts that it chose."""
    dt = _act("expert_route_bwd", logits)
    _check_i32("expert_route_bwd", experts)
    if not (logits.dim() == 2 and experts.dim() == 2 and experts.shape == dweights.shape
            and experts.shape[0] == logits.shape[0] and dweights.dtype == torch.float32):
        raise ValueError("expert_route_bwd takes logits [tokens, experts] and experts, f32 dweights [tokens, k]")
    _prepare(logits, experts, dweights)
    dlogits = torch.empty_like(logits)
    L.call("chelis_cuda_expert_route_bwd", dt, logits.data_ptr(), experts.data_ptr(),
           dweights.data_ptr(), logits.shape[0], logits.shape[1], experts.shape[1],
           int(renormalize), dlogits.data_ptr())
    return dlogits


def expert_sort(experts: torch.Tensor, n_experts: int) -> ExpertOrder:
    """The stable order by expert of the (token, slot) pairs of experts
    [tokens, k]; an id of -1 is a pair that goes nowhere.  Other ids outside
    [0, n_experts) count as -1 and raise at the next device_status()."""
    _check_i32("expert_sort", experts)
    if experts.dim() != 2:
        raise ValueError("expert_sort takes experts [tokens, k]")
    _prepare(experts)
    dev = experts.device
    order = ExpertOrder(torch.empty(max(n_experts, 0) + 1, dtype=torch.int32, device=dev),
                        torch.empty_like(experts),
                        torch.empty(experts.numel(), dtype=torch.int32, device=dev))
    L.call("chelis_cuda_expert_sort", experts.data_ptr(), experts.shape[0], experts.shape[1],
           n_experts, *(t.data_ptr() for t in order))
    return order


def expert_gather(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """Token rows x [tokens, hidden] to their experts' rows [tokens * k,
    hidden]; rows that no pair takes (the last ones) are zeros."""
    dt = _act("expert_gather", x)
    _check_order("expert_gather", order)
    if x.dim() != 2 or x.shape[0] != order.position.shape[0]:
        raise ValueError("expert_gather takes x [tokens, hidden]")
    _prepare(x, *order)
    tokens, k = order.position.shape
    xs = torch.empty(tokens * k, x.shape[1], dtype=x.dtype, device=x.device)
    L.call("chelis_cuda_expert_spread", dt, x.data_ptr(), order.position.data_ptr(), _routed(order),
           tokens, k, x.shape[1], xs.data_ptr())
    return xs


def _expert_combine(name, ys, weights, order):
    dt = _act(name, ys)
    _check_order(name, order)
    tokens, k = order.position.shape
    if ys.dim() != 2 or ys.shape[0] != tokens * k:
        raise ValueError(f"{name} takes rows [tokens * k, hidden]")
    if weights is not None and (weights.dtype != torch.float32 or weights.shape != (tokens, k)):
        raise ValueError(f"{name} takes f32 weights [tokens, k]")
    _prepare(ys, weights, *order)
    y = torch.empty(tokens, ys.shape[1], dtype=ys.dtype, device=ys.device)
    L.call("chelis_cuda_expert_combine", dt, ys.data_ptr(), _ptr(weights), order.position.data_ptr(),
           tokens, k, ys.shape[1], y.data_ptr())
    return y


def expert_gather_bwd(dxs: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """dx of expert_gather: each token's rows summed in slot order."""
    return _expert_combine("expert_gather_bwd", dxs, None, order)


def expert_combine(ys: torch.Tensor, weights: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """The way back: y[t] = sum_j weights[t, j] * ys[position[t, j]], f32 sums
    in slot order."""
    if weights is None:
        raise ValueError("expert_combine takes weights")
    return _expert_combine("expert_combine", ys, weights, order)


def expert_combine_bwd(dy: torch.Tensor, ys: torch.Tensor, weights: torch.Tensor, order: ExpertOrder):
    """(dys, dweights) of expert_combine."""
    dt = _act("expert_combine_bwd", dy)
    _check_order("expert_combine_bwd", order)
    tokens, k = order.position.shape
    if not (ys.dtype == dy.dtype and dy.dim() == 2 and dy.shape[0] == tokens
            and ys.shape == (tokens * k, dy.shape[1])):
        raise ValueError("expert_combine_bwd takes dy [tokens, hidden] and rows [tokens * k, hidden] of one dtype")
    if weights.dtype != torch.float32 or weights.shape != (tokens, k):
        raise ValueError("expert_combine_bwd takes f32 weights [tokens, k]")
    _prepare(dy, ys, weights, *order)
    dys = torch.empty_like(ys)
    dweights = torch.empty_like(weights)
    L.call("chelis_cuda_expert_combine_bwd", dt, dy.data_ptr(), ys.data_ptr(), weights.data_ptr(),
           order.position.data_ptr(), _routed(order), tokens, k, dy.shape[1], dys.data_ptr(),
           dweights.data_ptr())
    return dys, dweights


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


def quantize8(x: torch.Tensor, format: str = "e4m3", blocks: str = "rows") -> Blocks8:
    """x in 8 bits (e4m3 or e5m2) with a power-of-two scale for each block of
    128: along its rows ("rows", x [rows, cols]; activations, gradients) or
    128 x 128 ("tiles", x [rows, cols] or [experts, rows, cols]; weights)."""
    dt = _act("quantize8", x)
    if format not in _FLOAT8:
        raise ValueError("8-bit formats are e4m3 and e5m2")
    if blocks not in ("rows", "tiles"):
        raise ValueError("blocks are rows or tiles")
    if not (x.dim() == 2 or (x.dim() == 3 and blocks == "tiles")):
        raise ValueError("quantize8 takes a matrix, or a stack of matrices in tiles")
    _prepare(x)
    rows, cols = x.shape[-2:]
    batch = x.shape[0] if x.dim() == 3 else 1
    kb = _ceil(cols, 128)
    data = torch.empty(*x.shape[:-1], _ceil(cols, 16) * 16, dtype=_FLOAT8[format], device=x.device)
    shape = (kb, rows) if blocks == "rows" else (*x.shape[:-2], _ceil(rows, 128), kb)
    scales = torch.empty(*shape, dtype=torch.float32, device=x.device)
    L.call("chelis_cuda_quantize8", dt, _FORMAT[data.dtype],
           L.BLOCKS_ROWS if blocks == "rows" else L.BLOCKS_TILES, x.data_ptr(), batch, rows, cols,
           data.data_ptr(), scales.data_ptr())
    return Blocks8(data, scales, cols, blocks)


def quantize8_transposed(x: torch.Tensor, format: str = "e4m3",
                         offsets: torch.Tensor | None = None) -> Blocks8:
    """x [rows, cols] turned over and in 8 bits, blocks of 128 of its rows: the
    operand of matmul8_wgrad.  With offsets (expert_sort's) each expert's rows
    start on a block of their own."""
    dt = _act("quantize8_transposed", x)
    if format not in _FLOAT8:
        raise ValueError("8-bit formats are e4m3 and e5m2")
    if x.dim() != 2:
        raise ValueError("quantize8_transposed takes a matrix")
    groups = 0
    if offsets is not None:
        _check_i32("quantize8_transposed", offsets)
        if offsets.dim() != 1 or offsets.numel() < 2:
            raise ValueError("offsets are [experts + 1]")
        groups = offsets.numel() - 1
    _prepare(x, offsets)
    rows, cols = x.shape
    places = int(L.load().chelis_cuda_quantize8_places(rows, groups))
    data = torch.empty(cols, places, dtype=_FLOAT8[format], device=x.device)
    scales = torch.empty(places // 128, cols, dtype=torch.float32, device=x.device)
    L.call("chelis_cuda_quantize8_transposed", dt, _FORMAT[data.dtype], x.data_ptr(), _ptr(offsets),
           groups, rows, cols, data.data_ptr(), scales.data_ptr())
    return Blocks8(data, scales, places, "rows")


def _check_blocks8(name: str, b: Blocks8, blocks: str) -> None:
    data, scales, cols, kind = b
    if kind != blocks or data.dtype not in _FORMAT or scales.dtype != torch.float32:
        raise ValueError(f"{name} takes 8-bit {blocks} with f32 scales here")
    d, s = data.shape, scales.shape
    if len(d) < 2 or len(s) != (len(d) if blocks == "tiles" else 2):
        ok = False
    elif blocks == "tiles":
        ok = s[-1] == (cols + 127) // 128 and s[-2] == (d[-2] + 127) // 128 and s[:-2] == d[:-2]
    else:
        ok = s[0] == (cols + 127) // 128 and s[1] == d[-2]
    if not ok or d[-1] != (cols + 15) // 16 * 16:
        raise ValueError(f"{name}: data and scales do not belong together")


def matmul8(a: Blocks8, b: Blocks8, trans_b: bool = True, offsets: torch.Tensor | None = None,
            dtype: torch.dtype = torch.bfloat16, any_scales: bool = False) -> torch.Tensor:
    """a . b^T (b [n, k]: a layer's product) or a . b (trans_b=False, b [k, n]:
    its input gradient, from the same weights) of 8-bit row blocks a [rows, k]
    and tiles b; f32 sums, rounded once to dtype.  With offsets (expert_sort's)
    b is a stack of matrices and rows [offsets[e], offsets[e + 1]) meet matrix
    e; rows that no expert holds come out as zeros.  Scales are powers of two,
    as quantize8 makes them (others give NaN and raise at the next
    device_status(), whatever the size); any_scales admits every scale, at a
    lower rate."""
    if dtype not in _ACT:
        raise ValueError("matmul8 gives f32, bf16 or f16")
    _check_blocks8("matmul8", a, "rows")
    _check_blocks8("matmul8", b, "tiles")
    if a.data.dim() != 2 or b.data.dim() != (2 if offsets is None else 3):
        raise ValueError("matmul8 takes a matrix b, or a stack of them with offsets")
    groups = 1
    if offsets is not None:
        _check_i32("matmul8", offsets)
        groups = b.data.shape[0]
        if offsets.shape != (groups + 1,):
            raise ValueError("offsets are [experts + 1]")
    n, k = (b.data.shape[-2], b.cols) if trans_b else (b.cols, b.data.shape[-2])
    if a.cols != k:
        raise ValueError(f"contraction extents differ: {a.cols} vs {k}")
    _prepare(a.data, a.scales, b.data, b.scales, offsets)
    rows = a.data.shape[0]
    out = torch.empty(rows, n, dtype=dtype, device=a.data.device)
    L.call("chelis_cuda_matmul8", _FORMAT[a.data.dtype], _FORMAT[b.data.dtype], int(trans_b), rows, n,
           k, a.data.data_ptr(), a.scales.data_ptr(), b.data.data_ptr(), b.scales.data_ptr(),
           _ptr(offsets), groups, int(any_scales), _ACT[dtype], out.data_ptr())
    return out


def matmul8_wgrad(dy: Blocks8, x: Blocks8, offsets: torch.Tensor | None = None,
                  dtype: torch.dtype = torch.float32, any_scales: bool = False) -> torch.Tensor:
    """The weight gradient dy^T . x [n, k] from the transposed 8-bit forms of
    dy [rows, n] and x [rows, k] (quantize8_transposed); with offsets one
    matrix an expert, [experts, n, k], zeros for an expert without rows.
    any_scales as in matmul8."""
    if dtype not in _ACT:
        raise ValueError("matmul8_wgrad gives f32, bf16 or f16")
    _check_blocks8("matmul8_wgrad", dy, "rows")
    _check_blocks8("matmul8_wgrad", x, "rows")
    if dy.cols != x.cols or dy.cols % 128:
        raise ValueError("matmul8_wgrad takes operands over the same rows")
    n, k = dy.data.shape[0], x.data.shape[0]
    groups = 0
    if offsets is not None:
        _check_i32("matmul8_wgrad", offsets)
        if offsets.dim() != 1 or offsets.numel() < 2:
            raise ValueError("offsets are [experts + 1]")
        groups = offsets.numel() - 1
        if dy.cols < 128 * groups:
            raise ValueError("the operands were not turned over with these offsets")
    _prepare(dy.data, dy.scales, x.data, x.scales, offsets)
    shape = (n, k) if offsets is None else (groups, n, k)
    out = torch.empty(*shape, dtype=dtype, device=dy.data.device)
    L.call("chelis_cuda_matmul8_wgrad", _FORMAT[dy.data.dtype], _FORMAT[x.data.dtype], n, k, dy.cols,
           dy.data.data_ptr(), dy.scales.data_ptr(), x.data.data_ptr(), x.scales.data_ptr(),
           _ptr(offsets), max(groups, 1), int(any_scales), _ACT[dtype], out.data_ptr())
    return out


# ---------------------------------------------------------------- a feed-forward sublayer in 16 bits

_HALF = {torch.bfloat16: L.DTYPE_BF16, torch.float16: L.DTYPE_F16}
_ACTIVATION = {None: L.ACT_NONE, "relu": L.ACT_RELU, "gelu": L.ACT_GELU, "silu": L.ACT_SILU}
_NORM = {"layer": L.NORM_LAYER, "rms": L.NORM_RMS}
_dtype_of = operator.attrgetter("dtype")


class _Packed:
    """An entry called with its arguments packed (chelis_cuda_call_packed): with
    few tokens a call is mostly the binding's.  fmt: q an integer or a pointer, d a
    float; the stream comes first."""

    def __init__(self, entry: int, fmt: str):
        self.entry, self.pack, self.f = entry, struct.Struct("=q" + fmt).pack, None

    def __call__(self, *args) -> None:
        if self.f is None:
            self.f = L.load().chelis_cuda_call_packed
        status = self.f(self.entry, self.pack(*args))
        if status:
            L.check(status)


_matmul16 = _Packed(L.PACKED_MATMUL16, "16q")
_activation16_bwd = _Packed(L.PACKED_ACTIVATION16_BWD, "6q")
_column_sums16 = _Packed(L.PACKED_COLUMN_SUMS16, "5q")
_residual_norm = _Packed(L.PACKED_RESIDUAL_NORM, "10qd2qd2q")
_residual_norm_bwd = _Packed(L.PACKED_RESIDUAL_NORM_BWD, "12qdqd7q")
_expert_balance = _Packed(L.PACKED_EXPERT_BALANCE, "9q")
_expert_balance_bwd = _Packed(L.PACKED_EXPERT_BALANCE_BWD, "7qd3q")
_grad_norm = _Packed(L.PACKED_GRAD_NORM, "5q")
_clip_grads = _Packed(L.PACKED_CLIP_GRADS, "6qdq")


def _at(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _begin(name: str, *tensors: torch.Tensor | None) -> int:
    """The stream for a call on these tensors, which are contiguous and lie on one
    device, the current one."""
    dev = -1
    for t in tensors:
        if t is None:
            continue
        at = t.get_device()
        if at < 0:
            raise ValueError("chelis_b200 ops take CUDA tensors (device memory)")
        if not t.is_contiguous():
            raise ValueError("chelis_b200 ops take contiguous tensors")
        if dev < 0:
            dev = at
        elif at != dev:
            raise ValueError(f"{name}: tensors on different devices")
    return _on_device(name, dev)


def _on_device(name: str, dev: int) -> int:
    current = torch.cuda.current_device()
    if dev >= 0 and dev != current:
        raise ValueError(f"{name}: the tensors' device is not the current one")
    if current not in _initialised:
        L.call("chelis_cuda_init", current)
        _initialised.add(current)
    return _raw_stream(current)


def _half(name: str, t: torch.Tensor) -> int:
    if t.dtype not in _HALF:
        raise ValueError(f"{name} takes bf16 or f16 tensors")
    return _HALF[t.dtype]


def _activation(name: str, activation: str | None) -> int:
    if activation not in _ACTIVATION:
        raise ValueError(f"{name}: activations are relu, gelu and silu")
    return _ACTIVATION[activation]


def matmul16(a: torch.Tensor, b: torch.Tensor, trans_a: bool = False, trans_b: bool = False, *,
             bias: torch.Tensor | None = None, activation: str | None = None,
             residual: torch.Tensor | None = None, keep_pre: bool = False,
             through: tuple[torch.Tensor, str] | None = None, dtype: torch.dtype | None = None):
    """act(op(a).op(b) + bias) + residual of two bf16 or two f16 matrices: f32
    sums on the tensor cores, what follows them in the same kernel, one
    rounding to dtype (f32 or the operands' own, the default).  The tensor
    core's sums of normal numbers are 4e-6 off at k = 4096 and 2e-5 at 16384;
    without an activation they are added up from chunks, so that f32 results are
    1e-6 off and 16-bit ones no more than those 2e-5 at any k.  activation is
    relu, gelu (exact) or silu; bias [n] is f32 or of the operands' type, and
    residual [m, n] of dtype.  keep_pre: (y, z) with z = op(a).op(b) + bias, what
    the activation's gradient needs.

    through=(z, activation) gives the gradient through an activation that was
    taken at z [m, n], (op(a).op(b)) * act'(z), and goes with none of the
    others."""
    dt = _half("matmul16", a)
    if b.dtype != a.dtype or a.dim() != 2 or b.dim() != 2:
        raise ValueError("matmul16 takes two bf16 or two f16 matrices")
    dtype = a.dtype if dtype is None else dtype
    if dtype != a.dtype and dtype != torch.float32:
        raise ValueError("matmul16 gives f32 or its operands' type")
    m, k = a.shape[::-1] if trans_a else a.shape
    k2, n = b.shape[::-1] if trans_b else b.shape
    if k != k2:
        raise ValueError(f"contraction extents differ: {k} vs {k2}")
    z = None
    if through is not None:
        if bias is not None or activation is not None or residual is not None or keep_pre:
            raise ValueError("matmul16: through goes with no bias, activation, residual or keep_pre")
        z, activation = through
    act = _activation("matmul16", activation)
    if bias is not None and (bias.shape != (n,) or bias.dtype not in (a.dtype, torch.float32)):
        raise ValueError("matmul16: bias is [n], f32 or of the operands' type")
    for t in (residual, z):
        if t is not None and (t.shape != (m, n) or t.dtype != dtype):
            raise ValueError("matmul16: residual and through are [m, n] of the result's type")
    stream = _begin("matmul16", a, b, bias, residual, z)
    out = torch.empty(m, n, dtype=dtype, device=a.device)
    pre = torch.empty_like(out) if keep_pre else None
    _matmul16(stream, dt, int(trans_a), int(trans_b), m, n, k, a.data_ptr(), b.data_ptr(),
           _at(bias), 0 if bias is None else _ACT[bias.dtype], act, _at(residual), _at(z), _at(pre),
           _ACT[dtype], out.data_ptr())
    return (out, pre) if keep_pre else out


def activation16_bwd(dy: torch.Tensor, pre: torch.Tensor, activation: str | None) -> torch.Tensor:
    """dz = dy * act'(pre), of bf16 or f16 tensors."""
    dt = _half("activation16_bwd", dy)
    act = _activation("activation16_bwd", activation)
    if pre.dtype != dy.dtype or pre.shape != dy.shape:
        raise ValueError("activation16_bwd takes two tensors of one dtype and shape")
    stream = _begin("activation16_bwd", dy, pre)
    dz = torch.empty_like(dy)
    _activation16_bwd(stream, dt, act, dy.data_ptr(), pre.data_ptr(), dy.numel(), dz.data_ptr())
    return dz


def column_sums16(x: torch.Tensor) -> torch.Tensor:
    """The f32 sums over the rows of a bf16 or f16 matrix."""
    dt = _half("column_sums16", x)
    if x.dim() != 2:
        raise ValueError("column_sums16 takes a matrix")
    stream = _begin("column_sums16", x)
    out = torch.empty(x.shape[1], dtype=torch.float32, device=x.device)
    _column_sums16(stream, dt, x.data_ptr(), x.shape[0], x.shape[1], out.data_ptr())
    return out


def matmul16_bwd(dy: torch.Tensor, a: torch.Tensor, b: torch.Tensor, trans_b: bool = False, *,
                 through: tuple[torch.Tensor, str] | None = None, want_bias: bool = False,
                 weight_dtype: torch.dtype = torch.float32):
    """(da, db, dbias) of matmul16(a, b, trans_b=trans_b, bias=...) without an
    activation; of one with an activation, given dy = activation16_bwd's.  db has
    b's shape and weight_dtype (f32 or the operands' own), dbias is f32, None
    without want_bias.  through=(z, activation): a was that activation taken at
    z, and da is the gradient of z."""
    if dy.dim() != 2 or a.dim() != 2 or b.dim() != 2 or not dy.dtype == a.dtype == b.dtype:
        raise ValueError("matmul16_bwd takes matrices of one dtype")
    if dy.shape != (a.shape[0], b.shape[0] if trans_b else b.shape[1]):
        raise ValueError("matmul16_bwd: dy is not the product's shape")
    da = matmul16(dy, b, trans_b=not trans_b, through=through)
    if trans_b:
        db = matmul16(dy, a, trans_a=True, dtype=weight_dtype)
    else:
        db = matmul16(a, dy, trans_a=True, dtype=weight_dtype)
    return da, db, column_sums16(dy) if want_bias else None


class ResidualNormGrads(NamedTuple):
    """residual_norm_bwd's; None for what the forward call did not have."""
    dx: torch.Tensor
    dbranch: torch.Tensor | None
    dpost_gamma: torch.Tensor | None
    dpost_beta: torch.Tensor | None
    dgate: torch.Tensor | None
    dpre_gamma: torch.Tensor | None
    dpre_beta: torch.Tensor | None


def _check_norm(name, x, post_gamma, post_beta, gate, pre_gamma, pre_beta, kind):
    """(dtype, kind, rows, hidden, groups) of residual_norm's arguments."""
    dt = _act(name, x)
    if kind not in _NORM:
        raise ValueError(f"{name}: kinds are layer and rms")
    if x.dim() < 2:
        raise ValueError(f"{name} takes rows [..., hidden]")
    hidden = x.shape[-1]
    rows = x.numel() // hidden if hidden else 0
    for t in (post_gamma, post_beta, pre_gamma, pre_beta):
        if t is not None and (t.dtype != torch.float32 or t.shape != (hidden,)):
            raise ValueError(f"{name}: gammas and betas are f32 [hidden]")
    if (post_beta is not None and post_gamma is None) or (pre_beta is not None and pre_gamma is None):
        raise ValueError(f"{name}: a beta without its gamma")
    groups = 1
    if gate is not None:
        if gate.dtype != torch.float32 or gate.dim() not in (1, 2) or gate.shape[-1] != hidden:
            raise ValueError(f"{name}: a gate is f32 [hidden] or [groups, hidden]")
        groups = gate.shape[0] if gate.dim() == 2 else 1
        if groups < 1 or rows % groups:
            raise ValueError(f"{name}: the gate's groups divide the rows")
    return dt, _NORM[kind], rows, hidden, groups


def residual_norm(x: torch.Tensor, branch: torch.Tensor | None, *, post_gamma: torch.Tensor | None = None,
                  post_beta: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  scale: float = 1.0, pre_gamma: torch.Tensor | None = None,
                  pre_beta: torch.Tensor | None = None, eps: float = 1e-5, kind: str = "layer"):
    """What stands between two blocks, in one pass over the rows [..., hidden]:
    (y, h) with y = scale * x + gate * N(branch) and h = N(y), each norm with its
    own gamma and beta and left out without a gamma (h is None then), the gate
    [hidden], [groups, hidden] (equal runs of rows) or None.  kind is layer or rms.
    x, branch, y and h are f32, bf16 or f16 of one dtype, rows at most 8192 long,
    the parameters f32; h is taken of y before it is rounded.  With branch None: (x, N(x)), the first norm of all."""
    dt, norm, rows, hidden, groups = _check_norm("residual_norm", x, post_gamma, post_beta, gate, pre_gamma,
                                                 pre_beta, kind)
    if branch is None:
        if post_gamma is not None or gate is not None or scale != 1.0 or pre_gamma is None:
            raise ValueError("residual_norm: without a branch there is the second norm alone")
    elif branch.shape != x.shape or branch.dtype != x.dtype:
        raise ValueError("residual_norm: x and branch are of one dtype and shape")
    stream = _begin("residual_norm", x, branch, post_gamma, post_beta, gate, pre_gamma, pre_beta)
    y = None if branch is None else torch.empty_like(x)
    h = None if pre_gamma is None else torch.empty_like(x)
    _residual_norm(stream, dt, norm, rows, hidden, x.data_ptr(), _at(branch), _at(post_gamma),
           _at(post_beta), _at(gate), groups, float(scale), _at(pre_gamma), _at(pre_beta), float(eps),
           _at(y), _at(h))
    return x if y is None else y, h


def residual_norm_bwd(dy: torch.Tensor | None, dh: torch.Tensor | None, y: torch.Tensor,
                      branch: torch.Tensor | None, *, post_gamma: torch.Tensor | None = None,
                      post_beta: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                      scale: float = 1.0, pre_gamma: torch.Tensor | None = None,
                      pre_beta: torch.Tensor | None = None, eps: float = 1e-5,
                      kind: str = "layer") -> ResidualNormGrads:
    """The gradients of residual_norm, from dy (None: nothing else reads y) and
    dh (with pre_gamma), its result y, its branch and its parameters."""
    dt, norm, rows, hidden, groups = _check_norm("residual_norm_bwd", y, post_gamma, post_beta, gate, pre_gamma,
                                                 pre_beta, kind)
    if (dh is None) != (pre_gamma is None):
        raise ValueError("residual_norm_bwd: dh goes with pre_gamma")
    if dy is None and dh is None:
        raise ValueError("residual_norm_bwd takes dy, dh or both")
    if branch is None and (post_gamma is not None or gate is not None or scale != 1.0):
        raise ValueError("residual_norm_bwd: without a branch there is the second norm alone")
    for t in (dy, dh, branch):
        if t is not None and (t.shape != y.shape or t.dtype != y.dtype):
            raise ValueError("residual_norm_bwd: dy, dh, y and branch are of one dtype and shape")
    stream = _begin("residual_norm_bwd", dy, dh, y, branch, post_gamma, post_beta, gate, pre_gamma, pre_beta)

    def like(p):
        return None if p is None else torch.empty_like(p)

    g = ResidualNormGrads(torch.empty_like(y), like(branch), like(post_gamma), like(post_beta), like(gate),
                          like(pre_gamma), like(pre_beta))
    _residual_norm_bwd(stream, dt, norm, rows, hidden, _at(dy), _at(dh), y.data_ptr(),
           _at(branch), _at(post_gamma), _at(post_beta), _at(gate), groups, float(scale), _at(pre_gamma),
           float(eps), *(_at(t) for t in g))
    return g


def expert_balance(logits: torch.Tensor, experts: torch.Tensor, mask: torch.Tensor | None = None):
    """(loss f32 [], counts int32 [experts + 1]) of a router's logits [tokens,
    experts] and the experts [tokens, k] that it chose: loss = E / (k N^2) sum_e
    counts[e] sum_t softmax(logits[t])_e over the N tokens that count, all or
    those where mask (bool [tokens]) is true; 1 where both are even.  counts are
    the tokens' pairs by expert, then N.  An id of -1 counts nowhere; other ids
    outside [0, experts) too, and they raise at the next device_status()."""
    dt = _act("expert_balance", logits)
    _check_i32("expert_balance", experts)
    if logits.dim() != 2 or experts.dim() != 2 or experts.shape[0] != logits.shape[0]:
        raise ValueError("expert_balance takes logits [tokens, experts] and experts [tokens, k]")
    tokens, n = logits.shape
    if mask is not None and (mask.dtype != torch.bool or mask.shape != (tokens,)):
        raise ValueError("expert_balance: mask is bool [tokens]")
    stream = _begin("expert_balance", logits, experts, mask)
    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    counts = torch.empty(n + 1, dtype=torch.int32, device=logits.device)
    _expert_balance(stream, dt, logits.data_ptr(), experts.data_ptr(), _at(mask), tokens, n,
           experts.shape[1], loss.data_ptr(), counts.data_ptr())
    return loss, counts


def expert_balance_bwd(logits: torch.Tensor, counts: torch.Tensor, k: int, weight: float = 1.0,
                       dloss: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                       add: torch.Tensor | None = None) -> torch.Tensor:
    """dlogits = weight * dloss * (the gradient of expert_balance's loss) + add,
    rounded once: the gradient through the probabilities, the counts held
    constant.  dloss is an f32 scalar on the device (None: 1), add another
    gradient of the logits (expert_route_bwd's)."""
    dt = _act("expert_balance_bwd", logits)
    _check_i32("expert_balance_bwd", counts)
    if logits.dim() != 2 or counts.shape != (logits.shape[1] + 1,):
        raise ValueError("expert_balance_bwd takes logits [tokens, experts] and expert_balance's counts")
    tokens, n = logits.shape
    if mask is not None and (mask.dtype != torch.bool or mask.shape != (tokens,)):
        raise ValueError("expert_balance_bwd: mask is bool [tokens]")
    if dloss is not None and (dloss.dtype != torch.float32 or dloss.numel() != 1):
        raise ValueError("expert_balance_bwd: dloss is one f32 number")
    if add is not None and (add.dtype != logits.dtype or add.shape != logits.shape):
        raise ValueError("expert_balance_bwd: add has the logits' dtype and shape")
    stream = _begin("expert_balance_bwd", logits, counts, dloss, mask, add)
    dlogits = torch.empty_like(logits)
    _expert_balance_bwd(stream, dt, logits.data_ptr(), counts.data_ptr(), _at(mask), tokens, n, k,
           float(weight), _at(dloss), _at(add), dlogits.data_ptr())
    return dlogits


def _tensor_list(name: str, tensors: list):
    """The stream for a call on a list of tensors, and what it takes of them:
    (pointers, sizes, dtypes), host arrays."""
    devices = set(map(torch.Tensor.get_device, tensors))
    if len(devices) > 1:
        raise ValueError(f"{name}: tensors on different devices")
    if -1 in devices:
        raise ValueError("chelis_b200 ops take CUDA tensors (device memory)")
    if not all(map(torch.Tensor.is_contiguous, tensors)):
        raise ValueError("chelis_b200 ops take contiguous tensors")
    stream = _on_device(name, devices.pop() if devices else -1)
    try:
        dtypes = array.array("i", map(_ACT.__getitem__, map(_dtype_of, tensors)))
    except KeyError:
        raise ValueError(f"{name} takes f32, bf16 or f16 tensors") from None
    return (stream, array.array("Q", map(torch.Tensor.data_ptr, tensors)),
            array.array("q", map(torch.Tensor.numel, tensors)), dtypes)


def _address(a: array.array) -> int:
    return a.buffer_info()[0]


def grad_norm(grads) -> torch.Tensor:
    """The Euclidean norm over all numbers of a list of f32, bf16 or f16
    tensors, an f32 scalar on the device; sums in f64."""
    grads = list(grads)
    stream, *src = _tensor_list("grad_norm", grads)
    norm = torch.empty((), dtype=torch.float32, device="cuda" if not grads else grads[0].device)
    _grad_norm(stream, len(grads), *map(_address, src), norm.data_ptr())
    return norm


def clip_grads(grads, max_norm: float, out=None) -> torch.Tensor:
    """Scale a list of f32, bf16 or f16 tensors by min(1, max_norm / norm), norm
    their grad_norm, which is returned: in place, or with out into tensors of the
    same sizes (f32, bf16 or f16), which are written in any case.  A norm that is
    not finite changes nothing.  Tensors that overlap are refused."""
    grads = list(grads)
    n, own = len(grads), out is None
    if not own:
        grads += out
        if len(grads) != 2 * n:
            raise ValueError("clip_grads: out has the gradients' sizes")
    stream, ptrs, counts, dtypes = _tensor_list("clip_grads", grads)
    if not own and counts[:n] != counts[n:]:
        raise ValueError("clip_grads: out has the gradients' sizes")
    norm = torch.empty((), dtype=torch.float32, device="cuda" if not grads else grads[0].device)
    at, kinds, skip = _address(ptrs), _address(dtypes), 0 if own else n
    _clip_grads(stream, n, at, _address(counts), kinds, at + skip * ptrs.itemsize,
                kinds + skip * dtypes.itemsize, float(max_norm), norm.data_ptr())
    return norm
