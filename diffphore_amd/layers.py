"""Trainable layers on packed complexes: layer norm and attention, each with its forward and its backward pass.

The layers of the reference's attention variant (src/models/e3phore.py: layer norm, attention of the nodes of a complex over the nodes of its
pharmacophore with a bias per pair) as operators on the batch layout of this package: the nodes of all complexes of a batch one behind the other, CSR
offsets per complex (`engine.PackedBatch`).  `layer_norm` and `attention` take part in autograd; the `*_forward` / `*_backward` functions are the same
kernels for hosts that keep the book themselves.  fp32 and bf16; everything runs in libdiffphore_train.so, there is no fallback.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import _trainlib
from ._trainlib import TYPES, DptAttnArgs, Streams, call, need_gpu

_LN_MAX_WIDTH = 16384
_MAX_ROWS = 2 ** 31 - 1025                              # DPT_ATTN_MAX_ROWS


# ----------------------------------------------------------------------------------------------------------------------
# layer norm
# ----------------------------------------------------------------------------------------------------------------------
def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, width] with unit stride inside a row (a copy only where the strides do not allow a view)."""
    y = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return y if y.stride(1) == 1 or y.shape[1] == 1 else y.contiguous()


def _empty_like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _row_stride(x2: torch.Tensor) -> int:
    return x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]


def _check_affine(x, p, name):
    if p is None or (type(p) is torch.Tensor and p.dtype is x.dtype and p.shape == x.shape[-1:] and p.device == x.device and p.is_contiguous()):
        return
    need_gpu(p, name)
    if p.device != x.device:
        raise ValueError(f"{name} is on {p.device}, x on {x.device}")
    if p.dtype != x.dtype and p.dtype != torch.float32:
        raise TypeError(f"{name} is {p.dtype}: it has the type of x ({x.dtype}) or float32")
    if p.shape != x.shape[-1:]:
        raise ValueError(f"{name} has shape {tuple(p.shape)}, x has {x.shape[-1]} channels")
    if not p.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_ln(x, weight, bias):
    need_gpu(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x has shape {tuple(x.shape)}: a last dimension of at least 1 is wanted")
    if x.shape[-1] > _LN_MAX_WIDTH:
        raise ValueError(f"x has {x.shape[-1]} channels: at most {_LN_MAX_WIDTH} are supported")
    _check_affine(x, weight, "weight")
    _check_affine(x, bias, "bias")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight is {weight.dtype}, bias {bias.dtype}")


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """(y, mean, rstd): y = (x - mean) rstd weight + bias over the last dimension; mean and rstd fp32, one per row ([rows], row-major over x's other
    dimensions)."""
    _check_ln(x, weight, bias)
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps = {eps}")
    L = _trainlib.lib()
    x2 = _rows(x)
    rows, width = x2.shape
    y = _empty_like(x)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    w = weight if weight is not None else bias
    call("dpt_layer_norm_fwd", L.dpt_layer_norm_fwd, x.get_device(), TYPES[x.dtype], TYPES[w.dtype if w is not None else x.dtype], rows, width, x2.data_ptr(),
         _row_stride(x2), weight.data_ptr() if weight is not None else None, bias.data_ptr() if bias is not None else None, eps, y.data_ptr(), width,
         mean.data_ptr(), rstd.data_ptr())
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight: Optional[torch.Tensor] = None,
                        param_dtype: Optional[torch.dtype] = None, want_params: bool = True):
    """(dx, dweight, dbias) for the gradient dy of y; dweight and dbias in the weight's type (`param_dtype` where there is no weight, x's type by
    default), None each if `want_params` is False.  The sums over the rows are held in fp32 and joined in a fixed order."""
    _check_ln(x, weight, None)
    need_gpu(dy, "dy")
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError(f"dy is {tuple(dy.shape)} {dy.dtype} on {dy.device}, x is {tuple(x.shape)} {x.dtype} on {x.device}")
    L = _trainlib.lib()
    x2, dy2 = _rows(x), _rows(dy)
    rows, width = x2.shape
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        need_gpu(t, name)
        if t.dtype != torch.float32 or t.numel() != rows or t.device != x.device or not t.is_contiguous():
            raise ValueError(f"{name}: {rows} contiguous float32 values on {x.device} are wanted (layer_norm_forward's)")
    wtype = weight.dtype if weight is not None else param_dtype or x.dtype
    if wtype != x.dtype and wtype != torch.float32:
        raise TypeError(f"param_dtype {wtype}: x's type ({x.dtype}) or float32")
    dx = _empty_like(x)
    dw = db = ws = None
    n = 0
    if want_params:
        dw = torch.empty_like(weight) if weight is not None else torch.empty(width, dtype=wtype, device=x.device)
        db = torch.empty_like(dw)
        n = L.dpt_layer_norm_ws_bytes(rows, width)
        ws = torch.empty(n, dtype=torch.uint8, device=x.device)
    call("dpt_layer_norm_bwd", L.dpt_layer_norm_bwd, x.get_device(), TYPES[x.dtype], TYPES[wtype], rows, width, dy2.data_ptr(), _row_stride(dy2), x2.data_ptr(),
         _row_stride(x2), mean.data_ptr(), rstd.data_ptr(), weight.data_ptr() if weight is not None else None, dx.data_ptr(), width,
         dw.data_ptr() if want_params else None, db.data_ptr() if want_params else None, ws.data_ptr() if want_params else None, n)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.bias_dtype = bias.dtype if bias is not None else None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, mean, rstd, weight = ctx.saved_tensors
        want = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, param_dtype=ctx.bias_dtype, want_params=want)
        return dx if ctx.needs_input_grad[0] else None, dw if ctx.needs_input_grad[1] else None, db if ctx.needs_input_grad[2] else None, None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """Layer norm over the last dimension, differentiable (once) in x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, eps)


# ----------------------------------------------------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------------------------------------------------
def _offsets(p, name) -> np.ndarray:
    a = np.asarray(p.cpu() if isinstance(p, torch.Tensor) else p)
    if a.ndim != 1 or a.size < 1 or a.dtype.kind not in "iu":
        raise ValueError(f"{name}: a list of B + 1 integer offsets is wanted, got {a.dtype} {a.shape}")
    a = a.astype(np.int64)
    if a[0] != 0 or (np.diff(a) < 0).any():
        raise ValueError(f"{name}: offsets start at 0 and do not fall")
    if a[-1] > _MAX_ROWS:
        raise ValueError(f"{name}: {a[-1]} rows, at most {_MAX_ROWS} are supported")
    return a


class PairPlan:
    """Which query rows meet which key rows: complex b has the queries q_ptr[b] .. q_ptr[b+1] and the keys k_ptr[b] .. k_ptr[b+1] (host offsets, as the
    `lig_ptr` / `ph_ptr` of a packed batch) and its pairs, query-major, at pair_ptr[b] .. pair_ptr[b+1] of a pair array.  Built once per batch; the offsets
    are uploaded here, so a call with the plan touches no host data."""

    def __init__(self, q_ptr: Sequence[int], k_ptr: Sequence[int], device="cuda"):
        qp, kp = _offsets(q_ptr, "q_ptr"), _offsets(k_ptr, "k_ptr")
        if qp.size != kp.size:
            raise ValueError(f"q_ptr has {qp.size} offsets, k_ptr {kp.size}")
        nq, nk = np.diff(qp), np.diff(kp)
        pairs = np.concatenate(([0], np.cumsum(nq * nk)))
        self.B, self.n_q, self.n_k, self.n_pairs = int(nq.size), int(qp[-1]), int(kp[-1]), int(pairs[-1])
        self.max_nq, self.max_nk = int(nq.max(initial=0)), int(nk.max(initial=0))
        self.q_ptr, self.k_ptr, self.pair_ptr = qp, kp, pairs
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"device {device}: attention runs on the GPU only")
        self.device = torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)
        order = np.argsort(-(nq * nk), kind="stable")
        # one upload: pair_ptr (64 bits), then q_ptr, k_ptr, order
        host = np.concatenate((pairs.astype(np.int64).view(np.int32), qp.astype(np.int32), kp.astype(np.int32), order.astype(np.int32)))
        self._dev = torch.from_numpy(host).to(self.device)
        base, n = self._dev.data_ptr(), self.B + 1
        self._ptrs = (base + 8 * n, base + 12 * n, base, base + 16 * n)         # q_ptr, k_ptr, pair_ptr, order
        self._streams = Streams(self.device, [self._dev])

    def __reduce__(self):
        """A copy (copy.copy, copy.deepcopy, pickle) is a plan of its own: one with this plan's device addresses would outlive the memory behind them."""
        return PairPlan, (self.q_ptr, self.k_ptr, str(self.device))

    @classmethod
    def from_batch(cls, batch, queries: str = "ligand", keys: str = "phore") -> "PairPlan":
        """The plan of an `engine.PackedBatch`: the nodes of one kind attend over the nodes of another (or the same) kind of their complex."""
        counts = {"ligand": batch.nl, "phore": batch.np_}
        if queries not in counts or keys not in counts:
            raise ValueError(f"node kinds are 'ligand' and 'phore', got {queries!r}, {keys!r}")
        return cls(*(np.concatenate(([0], np.cumsum(np.asarray(counts[n], dtype=np.int64)))) for n in (queries, keys)), device=batch.device)


def _check_attn(q, k, v, plan, bias, scale):
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        need_gpu(t, name)
        if t.dim() != 3:
            raise ValueError(f"{name} has shape {tuple(t.shape)}: [rows, heads, dim] is wanted")
        if t.dtype is not q.dtype or t.get_device() != q.get_device():
            raise ValueError(f"{name} is {t.dtype} on {t.device}, q is {q.dtype} on {q.device}")
    if not isinstance(plan, PairPlan):
        raise TypeError(f"plan: a PairPlan is wanted, got {type(plan).__name__}")
    if plan.device.index != q.get_device():
        raise ValueError(f"the plan is on {plan.device}, q on {q.device}")
    heads, dim = q.shape[1:]
    if k.shape != v.shape or k.shape[2] != dim:
        raise ValueError(f"q is {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if heads < 1 or k.shape[1] < 1 or heads % k.shape[1]:
        raise ValueError(f"{heads} query heads cannot share {k.shape[1]} key heads")
    if not 1 <= dim <= 128:
        raise ValueError(f"head dimension {dim}: 1 to 128 are supported")
    if q.shape[0] != plan.n_q or k.shape[0] != plan.n_k:
        raise ValueError(f"{q.shape[0]} query and {k.shape[0]} key rows, the plan has {plan.n_q} and {plan.n_k}")
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:
        raise ValueError(f"scale = {scale}: a positive number from 2^-126 to 2^126 is wanted")
    if bias is not None:
        need_gpu(bias, "bias")
        if bias.shape != (heads, plan.n_pairs) or bias.dtype != q.dtype or bias.device != q.device:
            raise ValueError(f"bias is {tuple(bias.shape)} {bias.dtype} on {bias.device}: ({heads}, {plan.n_pairs}) {q.dtype} on {q.device} is wanted")


def _unit(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _attn_args(q, k, v, plan, bias, causal, scale) -> DptAttnArgs:
    a = DptAttnArgs()
    a.type, a.B, a.heads, a.kv_heads, a.dim, a.causal = TYPES[q.dtype], plan.B, q.shape[1], k.shape[1], q.shape[2], int(bool(causal))
    a.n_q, a.n_k, a.max_nq, a.max_nk, a.n_pairs, a.scale = plan.n_q, plan.n_k, plan.max_nq, plan.max_nk, plan.n_pairs, scale
    a.q_row, a.q_head, _ = q.stride()
    a.k_row, a.k_head, _ = k.stride()
    a.v_row, a.v_head, _ = v.stride()
    plan._streams.use()
    a.q_ptr, a.k_ptr, a.pair_ptr, a.order = plan._ptrs
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if bias is not None:
        a.bias_head, a.bias_pair = bias.stride()
        a.bias = bias.data_ptr()
    return a


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PairPlan, bias: Optional[torch.Tensor] = None, causal: bool = False,
                      scale: Optional[float] = None):
    """(out, stats) of softmax(scale q k^T + bias) v within each complex of the plan.

    q [n_q, heads, dim]; k, v [n_k, kv_heads, dim], heads a multiple of kv_heads (query head h reads key head h // (heads // kv_heads)); any strides with
    unit stride in dim.  bias [heads, n_pairs] (an expanded dimension is fine); -inf takes a pair out.  causal: query i sees key j iff
    j <= i + n_keys - n_queries of its complex.  scale: 1 / sqrt(dim) by default.  stats [2, heads, n_q] fp32: the largest score of a row and its sum of
    exponentials.  A row that sees no key has out = 0, stats = (-inf, 0)."""
    scale = 1.0 / math.sqrt(max(1, q.shape[-1])) if scale is None else float(scale)
    _check_attn(q, k, v, plan, bias, scale)
    L = _trainlib.lib()
    q, k, v = _unit(q), _unit(k), _unit(v)
    out = _empty_like(q)
    stats = torch.empty((2, q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device)
    a = _attn_args(q, k, v, plan, bias, causal, scale)
    a.out, a.stats = out.data_ptr(), stats.data_ptr()
    n = L.dpt_attn_ws_bytes(C.byref(a), 0)
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        a.ws, a.ws_bytes = ws.data_ptr(), n
    call("dpt_attn_fwd", L.dpt_attn_fwd, q.get_device(), C.byref(a))
    return out, stats


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, stats: torch.Tensor, plan: PairPlan,
                       bias: Optional[torch.Tensor] = None, causal: bool = False, scale: Optional[float] = None, want_bias: bool = True):
    """(dq, dk, dv, dbias) for the gradient dout of out; dbias [heads, n_pairs] for every pair, None without a bias or if `want_bias` is False.  The
    probabilities are formed again from the scores and `stats`."""
    scale = 1.0 / math.sqrt(max(1, q.shape[-1])) if scale is None else float(scale)
    _check_attn(q, k, v, plan, bias, scale)
    for t, name in ((dout, "dout"), (out, "out")):
        need_gpu(t, name)
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}, q is {tuple(q.shape)} {q.dtype} on {q.device}")
    need_gpu(stats, "stats")
    if stats.shape != (2, q.shape[1], q.shape[0]) or stats.dtype != torch.float32 or stats.device != q.device:
        raise ValueError(f"stats is {tuple(stats.shape)} {stats.dtype} on {stats.device}: attention_forward's is wanted")
    L = _trainlib.lib()
    q, k, v, dout, out, stats = _unit(q), _unit(k), _unit(v), _unit(dout), out.contiguous(), stats.contiguous()
    dq, dk, dv = _empty_like(q), _empty_like(k), _empty_like(v)
    dbias = _empty_like(bias) if bias is not None and want_bias else None
    a = _attn_args(q, k, v, plan, bias, causal, scale)
    a.dout_row, a.dout_head, _ = dout.stride()
    a.out, a.stats, a.dout, a.dq, a.dk, a.dv = (t.data_ptr() for t in (out, stats, dout, dq, dk, dv))
    if dbias is not None:
        a.dbias = dbias.data_ptr()
    n = L.dpt_attn_ws_bytes(C.byref(a), 1)
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        a.ws, a.ws_bytes = ws.data_ptr(), n
    call("dpt_attn_bwd", L.dpt_attn_bwd, q.get_device(), C.byref(a))
    return dq, dk, dv, dbias


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, plan, causal, scale):
        out, stats = attention_forward(q, k, v, plan, bias=bias, causal=causal, scale=scale)
        ctx.save_for_backward(q, k, v, bias, out, stats)
        ctx.how = plan, causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, bias, out, stats = ctx.saved_tensors
        plan, causal, scale = ctx.how
        need = ctx.needs_input_grad
        grads = attention_backward(dout, q, k, v, out, stats, plan, bias=bias, causal=causal, scale=scale, want_bias=need[3])
        return tuple(g if n else None for g, n in zip(grads, need)) + (None, None, None)


def attention(q, k, v, plan: PairPlan, bias=None, causal: bool = False, scale: Optional[float] = None):
    """`attention_forward`'s out, differentiable (once) in q, k, v and bias.  A bias shared by heads is passed expanded ([1, n_pairs] -> [heads, n_pairs]):
    its gradient is then summed over the heads by autograd."""
    return _Attention.apply(q, k, v, bias, plan, causal, scale)
