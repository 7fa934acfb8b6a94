"""The dense operators around a GAT layer: a linear layer with its epilogue, group normalisation with an
activation, embedding lookup, dropout (gat_amd/csrc/linear.hip, group_norm.hip, embedding.hip,
dropout.hip).

The reference's network has stock modules there or nothing; these are what a block around `GATConv` is
made of when it grows a skip connection, a per-node normalisation (no statistics over the batch, so none to
combine over the ranks of a partitioned graph) or categorical node features.  Each takes float32, bfloat16
or float16 tensors (all of one type), computes in float32 or wider and rounds every result once; the same
inputs give the same bits.  GPU only.  Gradients are those of one backward pass: a second derivative is
refused.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .glue import SEED_STEP

ACTIVATIONS = {"none": 0, "relu": 1, "elu": 2, "silu": 3, "gelu": 4}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
GROUP_NORM_MAX_CHANNELS = 8192      # GATMI_GROUP_NORM_MAX_CHANNELS


def _check(name: str, x: Tensor, *others) -> int:
    """Element type code of `x`, whose device and type the others (tensors or None) share."""
    if not x.is_cuda:
        raise RuntimeError(f"gat_amd.{name} runs on the GPU only (no CPU fallback)")
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"{name}: tensors must be float32, bfloat16 or float16, got {x.dtype}")
    for t in others:
        if t is None:
            continue
        if t.dtype != x.dtype:
            raise TypeError(f"{name}: all tensors must be {x.dtype}, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name}: tensors on {x.device} and {t.device}")
    return code


def _act(name: str, act: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"{name}: act must be one of {', '.join(ACTIVATIONS)}, got {act!r}")
    return code


_raw_stream = torch._C._cuda_getCurrentRawStream      # the current stream's handle, without a Stream object
_current = torch._C._cuda_getDevice


def _once(backward):
    """A backward that cannot itself be differentiated.  Without create_graph nothing could, and the guard
    (which costs as much as the call) is left out."""
    guarded = once_differentiable(backward)

    def run(ctx, grad_y):
        if _current() != grad_y.device.index:
            with torch.cuda.device(grad_y.device):
                return run(ctx, grad_y)
        return guarded(ctx, grad_y) if torch.is_grad_enabled() else backward(ctx, grad_y)
    return staticmethod(run)


class _NoCtx:
    """Stands for autograd's context where nothing needs a gradient"""

    def save_for_backward(self, *tensors):
        pass


def _apply(fn, x: Tensor, needs_grad: bool, *args):
    """fn on x's device, without autograd's machinery where nothing needs a gradient"""
    if _current() != x.device.index:
        with torch.cuda.device(x.device):
            return _apply(fn, x, needs_grad, *args)
    return fn.apply(*args) if needs_grad else fn.forward(_NoCtx(), *args)


# Workspace sizes by shape (a query through the C ABI costs as much as a small kernel)
@lru_cache(maxsize=4096)
def _linear_ws(device, rows, k, n, dtype, act):
    desc = _lib.Linear(rows, k, n, dtype, act)
    lib = _lib.lib()
    return (int(lib.gatmi_linear_fwd_workspace_bytes(C.byref(desc))),
            int(lib.gatmi_linear_bwd_workspace_bytes(C.byref(desc))))


@lru_cache(maxsize=4096)
def _embedding_ws(n, vocab, dim):
    return int(_lib.lib().gatmi_embedding_bwd_workspace_bytes(n, vocab, dim))


@lru_cache(maxsize=4096)
def _group_norm_ws(batch, length, groups, width, dtype):
    desc = _lib.GroupNorm(batch, length, groups, width, dtype, 0, 0.0, 0, None, None)
    return int(_lib.lib().gatmi_group_norm_workspace_bytes(C.byref(desc)))


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


# ---- linear ----------------------------------------------------------------------------------
class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, dtype, act, keep):
        lib, dev = _lib.lib(), x.device
        x, weight = x.contiguous(), weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        residual = None if residual is None else residual.contiguous()
        k, n = x.size(-1), weight.size(0)
        desc = _lib.Linear(x.numel() // k, k, n, dtype, act)
        st = _raw_stream(dev.index)
        y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=dev)
        slope = None
        if keep and act:
            slope = torch.empty(y.shape, dtype=torch.float32 if dtype == 0 else torch.int16, device=dev)
        need = _linear_ws(dev.index, desc.rows, k, n, dtype, act)[0]
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(lib.gatmi_linear_fwd(C.byref(desc), x.data_ptr(), weight.data_ptr(), _ptr(bias),
                                        _ptr(residual), y.data_ptr(), _ptr(slope), _ptr(ws), need, st),
                   "gatmi_linear_fwd")
        ctx.save_for_backward(x, weight, slope)
        ctx.desc = desc
        return y

    @_once
    def backward(ctx, grad_y):
        x, weight, slope = ctx.saved_tensors
        lib, dev, desc = _lib.lib(), x.device, ctx.desc
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        grad_res = grad_y if need_r else None
        gx = gw = gb = None
        if need_x or need_w or need_b:
            gy = grad_y.contiguous()
            st = _raw_stream(dev.index)
            gx = torch.empty_like(x) if need_x else None
            gw = torch.empty_like(weight) if need_w else None
            gb = torch.empty(weight.size(0), dtype=x.dtype, device=dev) if need_b else None
            need = _linear_ws(dev.index, desc.rows, desc.in_features, desc.out_features, desc.dtype, desc.act)[1]
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            _lib.check(lib.gatmi_linear_bwd(C.byref(desc), x.data_ptr(), weight.data_ptr(), _ptr(slope),
                                            gy.data_ptr(), _ptr(gx), _ptr(gw), _ptr(gb), ws.data_ptr(),
                                            need, st), "gatmi_linear_bwd")
        return gx, gw, gb, grad_res, None, None, None


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: str = "none",
               residual: Optional[Tensor] = None) -> Tensor:
    """act(x @ weight.T + bias) + residual in one kernel: x [..., in], weight [out, in], bias [out],
    residual [..., out]; act one of ACTIVATIONS ("gelu" is the exact form).  With `residual=conv(x)` it is
    the skip connection beside a GAT layer."""
    dtype = _check("linear_act", x, weight, bias, residual)
    code = _act("linear_act", act)
    if x.dim() < 1 or weight.dim() != 2 or x.size(-1) != weight.size(1) or weight.numel() == 0:
        raise ValueError(f"linear_act: x must be [..., {weight.size(-1) if weight.dim() else '?'}] and weight "
                         f"[out, in], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if bias is not None and bias.shape != (weight.size(0),):
        raise ValueError(f"linear_act: bias must be [{weight.size(0)}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != x.shape[:-1] + (weight.size(0),):
        raise ValueError(f"linear_act: residual must be {tuple(x.shape[:-1]) + (weight.size(0),)}, "
                         f"got {tuple(residual.shape)}")
    grad = torch.is_grad_enabled()
    keep = grad and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad))
    needs = keep or (grad and residual is not None and residual.requires_grad)
    return _apply(_LinearFn, x, needs, x, weight, bias, residual, dtype, code, keep)


# ---- group norm ------------------------------------------------------------------------------
def _gn_desc(shape, groups, dtype, act, eps, weight, bias):
    c = shape[-1]
    length = 1
    for s in shape[1:-1]:
        length *= s
    return _lib.GroupNorm(shape[0], length, groups, c // groups, dtype, act, eps, 0, weight.data_ptr(), bias.data_ptr())


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, dtype, act, eps, keep):
        lib, dev = _lib.lib(), x.device
        x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
        desc = _gn_desc(x.shape, groups, dtype, act, eps, weight, bias)
        st = _raw_stream(dev.index)
        y = torch.empty_like(x)
        stats = ws = None
        if keep or desc.length > 1 or desc.width > 2048:
            stats = torch.empty(2, x.size(0), groups, dtype=torch.float32, device=dev)
            ws = torch.empty(_group_norm_ws(desc.batch, desc.length, groups, desc.width, dtype), dtype=torch.uint8, device=dev)
        mean = _ptr(stats)
        _lib.check(lib.gatmi_group_norm_fwd(
            C.byref(desc), x.data_ptr(), y.data_ptr(), mean,
            None if stats is None else mean + 4 * x.size(0) * groups, _ptr(ws),
            0 if ws is None else ws.numel(), st), "gatmi_group_norm_fwd")
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.cfg = (groups, dtype, act, eps)
        return y

    @_once
    def backward(ctx, grad_y):
        x, weight, bias, stats = ctx.saved_tensors
        lib, dev = _lib.lib(), x.device
        desc = _gn_desc(x.shape, *ctx.cfg, weight, bias)
        gy = grad_y.contiguous()
        st = _raw_stream(dev.index)
        gx, gw, gb = torch.empty_like(x), torch.empty_like(weight), torch.empty_like(bias)
        need = _group_norm_ws(desc.batch, desc.length, desc.groups, desc.width, desc.dtype)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        mean = stats.data_ptr()
        _lib.check(lib.gatmi_group_norm_bwd(
            C.byref(desc), x.data_ptr(), gy.data_ptr(), mean, mean + 4 * x.size(0) * ctx.cfg[0],
            gx.data_ptr(), gw.data_ptr(), gb.data_ptr(), ws.data_ptr(), need, st), "gatmi_group_norm_bwd")
        return gx, gw, gb, None, None, None, None, None


def group_norm_act(x: Tensor, groups: int, weight: Tensor, bias: Tensor, eps: float = 1e-5,
                   act: str = "none") -> Tensor:
    """act(group_norm(x)) with channels last: x [N, C] or [N, ..., C], weight and bias [C], C = groups *
    width.  Mean and variance are those of one sample's group: its `width` channels at all positions between
    the first and the last axis.  For x [nodes, heads * channels] and groups = heads every node's heads are
    normalised one by one; for x [graphs, nodes, C] the statistics are a graph's."""
    dtype = _check("group_norm_act", x, weight, bias)
    code = _act("group_norm_act", act)
    groups = int(groups)
    if x.dim() < 2 or groups < 1 or x.size(-1) < 1 or x.size(-1) % groups:
        raise ValueError(f"group_norm_act: x must be [N, ..., C] with C a multiple of {groups} groups, got {tuple(x.shape)}")
    if x.size(-1) > GROUP_NORM_MAX_CHANNELS:
        raise ValueError(f"group_norm_act covers up to {GROUP_NORM_MAX_CHANNELS} channels, got {x.size(-1)}")
    if weight.shape != (x.size(-1),) or bias.shape != (x.size(-1),):
        raise ValueError(f"group_norm_act: weight and bias must be [{x.size(-1)}], got {tuple(weight.shape)}, "
                         f"{tuple(bias.shape)}")
    if x.dim() > 2 and x.size(0) > 0 and x.numel() == 0:
        raise ValueError(f"group_norm_act: samples without positions, {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"group_norm_act: eps must not be negative, got {eps}")
    keep = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or bias.requires_grad)
    return _apply(_GroupNormFn, x, keep, x, weight, bias, groups, dtype, code, float(eps), keep)


# ---- embedding -------------------------------------------------------------------------------
class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, dtype):
        lib, dev = _lib.lib(), table.device
        ids, table = ids.contiguous(), table.contiguous()
        vocab, dim = table.shape
        st = _raw_stream(dev.index)
        y = torch.empty(ids.shape + (dim,), dtype=table.dtype, device=dev)
        _lib.check(lib.gatmi_embedding_fwd(dtype, ids.numel(), vocab, dim, scale, ids.data_ptr(),
                                           table.data_ptr(), y.data_ptr(), st), "gatmi_embedding_fwd")
        ctx.save_for_backward(ids)
        ctx.cfg = (dtype, vocab, dim, scale)
        return y

    @_once
    def backward(ctx, grad_y):
        (ids,) = ctx.saved_tensors
        dtype, vocab, dim, scale = ctx.cfg
        lib, dev = _lib.lib(), ids.device
        gy = grad_y.contiguous()
        st = _raw_stream(dev.index)
        grad = torch.empty(vocab, dim, dtype=gy.dtype, device=dev)
        n = ids.numel()
        need = _embedding_ws(n, vocab, dim)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.check(lib.gatmi_embedding_bwd(dtype, n, vocab, dim, scale, ids.data_ptr(), gy.data_ptr(),
                                           grad.data_ptr(), ws.data_ptr(), need, st), "gatmi_embedding_bwd")
        return None, grad, None, None


def embedding(ids: Tensor, table: Tensor, scale: float = 1.0) -> Tensor:
    """scale * table[ids]: ids int64 of any shape, table [entries, dim] -> [..., dim].  An id outside the table
    (-1 for "none") gives a zero row and takes no gradient.  The table's gradient is dense, summed over the
    ids sorted by value in their own order (no float atomics)."""
    dtype = _check("embedding", table)
    if not ids.is_cuda or ids.device != table.device:
        raise ValueError(f"embedding: ids on {ids.device}, table on {table.device}")
    if ids.dtype != torch.int64:
        raise TypeError(f"embedding: ids must be int64, got {ids.dtype}")
    if table.dim() != 2 or table.size(1) < 1:
        raise ValueError(f"embedding: table must be [entries, dim], got {tuple(table.shape)}")
    return _apply(_EmbeddingFn, table, torch.is_grad_enabled() and table.requires_grad, ids, table, float(scale), dtype)


# ---- dropout ---------------------------------------------------------------------------------
class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, dtype):
        lib, dev = _lib.lib(), x.device
        x = x.contiguous()
        residual = None if residual is None else residual.contiguous()
        cols = x.size(-1)
        rows = x.numel() // cols if cols else 0
        st = _raw_stream(dev.index)
        y = torch.empty_like(x)
        used = None
        if isinstance(seed, Tensor):
            used = torch.empty(1, dtype=torch.int64, device=dev)
        _lib.check(lib.gatmi_dropout(dtype, rows, max(cols, 1), p, 0 if used is not None else seed,
                                     seed.data_ptr() if used is not None else None, _ptr(used), x.data_ptr(),
                                     _ptr(residual), y.data_ptr(), st), "gatmi_dropout")
        ctx.save_for_backward(used)
        ctx.cfg = (p, seed if used is None else 0, dtype, residual is not None)
        return y

    @_once
    def backward(ctx, grad_y):
        (used,) = ctx.saved_tensors
        p, seed, dtype, _ = ctx.cfg
        gx = None
        if ctx.needs_input_grad[0]:
            lib, dev = _lib.lib(), grad_y.device
            gy = grad_y.contiguous()
            cols = gy.size(-1)
            st = _raw_stream(dev.index)
            gx = torch.empty_like(gy)
            _lib.check(lib.gatmi_dropout(dtype, gy.numel() // cols if cols else 0, max(cols, 1), p, seed, _ptr(used),
                                         None, gy.data_ptr(), None, gx.data_ptr(), st), "gatmi_dropout")
        return gx, grad_y if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: Tensor, p: float, training: bool = True, seed=None, residual: Optional[Tensor] = None) -> Tensor:
    """x / (1 - p) where a counter-based draw of (seed, row, column) keeps it, else 0; plus `residual`.  No
    mask is stored: the backward draws it again.  Rows are x flattened to [rows, x.size(-1)], and the mask is
    `gat_amd.glue.dropout_mask(rows, cols, p, seed)`.  `seed`: an int; None draws one from torch's generator;
    a one-element int64 CUDA tensor is advanced in place on the device and read there, so the call can be
    captured in a HIP graph and every replay draws a new mask."""
    dtype = _check("dropout", x, residual)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout: p must be in [0, 1), got {p}")
    if x.dim() < 1:
        raise ValueError("dropout: x must have at least one axis")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"dropout: residual must be {tuple(x.shape)}, got {tuple(residual.shape)}")
    if isinstance(seed, Tensor) and (seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device):
        raise ValueError(f"dropout: a seed tensor is one int64 on {x.device}, got {seed.dtype} "
                         f"{tuple(seed.shape)} on {seed.device}")
    if not training or p == 0.0:
        return x if residual is None else x + residual
    if isinstance(seed, Tensor):
        seed.add_(SEED_STEP)
    elif seed is None:
        seed = int(torch.empty((), dtype=torch.int64).random_().item())
    else:
        seed = int(seed) & 0xFFFFFFFFFFFFFFFF
    needs = torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad))
    return _apply(_DropoutFn, x, needs, x, residual, float(p), seed, dtype)
