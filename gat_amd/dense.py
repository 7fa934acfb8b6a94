"""The dense operators around a GAT layer: a linear layer with its epilogue, group normalisation with an
activation, embedding lookup, dropout (gat_amd/csrc/linear.hip, group_norm.hip, embedding.hip,
dropout.hip).

The reference's network has stock modules there or nothing; these are what a block around `GATConv` is
made of when it grows a skip connection, a per-node normalisation (no statistics over the batch, so none to
combine over the ranks of a partitioned graph) or categorical node features.  Each takes float32, bfloat16
or float16 tensors (all of one type, any strides), computes in float32 or wider and rounds every result
once; the same inputs give the same bits.  GPU only.  Gradients are those of one backward pass: a second
derivative, a forward-mode tangent and a recording by torch.jit.trace are refused.

Checks, outputs, workspaces and the autograd nodes are native (gat_amd/csrc/torch_dense.cpp, built with the
library as gat_amd/_torch_dense.so) over the same C ABI any other host uses (include/gat_mi355.h).
Arguments of a wrong shape or device raise ValueError, of a wrong type TypeError, everything else
RuntimeError.
"""
from __future__ import annotations

import importlib.util
import os
from typing import Optional

import torch
from torch import Tensor

from . import _lib
from .glue import SEED_STEP

ACTIVATIONS = {"none": 0, "relu": 1, "elu": 2, "silu": 3, "gelu": 4}
GROUP_NORM_MAX_CHANNELS = 8192      # GATMI_GROUP_NORM_MAX_CHANNELS

_native = None


def _load():
    """The native module, bound to the library file gat_amd._lib names"""
    global _native
    if _native is None:
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_torch_dense.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; "
                               "g.build()'` (or `make -C gat_amd/csrc`).  gat_amd has no fallback path.")
        spec = importlib.util.spec_from_file_location("gat_amd._torch_dense", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _lib.lib()                    # checks that the library is there and whole
        module.load(_lib.LIB_PATH)
        _native = module
    return _native


def _act(name: str, act: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"{name}: act must be one of {', '.join(ACTIVATIONS)}, got {act!r}")
    return code


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: str = "none",
               residual: Optional[Tensor] = None) -> Tensor:
    """act(x @ weight.T + bias) + residual in one kernel: x [..., in], weight [out, in], bias [out],
    residual [..., out]; act one of ACTIVATIONS ("gelu" is the exact form).  With `residual=conv(x)` it is
    the skip connection beside a GAT layer.  float32 operands smaller than 2^-110 (7.7e-34) count as the nearest
    multiple of 2^-133."""
    return (_native or _load()).linear_act(x, weight, bias, _act("linear_act", act), residual)


def group_norm_act(x: Tensor, groups: int, weight: Tensor, bias: Tensor, eps: float = 1e-5,
                   act: str = "none") -> Tensor:
    """act(group_norm(x)) with channels last: x [N, C] or [N, ..., C], weight and bias [C], C = groups *
    width.  Mean and variance are those of one sample's group: its `width` channels at all positions between
    the first and the last axis.  For x [nodes, heads * channels] and groups = heads every node's heads are
    normalised one by one; for x [graphs, nodes, C] the statistics are a graph's."""
    return (_native or _load()).group_norm_act(x, int(groups), weight, bias, float(eps), _act("group_norm_act", act))


def stock_group_norm(x: Tensor, norm: torch.nn.GroupNorm) -> Tensor:
    """norm(x) for x [N, C] in elementary torch operations, any device and type: what the networks' stock paths take.
    Not F.group_norm: its weight and bias gradients are wrong on this platform for rows without further axes
    (more than 128 of them)."""
    v = x.reshape(x.size(0), norm.num_groups, x.size(1) // norm.num_groups)
    var, mean = torch.var_mean(v, dim=2, unbiased=False, keepdim=True)
    v = ((v - mean) * torch.rsqrt(var + norm.eps)).view_as(x)
    return v * norm.weight + norm.bias


def embedding(ids: Tensor, table: Tensor, scale: float = 1.0) -> Tensor:
    """scale * table[ids]: ids int64 of any shape, table [entries, dim] -> [..., dim].  An id outside the table
    (-1 for "none") gives a zero row and takes no gradient.  The table's gradient is dense, summed over the
    ids sorted by value in their own order (no float atomics)."""
    return (_native or _load()).embedding(ids, table, float(scale))


def dropout(x: Tensor, p: float, training: bool = True, seed=None, residual: Optional[Tensor] = None) -> Tensor:
    """x / (1 - p) where a counter-based draw of (seed, row, column) keeps it, else 0; plus `residual`; 0 <= p < 1.  No
    mask is stored: the backward draws it again.  Rows are x flattened to [rows, x.size(-1)], and the mask is
    `gat_amd.glue.dropout_mask(rows, cols, p, seed)`.  `seed`: an int; None draws one from torch's generator;
    a one-element int64 CUDA tensor is advanced in place on the device and read there, so the call can be
    captured in a HIP graph and every replay draws a new mask."""
    on_device = None
    if isinstance(seed, Tensor):
        on_device, seed = seed, 0
    elif seed is None:
        seed = int(torch.empty((), dtype=torch.int64).random_().item()) if training and p > 0.0 else 0
    else:
        seed = int(seed) & 0xFFFFFFFFFFFFFFFF
    return (_native or _load()).dropout(x, float(p), bool(training), seed, on_device, SEED_STEP, residual)
