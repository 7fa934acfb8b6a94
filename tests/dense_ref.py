"""The dense operators (gat_amd/dense.py) restated in 64 bits on the CPU, with error bounds element by
element: what f32 arithmetic, the 16-bit codings named below and one rounding of the result can be off by.
Used by the tests only.

u(T) = finfo(T).eps / 2 is half a step of the result's type; U = 2^-24 that of f32.  A sum of n terms kept
in f32 is off by at most n U times the sum of its terms' sizes, whatever their order."""
import math

import torch

U = 2.0 ** -24
ACTS = ("none", "relu", "elu", "silu", "gelu")


def u(dtype):
    return torch.finfo(dtype).eps / 2


def act(z, name):
    """(value, first derivative) in float64"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "elu":
        e = torch.expm1(z.clamp(max=0))
        return torch.where(z > 0, z, e), torch.where(z > 0, torch.ones_like(z), e + 1)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    p = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
    return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def act_error(z, ez, dtype):
    """(value error, slope error) of an activation of z known to `ez`: first derivatives are below 1.13,
    second ones below 1; the functions themselves are good to a few f32 steps of 1 + |z| (f32) or to 2^-20
    of it (16 bits: v_exp forms, and 1.5e-7 absolute on erf)."""
    own = (8 * U if dtype == torch.float32 else 2.0 ** -20) * (1 + z.abs())
    return 1.13 * ez + own, ez + own


class Linear:
    """y = act(x W^T + b) + res and its gradients for dy, with bounds (each a pair value, bound)."""

    def __init__(self, x, w, b, res, name, dy, dtype):
        X, W = x.double(), w.double()
        k, n, m = X.size(1), W.size(0), X.size(0)
        z, s = X @ W.t(), X.abs() @ W.abs().t()
        if b is not None:
            z, s = z + b.double(), s + b.double().abs()
        ez = (k + 8) * U * s                # the products' own rounding and the f32 pieces' are within the 8
        a, d = act(z, name)
        ea, ed = (ez, 0 * ez) if name == "none" else act_error(z, ez, dtype)
        if name == "relu":                  # exact on either side of 0; z closer to it than its error can be on the other
            ea, ed = ez, (z.abs() <= ez).double()
        y = a if res is None else a + res.double()
        self.y = (y, ea + U * (a.abs() + y.abs()) + u(dtype) * y.abs())
        if dy is None:
            return
        dy = dy.double()
        dz = dy * d
        # the slope is kept in steps of 2^-15 for 16-bit tensors (half a step: 2^-16), dz is rounded to the type
        coding = 0.0 if dtype == torch.float32 or name in ("none", "relu") else 2.0 ** -16
        ebefore = dy.abs() * (ed + coding) + 2 * U * dz.abs()
        edz = ebefore + (0.0 if name == "none" else u(dtype) * (dz.abs() + ebefore))
        size = dz.abs() + edz
        dx, dw, db = dz @ W, dz.t() @ X, dz.sum(0)
        self.dx = (dx, edz @ W.abs() + (n + 8) * U * (size @ W.abs()) + u(dtype) * dx.abs())
        self.dw = (dw, edz.t() @ X.abs() + (m + 8) * U * (size.t() @ X.abs()) + u(dtype) * dw.abs())
        self.db = (db, ebefore.sum(0) + (m + 8) * U * size.sum(0) + u(dtype) * db.abs())


class GroupNorm:
    """x [batch, length, groups, width] viewed so; `depth` bounds how many f32 additions one value passes
    through in a group's sums (a lane's own values, then the tree), `pdepth` in the parameter sums."""

    def __init__(self, x, groups, w, b, name, dy, dtype, eps=1e-5, depth=256, pdepth=1024):
        n, c = x.size(0), x.size(-1)
        shape = (n, -1, groups, c // groups)
        X = x.double().reshape(shape)
        W, B = w.double().view(groups, -1), b.double().view(groups, -1)
        mean = X.mean((1, 3), keepdim=True)
        var = (X - mean).pow(2).mean((1, 3), keepdim=True)
        rstd = (var + eps).rsqrt()
        xh = (X - mean) * rstd
        # the mean is off by depth U mean|x|, a shifted value by U of itself besides, the variance by
        # (2 depth U) of itself and the square of the mean's error
        emean = depth * U * X.abs().mean((1, 3), keepdim=True)
        rel = depth * U + emean * emean / (var + eps)
        exh = rstd * (emean + 2 * U * X.abs()) + rel * xh.abs()
        z = xh * W + B
        ez = W.abs() * exh + 2 * U * (z.abs() + B.abs())
        a, d = act(z, name)
        ea, ed = (ez, 0 * ez) if name == "none" else act_error(z, ez, dtype)
        if name == "relu":
            ea, ed = ez, (z.abs() <= ez).double()
        self.y = (a.reshape(x.shape), (ea + U * a.abs() + u(dtype) * a.abs()).reshape(x.shape))
        if dy is None:
            return
        dy = dy.double().reshape(shape)
        du = dy * d
        edu = dy.abs() * ed + 2 * U * du.abs()
        g, eg = du * W, edu * W.abs() + U * (du * W).abs()
        m1, m2 = g.mean((1, 3), keepdim=True), (g * xh).mean((1, 3), keepdim=True)
        em1 = eg.mean((1, 3), keepdim=True) + depth * U * g.abs().mean((1, 3), keepdim=True)
        em2 = (eg * xh.abs() + g.abs() * exh).mean((1, 3), keepdim=True) + depth * U * (g * xh).abs().mean((1, 3), keepdim=True)
        dx = rstd * (g - m1 - xh * m2)
        size = g.abs() + m1.abs() + (xh * m2).abs()
        edx = rstd * (eg + em1 + xh.abs() * em2 + exh * m2.abs() + 4 * U * size) + rel * rstd * size
        self.dx = (dx.reshape(x.shape), (edx + u(dtype) * dx.abs()).reshape(x.shape))
        dw, db = (du * xh).sum((0, 1)), du.sum((0, 1))
        edw = (edu * xh.abs() + du.abs() * exh).sum((0, 1)) + pdepth * U * (du * xh).abs().sum((0, 1))
        edb = edu.sum((0, 1)) + pdepth * U * du.abs().sum((0, 1))
        self.dw = (dw.reshape(c), (edw + u(dtype) * dw.abs()).reshape(c))
        self.db = (db.reshape(c), (edb + u(dtype) * db.abs()).reshape(c))


def embedding(ids, table, scale, dy, dtype):
    """(y, bound), (grad, bound)"""
    ids, T = ids.reshape(-1), table.double()
    here = (ids >= 0) & (ids < T.size(0))
    y = torch.zeros(ids.numel(), T.size(1), dtype=torch.float64)
    y[here] = T[ids[here]] * scale
    out = [(y, (0.0 if scale == 1.0 else 2 * U + u(dtype)) * y.abs())]
    if dy is not None:
        D = dy.double().reshape(ids.numel(), -1)[here]
        g, s, n = torch.zeros_like(T), torch.zeros_like(T), torch.zeros(T.size(0), 1, dtype=torch.float64)
        g.index_add_(0, ids[here], D * scale)
        s.index_add_(0, ids[here], D.abs() * abs(scale))
        n.index_add_(0, ids[here], torch.ones(D.size(0), 1, dtype=torch.float64))
        out.append((g, (n + 2) * U * s + u(dtype) * g.abs()))
    return out


def check(got, want, name):
    """every element within its bound (and the tiniest subnormal step of its type)"""
    value, bound = want
    got = got.detach().cpu()
    tiny = torch.finfo(got.dtype).tiny
    assert tuple(got.shape) == tuple(value.shape), f"{name}: {tuple(got.shape)} for {tuple(value.shape)}"
    off = (got.double() - value).abs()
    bad = ~(off <= bound + tiny)
    if bool(bad.any()):
        at = int(torch.argmax((off / (bound + tiny)).reshape(-1).nan_to_num(nan=float("inf"))))
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside; worst at {at}: got "
                             f"{float(got.reshape(-1)[at])!r}, want {float(value.reshape(-1)[at])!r} within "
                             f"{float(bound.reshape(-1)[at]):.3g}")
