"""linear_act in f32 at both ends of its range, on the matrix cores (more than sixteen rows; the weights cut on the way
below 2048 rows, ahead of the product from there on), forward and backward."""
import pytest
import torch

import dense_ref as R

pytestmark = pytest.mark.gpu
F32 = torch.float32
MAX = torch.finfo(F32).max
SIZES = [(17, 64, 24), (40, 64, 70), (2500, 64, 70), (40, 1024, 30), (66000, 64, 128)]


def wider(ref, x, w):
    """ref for C = x w^T, its bound with what the pieces of small operands leave: three bf16 pieces hold an f32 number
    exactly from 2^-110 on, whose last bit is 2^-133, bf16's smallest number; a smaller one to half of that"""
    value, bound = ref
    step = 2.0 ** -134
    return value, bound + 1.01 * step * (x.double().abs().sum(1)[:, None] + w.double().abs().sum(1)[None])


@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_next_to_the_largest_float(cuda, m, k, n):
    """the largest floats' first piece rounds up to infinity"""
    import gat_amd
    g = torch.Generator().manual_seed(m + k + n)
    x, w = torch.randn(m, k, generator=g), (torch.rand(n, k, generator=g) - 0.5)
    x[3, 0], x[7, 5], x[m - 1, k - 1] = MAX, -0.999 * MAX, MAX
    small = torch.rand(m, n, generator=g) * 0.5 / m
    ref = R.Linear(x, w, None, None, "none", small, F32)
    xd, wd = x.to(cuda).requires_grad_(True), w.to(cuda).requires_grad_(True)
    y = gat_amd.linear_act(xd, wd)
    R.check(y, ref.y, "y")
    gx, gw = torch.autograd.grad(y, (xd, wd), small.to(cuda))
    R.check(gx, ref.dx, "dx")
    R.check(gw, ref.dw, "dw")
    dy = small.clone()
    dy[3, 1], dy[m - 1, n - 1] = MAX, -MAX
    ref = R.Linear(torch.zeros(m, k), w, None, None, "none", dy, F32)
    xd = torch.zeros(m, k, device=cuda, requires_grad=True)
    (gx,) = torch.autograd.grad(gat_amd.linear_act(xd, w.to(cuda)), xd, dy.to(cuda))
    R.check(gx, ref.dx, "dx of the largest")
    w2 = w.clone()
    w2[1, 2], w2[n - 1, 0] = MAX, -MAX
    x2 = torch.rand(m, k, generator=g) * 0.5 / k
    R.check(gat_amd.linear_act(x2.to(cuda), w2.to(cuda)), R.Linear(x2, w2, None, None, "none", None, F32).y, "y of large weights")


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("e", [100, 109, 112, 116, 120, 126, 132, 140])
def test_linear_of_small_operands(cuda, m, k, n, e):
    """x, W or dy of size 2^-e against a factor that brings the result back to ordinary numbers"""
    import gat_amd
    g = torch.Generator().manual_seed(e)
    tiny = lambda *s: (torch.randn(*s, generator=g).double() * 2.0 ** -e).float()
    big = lambda *s: torch.randn(*s, generator=g) * 2.0 ** 100
    for x, w, dy in ((tiny(m, k), big(n, k), big(m, n)), (big(m, k), tiny(n, k), tiny(m, n))):
        xd, wd = x.to(cuda).requires_grad_(True), w.to(cuda).requires_grad_(True)
        y = gat_amd.linear_act(xd, wd)
        ref = R.Linear(x, w, None, None, "none", None, F32)
        R.check(y, wider(ref.y, x, w), "y")
        # (an ordinary dy where both factors would be small or large)
        for a, c, which in ((dy, w, 0), (dy, x, 1)):
            if (float(a.abs().max()) < 1.0) == (float(c.abs().max()) < 1.0):
                a = torch.randn(a.shape, generator=g)
            ref = R.Linear(x, w, None, None, "none", a, F32)
            (got,) = torch.autograd.grad(y, (xd, wd)[which], a.to(cuda), retain_graph=True)
            if which == 0:
                R.check(got, wider(ref.dx, a, w.t()), "dx")
            else:
                R.check(got, wider(ref.dw, a.t(), x.t()), "dw")
