"""The dense operators on the GPU where single roundings and saturated units show: every result here is ONE term (or
one function value), so that no averaging over a sum hides what was lost on the way.  Bounds are relative
(tests/dense_tails.py)."""
import pytest
import torch

import dense_tails as T

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def uniform(shape, dtype, lo, hi, seed, scale=1.0):
    """values in [lo, hi), and an upstream gradient"""
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(*shape, generator=g) * (hi - lo) + lo).to(dtype), (torch.randn(*shape, generator=g) * scale).to(dtype)


def pieces(dz, dtype):
    """dz of a 16-bit tensor enters the products as two numbers of its type, the second what the first one's rounding
    left: half a step of a half step, and f16's own smallest step"""
    return T.u(dtype) ** 2 * dz.abs() + (2.0 ** -25 if dtype == F16 else 0.0)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["elu", "silu", "gelu"])
@pytest.mark.parametrize("m,n", [(3, 64), (40, 64), (333, 72), (2500, 40), (40, 5), (700, 1200), (66000, 128)])
def test_linear_dx_is_rounded_once(cuda, dtype, act, m, n):
    """W = 1.7 on the diagonal: dx is one product, dy act'(z) W, of which only the result may be rounded to the type"""
    import gat_amd
    x, dy = uniform((m, n), dtype, -0.3, 1.2, m + n)
    w = (torch.eye(n) * 1.7).to(dtype)
    z = x.double() * float(w[0, 0])              # exact in f32 too: 8 by 8 or 11 by 11 bits
    _, d, _, size = T.act(z, act)
    dz = dy.double() * d
    edz = dy.double().abs() * (T.own(z, dtype) * size + T.coding(d, dtype, act)) * 1.01 + pieces(dz, dtype) + 4 * T.U * dz.abs()
    dx = dz * float(w[0, 0])
    xd = x.to(cuda).requires_grad_(True)
    y = gat_amd.linear_act(xd, w.to(cuda), act=act)
    (gx,) = torch.autograd.grad(y, xd, dy.to(cuda))
    T.within(gx, dx, edz * 1.75 + T.u(dtype) * dx.abs(), "dx")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["elu", "silu", "gelu"])
@pytest.mark.parametrize("m,k,n", [(64, 40, 64), (333, 72, 30), (2500, 300, 140), (50, 5, 40), (50, 40, 3)])
def test_linear_dw_is_rounded_once(cuda, dtype, act, m, k, n):
    """W = 0, so z is the bias; one row of x for each of its columns: dW is one product, dy act'(z) x"""
    import gat_amd
    b, _ = uniform((n,), dtype, -0.3, 1.9, n)
    v, dy = uniform((k, n), dtype, 0.6, 1.9, k)
    dy = torch.cat([dy, torch.ones(m, n).to(dtype)])[:m]
    x = torch.zeros(m, k, dtype=dtype)
    x[torch.arange(min(k, m)), torch.arange(min(k, m))] = v[: min(k, m), 0]
    z = b.double().expand(m, n)
    _, d, _, size = T.act(z, act)
    dz = dy.double() * d
    edz = dy.double().abs() * (T.own(z, dtype) * size + T.coding(d, dtype, act)) * 1.01 + pieces(dz, dtype) + 4 * T.U * dz.abs()
    wd = torch.zeros(n, k, dtype=dtype, device=cuda, requires_grad=True)
    y = gat_amd.linear_act(x.to(cuda), wd, b.to(cuda), act)
    (gw,) = torch.autograd.grad(y, wd, dy.to(cuda))
    X = x.double()
    dw = dz.t() @ X
    T.within(gw, dw, edz.t() @ X + T.u(dtype) * dw.abs(), "dw")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,k,n", [(40, 50, 70), (2500, 140, 90), (64, 40, 1200), (30, 5, 6), (66000, 64, 72), (33000, 256, 64)])
def test_linear_gradients_not_finite(cuda, dtype, m, k, n):
    """an infinity or NaN in x, W or dy gives what the formula gives, where dz is two numbers as elsewhere: the same
    infinities and NaN, and every other value as if they were not there"""
    import gat_amd
    g = torch.Generator().manual_seed(m + n)
    base = [torch.randn(m, k, generator=g).to(dtype), (torch.randn(n, k, generator=g) / k ** 0.5).to(dtype),
            torch.randn(m, n, generator=g).to(dtype)]
    inf = float("inf")
    for which, at, value in ((0, (3, 4), inf), (1, (5, 2), -inf), (2, (9, 1), inf), (2, (7, 0), float("nan")),
                             (0, (m - 1, k - 1), float("nan")), (1, (n - 1, k - 1), inf)):
        x, w, dy = (t.clone() for t in base)
        (x, w, dy)[which][at] = value
        xd, wd = x.to(cuda).requires_grad_(True), w.to(cuda).requires_grad_(True)
        y = gat_amd.linear_act(xd, wd, act="elu")
        got = torch.autograd.grad(y, (xd, wd), dy.to(cuda))
        X, W, D = x.to(cuda).double(), w.to(cuda).double(), dy.to(cuda).double()
        dz = D * T.act(X @ W.t(), "elu")[1]
        for have, want in zip(got, (dz @ W, dz.t() @ X)):
            have = have.double()
            assert torch.equal(torch.isnan(have), torch.isnan(want)), (which, at)
            assert torch.equal(have[torch.isinf(want)], want[torch.isinf(want)]), (which, at)
            fine = torch.isfinite(want)
            # (no more than: nothing else was touched)
            if bool(fine.any()):
                assert float((have - want)[fine].abs().max()) <= 2e-2 * float(want[fine].abs().max()), (which, at)


def test_linear_gradient_past_the_range_of_f16(cuda):
    """dz = dy act'(z) may be larger than any f16 where dx is not: GELU's slope goes up to 1.129"""
    import gat_amd
    for m in (40, 3):
        x = torch.full((m, 64), 1.5, dtype=F16)
        w = torch.eye(64, dtype=F16) * 0.25
        dy = torch.full((m, 64), 65504.0, dtype=F16)
        dy[1] *= -1
        b = torch.full((64,), 1.0, dtype=F16)
        xd = x.to(cuda).requires_grad_(True)
        y = gat_amd.linear_act(xd, w.to(cuda), b.to(cuda), act="gelu")
        (gx,) = torch.autograd.grad(y, xd, dy.to(cuda))
        dx = dy.double() * T.act(x.double() * 0.25 + 1.0, "gelu")[1] * 0.25
        assert float(dx.abs().min()) * 4 > 65520
        T.within(gx, dx, dx.abs() * (T.u(F16) + 2.0 ** -11), "dx")


def gradient_of_saturated_units(cuda, dtype, act, m, n, lo=-12.0, hi=-4.0):
    """W = 1: z = x and dx = dy act'(x), to the type's precision whether z is -4 or -12.  (f16: dy of a size at which
    these gradients are normal numbers.)"""
    import gat_amd
    x, dy = uniform((m, n), dtype, lo, hi, m + n, 1024.0 if dtype == F16 else 1.0)
    z = x.double()
    _, d, _, size = T.act(z, act)
    dx = dy.double() * d
    edz = dy.double().abs() * (T.own(z, dtype) * size + T.coding(d, dtype, act)) * 1.01 + 4 * T.U * dx.abs()
    # f32: three bf16 pieces of dz, of which the last is rounded to a multiple of bf16's smallest number, 2^-133, at
    # the coarsest: half of that, times W = 1
    edz = edz + (2.0 ** -134 if dtype == F32 else pieces(dx, dtype))
    xd = x.to(cuda).requires_grad_(True)
    y = gat_amd.linear_act(xd, torch.eye(n, dtype=dtype, device=cuda), act=act)
    (gx,) = torch.autograd.grad(y, xd, dy.to(cuda))
    T.within(gx, dx, edz + T.u(dtype) * dx.abs(), "dx")


SIZES = [(3, 64), (40, 64), (333, 72), (2500, 40), (40, 5), (66000, 128)]


@pytest.mark.parametrize("m,n", SIZES)
def test_elu_slope_of_saturated_units_f32(cuda, m, n):
    gradient_of_saturated_units(cuda, F32, "elu", m, n)
    gradient_of_saturated_units(cuda, F32, "elu", m, n, -80.0, -10.0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_elu_slope_of_saturated_units_group_norm(cuda, dtype):
    """one sample, weight 1 and bias far below 0: the bias's gradient is dy act'(z), one term"""
    import gat_amd
    for shape in ((1, 64), (1, 1, 64)):
        b, dy = uniform((64,), dtype, -12.0, -6.0, 3, 1024.0 if dtype == F16 else 1.0)
        bd = b.to(cuda).requires_grad_(True)
        w = torch.zeros(64, dtype=dtype, device=cuda)          # z = bias, exactly
        x = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(dtype).to(cuda)
        y = gat_amd.group_norm_act(x, 4, w, bd, act="elu")
        (gb,) = torch.autograd.grad(y, bd, dy.to(cuda).view(shape))
        _, d, _, size = T.act(b.double(), "elu")
        want = dy.double() * d
        T.within(gb, want, dy.double().abs() * T.own(b.double(), dtype) * size + (T.u(dtype) + 4 * T.U) * want.abs(), "db")


@pytest.mark.parametrize("dtype,lo", [(F32, -12.0), (BF16, -12.0), (F16, -5.5)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,n", SIZES)
def test_values_of_saturated_units(cuda, dtype, lo, act, m, n):
    """W = 1: y = act(x) where it is small itself"""
    import gat_amd
    x, _ = uniform((m, n), dtype, lo, -0.5, m + n)
    a, _, size, _ = T.act(x.double(), act)
    y = gat_amd.linear_act(x.to(cuda), torch.eye(n, dtype=dtype, device=cuda), act=act)
    T.within(y, a, T.own(x.double(), dtype) * size + T.u(dtype) * a.abs(), "y")


@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_slope_of_saturated_units_f32(cuda, act, m, n):
    gradient_of_saturated_units(cuda, F32, act, m, n)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["elu", "silu", "gelu"])
@pytest.mark.parametrize("m,n", SIZES)
def test_slope_of_saturated_units_16_bit(cuda, dtype, act, m, n):
    gradient_of_saturated_units(cuda, dtype, act, m, n)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["relu", "elu"])
def test_slope_of_special_values(cuda, dtype, act):
    """0 and 1 are exact slopes, and NaN is one of its own row only"""
    import gat_amd
    x = torch.tensor([3.0, 1.0, 200.0, -200.0]).to(dtype).repeat(20, 16)
    x[:, 7] = 0.0
    dy = torch.full_like(x, 1.25)
    x[11, 5] = float("nan")
    xd = x.to(cuda).requires_grad_(True)
    y = gat_amd.linear_act(xd, torch.eye(64, dtype=dtype, device=cuda), act=act)
    (gx,) = torch.autograd.grad(y, xd, dy.to(cuda))
    want = torch.where(x > 0, 1.25, 0.0).to(dtype)
    want[:, 7] = 0.0 if act == "relu" else 1.25
    got = gx.cpu()
    rows = torch.arange(20) != 11
    assert torch.equal(got[rows], want[rows])
    assert bool(torch.isnan(got[11]).all())      # every column of that row's x W^T has NaN among its terms


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("act", ["elu", "silu", "gelu"])
def test_activations_at_the_ends_of_their_range(cuda, dtype, act):
    """W = 0 and z the bias: far beyond any exponential's range values and slopes are those of the limit, infinities
    and NaN as z * factor gives them"""
    import gat_amd
    inf, nan, top = float("inf"), float("nan"), torch.finfo(dtype).max
    far = [top, -top, top / 3, -top / 3, 100.0, -100.0, 89.0, -89.0, 30.0, -30.0, 20.5, -20.5, 0.0, -0.0]
    b = torch.tensor(far + [inf, -inf, nan] + [1.0] * 7).to(dtype)
    for m in (1, 20):
        x, w = torch.zeros(m, 8, dtype=dtype, device=cuda), torch.zeros(24, 8, dtype=dtype, device=cuda)
        bd = b.to(cuda).requires_grad_(True)
        y = gat_amd.linear_act(x, w, bd, act)
        (db,) = torch.autograd.grad(y, bd, torch.tensor([1.0] + [0.0] * (m - 1), dtype=dtype, device=cuda)[:, None].expand(m, 24))
        n = len(far)
        z = b[:n].double()
        a, d, size, dsize = T.act(z, act)
        # v_exp_f32 gives 0 for a subnormal result: exp(-89) = 2.2e-39 and what it multiplies, |z| <= 89, are within that
        # many times the smallest normal f32 number of 0
        flushed = 90 * torch.finfo(F32).smallest_normal
        T.within(y[0, :n], a, T.own(z.clamp(-20, 20), dtype) * size + T.u(dtype) * a.abs() + flushed, "y")
        T.within(db[:n], d, T.own(z.clamp(-20, 20), dtype) * dsize + T.coding(d, dtype, act) + T.u(dtype) * d.abs() + flushed, "slope")
        y = y.detach().cpu()
        assert float(y[0, n]) == inf and bool(torch.isnan(y[0, n + 2])) and bool(torch.isnan(db[n + 2]))
        assert float(y[0, n + 1]) == -1.0 if act == "elu" else bool(torch.isnan(y[0, n + 1]))
        assert bool(torch.isfinite(y[0, n + 3:]).all())


@pytest.mark.parametrize("act", ["gelu", "elu"])
def test_linear_gradients_not_finite_cost_no_plain_sums(cuda, act):
    """an infinity in x or W sends no element through a sum of its own: the step stays within a few times an ordinary one
    (it was three hundred times), and what does not meet the infinity keeps the ordinary precision"""
    import gat_amd
    m = 400000
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(m, 256, generator=g).to(BF16).to(cuda), (torch.randn(256, 256, generator=g) / 16).to(BF16).to(cuda)
    dy = torch.randn(m, 256, generator=g).to(BF16).to(cuda)

    def step(x, w):
        xd, wd = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = gat_amd.linear_act(xd, wd, act=act)
        first, last = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.autograd.grad(y, (xd, wd), dy, retain_graph=True)
        first.record()
        got = torch.autograd.grad(y, (xd, wd), dy)
        last.record()
        torch.cuda.synchronize()
        return first.elapsed_time(last), got

    ms, plain = step(x, w)
    for which, at in ((0, (77, 3)), (1, (3, 200))):
        xs = [x.clone(), w.clone()]
        xs[which][at] = float("inf")
        slow, got = step(*xs)
        assert slow < 20 * ms + 1.0, (slow, ms)
        dx, dw = got
        rows, cols = torch.arange(m, device=cuda) != 77, torch.arange(256, device=cuda)
        # z is infinite in row 77, or in column 3.  The slope there is 0 or 1 for ELU, and inf * 0, NaN, for GELU.
        if which == 0:
            assert torch.equal(dx[rows], plain[0][rows])
            assert not bool(torch.isfinite(dw[:, 3]).any())
            assert bool(torch.isfinite(dw[:, cols != 3]).all() if act == "elu" else torch.isnan(dw).all())
            assert bool(torch.isfinite(dx[77]).all() if act == "elu" else torch.isnan(dx[77]).all())
        else:
            assert torch.equal(dw[cols != 3], plain[1][cols != 3])
            if act == "elu":
                assert bool(torch.isfinite(dx[:, cols != 200]).all()) and not bool(torch.isfinite(dx[:, 200]).any())
            else:
                assert bool(torch.isnan(dx).all()) and bool(torch.isnan(dw[3]).all())
