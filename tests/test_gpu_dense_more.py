"""The dense operators on the GPU: gradients against differences, sizes past one launch, calls at the edge of
what their arguments allow."""
import pytest
import torch

import dense_diff as D
import dense_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def run(op, p, kw):
    import gat_amd
    if op == "linear":
        return gat_amd.linear_act(p[0], p[1], p[2], kw["act"], p[3])
    if op == "group_norm":
        return gat_amd.group_norm_act(p[0], kw["groups"], p[1], p[2], act=kw["act"])
    if op == "embedding":
        return gat_amd.embedding(kw["ids"].to(p[0].device), p[0], kw["scale"])
    return gat_amd.dropout(p[0], kw["p"], seed=kw["seed"], residual=p[1])


@pytest.mark.parametrize("which", range(len(D.CASES)))
def test_gradient_is_the_difference(cuda, which):
    op, kw, shapes = D.CASES[which]
    if op == "dropout":
        from gat_amd.glue import dropout_mask
        kw = dict(kw, keep=dropout_mask(*shapes[0], kw["p"], kw["seed"], cuda).cpu())
    p, hi, lo, c, v, t, want, bound = D.case(op, kw, shapes)
    leaves = [q.to(cuda).requires_grad_(True) for q in p]
    grads = torch.autograd.grad(run(op, leaves, kw), leaves, c.to(cuda).view(kw["out"]))
    along = sum(float((g.cpu().double() * d).sum()) for g, d in zip(grads, v))
    with torch.no_grad():
        yh, yl = (run(op, [q.to(cuda) for q in s], kw).cpu().double().view(c.shape) for s in (hi, lo))
    diff = float((c.double() * (yh - yl)).sum()) / (2 * t)
    assert abs(diff - along) <= bound, (diff, along, want, bound)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_more_samples_than_a_launch(cuda, dtype):
    import gat_amd
    g = torch.Generator().manual_seed(2)
    shape = (65535 + 300, 2, 12)
    x, dy = torch.randn(*shape, generator=g).to(dtype), torch.randn(*shape, generator=g).to(dtype)
    w, b = torch.randn(12, generator=g).to(dtype), torch.randn(12, generator=g).to(dtype)
    ref = R.GroupNorm(x, 3, w, b, "silu", dy, dtype)
    leaves = [q.to(cuda).requires_grad_(True) for q in (x, w, b)]
    y = gat_amd.group_norm_act(leaves[0], 3, leaves[1], leaves[2], act="silu")
    y.backward(dy.to(cuda))
    R.check(y, ref.y, "y")
    for q, r, name in zip(leaves, (ref.dx, ref.dw, ref.db), ("dx", "dw", "db")):
        R.check(q.grad, r, name)


def test_linear_more_tiles_than_a_launch(cuda):
    """one product a result: rounded once, as torch's own multiplication is"""
    import gat_amd
    rows = (1 << 29) + 65
    x = torch.randn(rows, 1, device=cuda, dtype=BF16)
    w = torch.tensor([[1.7]], device=cuda, dtype=BF16)
    xd = x.requires_grad_(True)
    y = gat_amd.linear_act(xd, w)
    (dx,) = torch.autograd.grad(y, xd, x.detach())
    with torch.no_grad():
        want = x * w[0]
        assert torch.equal(y, want) and torch.equal(dx, want)


def test_linear_refuses_what_it_does_not_cover(cuda):
    import gat_amd
    x, w = torch.zeros(2, 65537, device=cuda), torch.zeros(1, 65537, device=cuda)
    with pytest.raises(ValueError, match="65536"):
        gat_amd.linear_act(x, w)
    with pytest.raises(ValueError, match="65536"):
        gat_amd.linear_act(w[:, :1], w.t())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_dropout_off_with_residual(cuda, dtype):
    import gat_amd
    x, r = (torch.randn(33, 7, device=cuda).to(dtype).requires_grad_(True) for _ in range(2))
    seed = torch.tensor([5], device=cuda)
    for y in (gat_amd.dropout(x, 0.5, training=False, seed=seed, residual=r), gat_amd.dropout(x, 0.0, residual=r)):
        assert torch.equal(y, x + r)
        up = torch.randn_like(y)
        assert all(torch.equal(g, up) for g in torch.autograd.grad(y, (x, r), up))
    assert int(seed) == 5        # nothing drawn, not moved on


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,k,n", [(17, 1024, 64), (5, 700, 30), (16, 2050, 9), (64, 515, 1025), (300, 1001, 3),
                                   (200, 40, 1500), (1, 33, 3001), (3000, 777, 7)])
def test_linear_split_contraction(cuda, dtype, m, k, n):
    """few tiles and a long contraction (of the forward's, the second half of the gradient's)"""
    from test_gpu_dense import linear_case
    linear_case(cuda, dtype, m, k, n, "silu", True, True)
    linear_case(cuda, dtype, m, k, n, "none", False, False)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,k,n", [(33000, 256, 192), (32769, 192, 200), (66001, 64, 72)])
def test_linear_whole_steps(cuda, dtype, m, k, n):
    """contractions of whole steps over many large tiles, the last of them partial"""
    from test_gpu_dense import linear_case
    linear_case(cuda, dtype, m, k, n, "elu", True, True)


def test_linear_split_contraction_not_finite(cuda):
    """infinities and NaN in f32 as plain f32 sums have them, forward and backward, when the contraction is split"""
    import gat_amd
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn(40, 1024, generator=g), torch.randn(70, 1024, generator=g)
    x[3, 5], x[7, 900], w[11, 2], x[9, 9], w[20, 9] = float("inf"), float("nan"), float("-inf"), 3.0e38, 0.999
    x[12, :2], w[12, :2] = torch.tensor([3.0e38, -3.0e38]), 1.0
    xd, wd = x.to(cuda).requires_grad_(True), w.to(cuda).requires_grad_(True)
    y = gat_amd.linear_act(xd, wd)
    want = x.double() @ w.double().t()
    # where the terms' sizes sum up to a float, every partial sum is one, whatever the order; elsewhere (3e38 * 2)
    # plain f32 sums overflow too
    same = x.double().abs() @ w.double().abs().t() < 3.4e38
    got = y.detach().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)].double(), want[torch.isinf(want)])
    assert bool(torch.isfinite(got[same]).all())
    dy = torch.randn(40, 70, generator=g)
    dy[2, 8] = float("inf")
    gx, gw = torch.autograd.grad(y, (xd, wd), dy.to(cuda))
    for got, want in ((gx, dy.double() @ w.double()), (gw, dy.double().t() @ x.double())):
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        inf = torch.isinf(want)
        assert torch.equal(got.cpu().double()[inf], want[inf])


def test_linear_gradient_of_the_bias_alone(cuda):
    """weights frozen, many splits of the rows, more columns of x than one tile"""
    import gat_amd
    g = torch.Generator().manual_seed(9)
    x, w, b = torch.randn(9000, 300, generator=g), torch.randn(140, 300, generator=g) / 17, torch.randn(140, generator=g)
    dy = torch.randn(9000, 140, generator=g)
    ref = R.Linear(x, w, b, None, "gelu", dy, F32)
    bd = b.to(cuda).requires_grad_(True)
    (db,) = torch.autograd.grad(gat_amd.linear_act(x.to(cuda), w.to(cuda), bd, "gelu"), bd, dy.to(cuda))
    R.check(db, ref.db, "db")
