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


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_axis_and_empty_axes(cuda, dtype):
    import gat_amd
    g = torch.Generator().manual_seed(3)
    x, w, b, dy = (torch.randn(*s, generator=g).to(dtype) for s in ((30,), (11, 30), (11,), (11,)))
    ref = R.Linear(x[None], w, b, None, "silu", dy[None], dtype)
    xd, wd = x.to(cuda).requires_grad_(True), w.to(cuda).requires_grad_(True)
    y = gat_amd.linear_act(xd, wd, b.to(cuda), "silu")
    y.backward(dy.to(cuda))
    R.check(y[None], ref.y, "y")
    R.check(xd.grad[None], ref.dx, "dx")
    R.check(wd.grad, ref.dw, "dw")
    e = torch.zeros(4, 0, 30, device=cuda, dtype=dtype, requires_grad=True)
    z = gat_amd.linear_act(e, wd, b.to(cuda))
    assert z.shape == (4, 0, 11)
    ge, gw = torch.autograd.grad(z, (e, wd), torch.zeros_like(z))
    assert ge.shape == e.shape and not gw.any()
    d = gat_amd.dropout(x.to(cuda), 0.5, seed=4)
    assert torch.equal(d, gat_amd.dropout(x.to(cuda)[None], 0.5, seed=4)[0])
    for shape in ((3, 0), (0, 3), (2, 0, 5)):
        assert gat_amd.dropout(torch.zeros(*shape, device=cuda, dtype=dtype), 0.5).shape == shape


def test_an_operand_used_twice(cuda):
    """x as its own residual, one weight in two products, weight and bias of a norm the same tensor"""
    import gat_amd
    g = torch.Generator().manual_seed(5)
    x, w, v, dy = (torch.randn(*s, generator=g) for s in ((70, 24), (24, 24), (24,), (70, 24)))
    xd, wd, vd = (t.to(cuda).requires_grad_(True) for t in (x, w, v))
    h = gat_amd.linear_act(xd, wd, vd, "elu", xd)
    y = gat_amd.group_norm_act(gat_amd.linear_act(h, wd, None, "none", h), 4, vd, vd)
    got = torch.autograd.grad(y, (xd, wd, vd), dy.to(cuda))
    X, W, V = (t.double().requires_grad_(True) for t in (x, w, v))
    H = torch.nn.functional.elu(X @ W.t() + V) + X
    H = H @ W.t() + H
    Y = torch.nn.functional.group_norm(H, 4, V, V, 1e-5)
    # four f32 operators in a row, sums of at most 70 x 24 terms: each a few dozen steps of its summands, under
    # 100 U = 6e-6 of the largest value together
    for a, r in zip(got, torch.autograd.grad(Y, (X, W, V), dy.double())):
        assert float((a.cpu().double() - r).abs().max()) < 1e-5 * float(r.abs().max())


def test_backward_twice_and_checkpointed(cuda):
    """a retained graph gives the same gradients again; a checkpointed block draws the same mask again"""
    import gat_amd
    from torch.utils.checkpoint import checkpoint
    x = torch.randn(300, 64, device=cuda, requires_grad=True)
    w = torch.randn(64, 64, device=cuda, requires_grad=True)

    def block(x, w):
        return gat_amd.linear_act(gat_amd.dropout(x, 0.4), w, None, "gelu")

    torch.manual_seed(8)
    y = block(x, w)
    dy = torch.randn_like(y)
    first = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    again = torch.autograd.grad(y, (x, w), dy)
    torch.manual_seed(8)
    z = checkpoint(block, x, w, use_reentrant=False)
    torch.manual_seed(9)
    other = torch.autograd.grad(z, (x, w), dy)
    assert torch.equal(y, z)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, again, other))


def test_changed_in_place_before_the_backward(cuda):
    """what the backward needs is guarded as by torch's own operators"""
    import gat_amd
    x = torch.randn(40, 16, device=cuda)
    w = torch.randn(8, 16, device=cuda, requires_grad=True)
    y = gat_amd.linear_act(x, w)
    x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_two_streams_at_once(cuda):
    """long calls that overlap on two streams, each with workspaces of its own"""
    import gat_amd
    g = torch.Generator().manual_seed(6)
    sets = []
    for i in range(2):
        x = torch.randn(60000, 200, generator=g).to(cuda).requires_grad_(True)
        w = (torch.randn(96, 200, generator=g) / 14).to(cuda).requires_grad_(True)
        ids = torch.randint(0, 5000, (60000,), generator=g).to(cuda)
        t = torch.randn(5000, 96, generator=g).to(cuda).requires_grad_(True)
        v = torch.randn(96, generator=g).to(cuda)
        dy = torch.randn(60000, 96, generator=g).to(cuda)
        sets.append((x, w, ids, t, v, dy))

    def work(s):
        x, w, ids, t, v, dy = s
        y = gat_amd.linear_act(x, w, v, "silu", gat_amd.embedding(ids, t))
        y = gat_amd.group_norm_act(y.view(6, 10000, 96), 3, v, v, act="elu").view(60000, 96)
        return [y.detach(), *torch.autograd.grad(y, (x, w, t), dy)]

    want = [work(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for turn in range(3):
        got = []
        for s, st in zip(sets, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(work(s))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b)), turn
