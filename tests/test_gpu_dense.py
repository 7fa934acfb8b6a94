"""The dense operators (gat_amd/dense.py, csrc/linear.hip, group_norm.hip, embedding.hip, dropout.hip) on the
GPU against their definitions in 64 bits (tests/dense_ref.py), element by element within derived bounds."""
import pytest
import torch

import dense_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def leaf(t, cuda):
    return t.to(cuda).requires_grad_(True)


# ---- linear ----------------------------------------------------------------------------------
def linear_case(cuda, dtype, m, k, n, act, bias, res, seed=0, scale=1.0):
    import gat_amd
    g = gen(seed + 7 * m + 31 * k + n)
    x = (torch.randn(m, k, generator=g) * scale).to(dtype)
    w = (torch.randn(n, k, generator=g) / k ** 0.5).to(dtype)
    b = (torch.randn(n, generator=g) * 0.3).to(dtype) if bias else None
    r = torch.randn(m, n, generator=g).to(dtype) if res else None
    dy = torch.randn(m, n, generator=g).to(dtype)
    ref = R.Linear(x, w, b, r, act, dy, dtype)
    leaves = [None if t is None else leaf(t, cuda) for t in (x, w, b, r)]
    with torch.no_grad():
        R.check(gat_amd.linear_act(leaves[0], leaves[1], leaves[2], act, leaves[3]), ref.y, "y, no gradient")
    y = gat_amd.linear_act(leaves[0], leaves[1], leaves[2], act, leaves[3])
    y.backward(dy.to(cuda))
    R.check(y, ref.y, "y")
    R.check(leaves[0].grad, ref.dx, "dx")
    R.check(leaves[1].grad, ref.dw, "dw")
    if bias:
        R.check(leaves[2].grad, ref.db, "db")
    if res:
        assert torch.equal(leaves[3].grad, dy.to(cuda))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 240, 240), (2, 7, 3), (3, 25, 9), (17, 240, 2), (64, 64, 64),
                                   (127, 33, 129), (128, 128, 128), (129, 130, 131), (300, 100, 256), (513, 8, 40),
                                   (1000, 256, 256), (2500, 61, 47), (4, 1500, 700), (40, 515, 1)])
def test_linear_matches(cuda, dtype, m, k, n):
    linear_case(cuda, dtype, m, k, n, "gelu", True, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("bias,res", [(False, False), (True, False), (False, True)])
def test_linear_activations(cuda, dtype, act, bias, res):
    linear_case(cuda, dtype, 333, 48, 72, act, bias, res, scale=2.0)


def test_linear_many_rows(cuda):
    for dtype in DTYPES:
        linear_case(cuda, dtype, 70001, 24, 30, "elu", True, True)


def test_linear_leading_axes_strides_and_alignment(cuda):
    """x [a, b, in], transposed and sliced operands, tensors that start one element into an allocation"""
    import gat_amd
    g = gen(5)
    for dtype in DTYPES:
        base = torch.randn(11 * 5 * 37 + 1, generator=g).to(dtype)
        wt = torch.randn(37, 21, generator=g).to(dtype)
        bb = torch.randn(43, generator=g).to(dtype)
        rt = torch.randn(21, 5, 11, generator=g).to(dtype)
        xd = base.to(cuda)[1:].view(11, 5, 37).requires_grad_(True)
        y = gat_amd.linear_act(xd, wt.to(cuda).t(), bb.to(cuda)[1:43:2], "silu", rt.to(cuda).permute(2, 1, 0))
        dy = torch.randn(5, 11, 21, generator=g).to(dtype)
        ref = R.Linear(base[1:].view(55, 37), wt.t(), bb[1:43:2], rt.permute(2, 1, 0).reshape(55, 21), "silu",
                       dy.transpose(0, 1).reshape(55, 21), dtype)
        (gx,) = torch.autograd.grad(y, xd, dy.to(cuda).transpose(0, 1))
        R.check(y.reshape(55, 21), ref.y, "y")
        R.check(gx.reshape(55, 37), ref.dx, "dx")


def test_linear_gradients_of_some_operands(cuda):
    import gat_amd
    g = gen(6)
    x, w, b = (torch.randn(*s, generator=g) for s in ((50, 20), (30, 20), (30,)))
    dy = torch.randn(50, 30, generator=g)
    ref = R.Linear(x, w, b, None, "elu", dy, F32)
    for want in ((0,), (1,), (2,), (0, 2), (1, 2)):
        ts = [t.to(cuda).requires_grad_(i in want) for i, t in enumerate((x, w, b))]
        grads = torch.autograd.grad(gat_amd.linear_act(*ts, act="elu"), [ts[i] for i in want], dy.to(cuda))
        for i, got in zip(want, grads):
            R.check(got, (ref.dx, ref.dw, ref.db)[i], str(i))
    # a broadcast gradient (stride 0) arrives from sum()
    xd = leaf(x, cuda)
    gat_amd.linear_act(xd, w.to(cuda), b.to(cuda)).sum().backward()
    R.check(xd.grad, R.Linear(x, w, b, None, "none", torch.ones(50, 30), F32).dx, "dx of a sum")


def test_linear_of_no_rows(cuda):
    import gat_amd
    for dtype in DTYPES:
        x, w, b = (torch.zeros(*s, dtype=dtype, device=cuda, requires_grad=True) for s in ((0, 5), (7, 5), (7,)))
        y = gat_amd.linear_act(x, w, b, "gelu")
        assert y.shape == (0, 7)
        y.backward(torch.zeros(0, 7, dtype=dtype, device=cuda))
        assert x.grad.shape == (0, 5) and not w.grad.any() and not b.grad.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_infinities_and_nan_stay_in_their_rows(cuda, dtype):
    """an infinite operand gives what the sum gives, and no other row or column is touched"""
    import gat_amd
    g = gen(8)
    x, w = torch.randn(200, 50, generator=g).to(dtype), torch.randn(70, 50, generator=g).to(dtype)
    x[3, 4], x[150, 49], x[151, 0] = float("inf"), float("nan"), -float("inf")
    w[5, 4] = 0.5                                  # exact in every type: its low pieces are zero
    w[6, 4] = 0.0
    ref = x.double() @ w.double().t()
    y = gat_amd.linear_act(x.to(cuda), w.to(cuda)).cpu().double()
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(torch.isinf(y), torch.isinf(ref))
    assert torch.equal(y[torch.isinf(y)], ref[torch.isinf(ref)])
    xd, wd = leaf(x, cuda), leaf(w, cuda)
    dy = torch.ones(200, 70, dtype=dtype)
    dy[9, 9] = float("inf")
    gat_amd.linear_act(xd, wd).backward(dy.to(cuda))
    rx, rw = dy.double() @ w.double(), dy.double().t() @ x.double()
    for got, want in ((xd.grad, rx), (wd.grad, rw)):
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))


def test_linear_f32_at_the_edge_of_its_range(cuda):
    """values whose first bf16 piece rounds up to infinity, and ones whose pieces are subnormal"""
    import gat_amd
    big = torch.finfo(F32).max
    x = torch.tensor([[big, 0.0], [big * 0.999, 1.0], [1e-30, 3.0], [-big, 0.0]])
    w = torch.tensor([[1.0, 0.0], [0.5, 1.0], [-1.0, 2.0]])
    ref = R.Linear(x, w, None, None, "none", None, F32)
    R.check(gat_amd.linear_act(x.to(cuda), w.to(cuda)), ref.y, "y")


def test_linear_same_inputs_same_bits(cuda):
    import gat_amd
    for dtype in DTYPES:
        x = torch.randn(5000, 130, device=cuda).to(dtype).requires_grad_(True)
        w = torch.randn(90, 130, device=cuda).to(dtype).requires_grad_(True)
        dy = torch.randn(5000, 90, device=cuda).to(dtype)
        runs = []
        for _ in range(2):
            y = gat_amd.linear_act(x, w, act="gelu")
            runs.append([y, *torch.autograd.grad(y, (x, w), dy)])
        assert all(torch.equal(a, b) for a, b in zip(*runs))


# ---- group norm ------------------------------------------------------------------------------
def group_norm_case(cuda, dtype, shape, groups, act, shift=0.3, scale=1.5, seed=0):
    import gat_amd
    c = shape[-1]
    g = gen(seed + sum(shape) * 13 + groups)
    x = (torch.randn(*shape, generator=g) * scale + shift).to(dtype)
    w, b = (torch.randn(c, generator=g) * 0.2 + 1).to(dtype), (torch.randn(c, generator=g) * 0.3).to(dtype)
    dy = torch.randn(*shape, generator=g).to(dtype)
    ref = R.GroupNorm(x, groups, w, b, act, dy, dtype)
    xd, wd, bd = (leaf(t, cuda) for t in (x, w, b))
    with torch.no_grad():
        R.check(gat_amd.group_norm_act(xd, groups, wd, bd, act=act), ref.y, "y, no gradient")
    y = gat_amd.group_norm_act(xd, groups, wd, bd, act=act)
    y.backward(dy.to(cuda))
    R.check(y, ref.y, "y")
    R.check(xd.grad, ref.dx, "dx")
    R.check(wd.grad, ref.dw, "dw")
    R.check(bd.grad, ref.db, "db")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", [
    ((1, 8), 1), ((5, 6), 6), ((3, 14), 2), ((2708, 240), 8), ((999, 64), 4), ((70, 7), 1), ((33, 66), 2), ((100, 320), 8),
    ((50, 1000), 1), ((9, 4100), 2), ((4, 2049), 1), ((3, 8192), 1), ((1000, 21), 3), ((6, 8000), 1000), ((4097, 30), 5),
    ((2, 5, 12), 3), ((1, 1000, 16), 2), ((3, 333, 48), 4), ((2, 7000, 30), 5), ((5, 40, 2050), 2), ((2, 3, 4, 20), 4),
    ((70, 2, 3), 3), ((1, 2, 4100), 4), ((4, 1, 24), 2), ((1, 20011, 8), 8)])
def test_group_norm_matches(cuda, dtype, shape, groups):
    group_norm_case(cuda, dtype, shape, groups, "silu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("shape", [(400, 60), (2, 300, 60)])
def test_group_norm_activations(cuda, dtype, act, shape):
    group_norm_case(cuda, dtype, shape, 4, act)


def test_group_norm_far_from_zero(cuda):
    """mean >> deviation: a variance from sums of squares would lose every digit"""
    group_norm_case(cuda, F32, (500, 128), 2, "none", shift=500.0, scale=0.05)
    group_norm_case(cuda, F32, (2, 3000, 32), 2, "none", shift=500.0, scale=0.05)


def test_group_norm_constant_groups(cuda):
    """variance 0: xh is 0 whatever the group's value, y = act(bias), dx as the formula with rstd = eps^-1/2"""
    import gat_amd
    for shape in ((6, 24), (2, 50, 24)):
        for dtype in DTYPES:
            x = torch.full(shape, 3.0).to(dtype)
            w, b = torch.linspace(0.5, 1.5, 24).to(dtype), torch.linspace(-1, 1, 24).to(dtype)
            y = gat_amd.group_norm_act(x.to(cuda), 3, w.to(cuda), b.to(cuda), act="none")
            assert torch.equal(y.cpu(), b.expand(shape))


def test_group_norm_strides_alignment_empty(cuda):
    import gat_amd
    g = gen(11)
    for dtype in DTYPES:
        base = torch.randn(40 * 30 + 1, generator=g).to(dtype)
        w, b = torch.randn(61, generator=g).to(dtype), torch.randn(31, generator=g).to(dtype)
        xd = base.to(cuda)[1:].view(40, 30).requires_grad_(True)
        dy = torch.randn(30, 40, generator=g).to(dtype)
        ref = R.GroupNorm(base[1:].view(40, 30), 3, w[1::2], b[1:], "elu", dy.t(), dtype)
        y = gat_amd.group_norm_act(xd, 3, w.to(cuda)[1::2], b.to(cuda)[1:], act="elu")
        (gx,) = torch.autograd.grad(y, xd, dy.to(cuda).t())
        R.check(y, ref.y, "y")
        R.check(gx, ref.dx, "dx")
        # channels first in memory, channels last in shape
        xt = torch.randn(2, 24, 50, generator=g).to(dtype)
        w2, b2 = torch.randn(24, generator=g).to(dtype), torch.randn(24, generator=g).to(dtype)
        ref = R.GroupNorm(xt.transpose(1, 2), 4, w2, b2, "none", None, dtype)
        R.check(gat_amd.group_norm_act(xt.to(cuda).transpose(1, 2), 4, w2.to(cuda), b2.to(cuda)), ref.y, "y")
        x0 = torch.zeros(0, 24, dtype=dtype, device=cuda, requires_grad=True)
        wd, bd = leaf(w2, cuda), leaf(b2, cuda)
        gat_amd.group_norm_act(x0, 4, wd, bd).backward(torch.zeros(0, 24, dtype=dtype, device=cuda))
        assert x0.grad.shape == (0, 24) and not wd.grad.any() and not bd.grad.any()


def test_group_norm_nan_stays_in_its_group(cuda):
    import gat_amd
    x = torch.randn(20, 40, generator=gen(3))
    x[4, 13], x[7, 0] = float("nan"), float("inf")
    y = gat_amd.group_norm_act(x.to(cuda), 4, torch.ones(40, device=cuda), torch.zeros(40, device=cuda), act="elu").cpu()
    bad = torch.zeros(20, 40, dtype=torch.bool)
    bad[4, 10:20], bad[7, 0:10] = True, True
    assert torch.equal(torch.isnan(y), bad)


# ---- embedding -------------------------------------------------------------------------------
def embedding_case(cuda, dtype, ids, vocab, dim, scale, seed=0):
    import gat_amd
    g = gen(seed + vocab + dim)
    table = torch.randn(vocab, dim, generator=g).to(dtype)
    dy = torch.randn(*ids.shape, dim, generator=g).to(dtype)
    y_ref, g_ref = R.embedding(ids, table, scale, dy, dtype)
    td = leaf(table, cuda)
    y = gat_amd.embedding(ids.to(cuda), td, scale)
    y.backward(dy.to(cuda))
    assert y.shape == ids.shape + (dim,)
    R.check(y.reshape(-1, dim), y_ref, "y")
    R.check(td.grad, g_ref, "grad")
    (again,) = torch.autograd.grad(gat_amd.embedding(ids.to(cuda), td, scale), td, dy.to(cuda))
    assert torch.equal(again, td.grad)                       # no order but the ids'


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (1, 5, 30), (7, 3, 2), (169, 1025, 30), (256, 256, 8), (257, 255, 16),
                                         (4096, 40, 33), (4097, 70000, 5), (5000, 300, 3), (20000, 17, 64),
                                         (9000, 9000, 100), (300, 66000, 257), (2000, 7, 513), (50, 11, 2100)])
def test_embedding_matches(cuda, dtype, n, vocab, dim):
    ids = torch.randint(0, vocab, (n,), generator=gen(n + dim))
    embedding_case(cuda, dtype, ids, vocab, dim, 1.0 if n % 2 else dim ** 0.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_frequent_ids(cuda, dtype):
    """one id nearly everywhere (its sum crosses many chunks), runs of equal ids, ids in descending order"""
    g = gen(2)
    ids = torch.full((30011,), 6)
    ids[torch.randint(0, 30011, (500,), generator=g)] = torch.randint(0, 50, (500,), generator=g)
    embedding_case(cuda, dtype, ids, 50, 12, 1.0)
    embedding_case(cuda, dtype, torch.full((17000,), 2), 3, 40, 0.5)
    embedding_case(cuda, dtype, torch.arange(9999, -1, -1) // 100, 100, 20, 1.0)
    embedding_case(cuda, dtype, torch.arange(3000) % 16, 16, 20, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_ids_outside_the_table(cuda, dtype):
    g = gen(4)
    ids = torch.randint(-3, 40, (1000, 3), generator=g)      # 33 .. 39 are past the end
    ids[0, 0], ids[1, 0], ids[2, 0] = 1 << 40, -(1 << 62), (1 << 32) + 5
    embedding_case(cuda, dtype, ids, 33, 24, 2.0)
    embedding_case(cuda, dtype, torch.full((600,), -1), 33, 24, 1.0)


def test_embedding_shapes_strides_empty(cuda):
    import gat_amd
    for dtype in DTYPES:
        table = torch.randn(24, 41, generator=gen(9)).to(dtype)
        ids = torch.randint(0, 41, (6, 50), generator=gen(10))
        y = gat_amd.embedding(ids.to(cuda).t(), table.to(cuda).t())
        assert torch.equal(y.cpu(), table.t()[ids.t()])
        one = torch.tensor([3.0, 4.0, 5.0, 6.0, 7.0]).to(dtype).to(cuda)[1:].view(2, 2)   # odd start
        assert torch.equal(gat_amd.embedding(torch.tensor(1, device=cuda), one).cpu(), torch.tensor([6.0, 7.0]).to(dtype))
        td = leaf(table, cuda)
        y = gat_amd.embedding(torch.zeros(0, 4, dtype=torch.long, device=cuda), td)
        assert y.shape == (0, 4, 41)
        y.sum().backward()
        assert td.grad.shape == (24, 41) and not td.grad.any()


# ---- dropout ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,p", [(1, 1, 0.5), (100, 25, 0.425), (7, 1000, 0.1), (5000, 8, 0.9), (333, 33, 0.3),
                                         (3, 100003, 0.25), (70001, 3, 0.7), (900, 256, 0.5)])
@pytest.mark.parametrize("res", [False, True])
def test_dropout_matches(cuda, dtype, rows, cols, p, res):
    import gat_amd
    from gat_amd.glue import dropout_mask
    g = gen(rows + cols)
    seed = 0x1234567_89ABCDEF + rows
    x, dy = torch.randn(rows, cols, generator=g).to(dtype), torch.randn(rows, cols, generator=g).to(dtype)
    r = torch.randn(rows, cols, generator=g).to(dtype) if res else None
    keep = dropout_mask(rows, cols, p, seed, cuda).cpu()
    assert abs(float(keep.float().mean()) - (1 - p)) < 5 * (p * (1 - p) / (rows * cols)) ** 0.5 + 1e-6
    xd, rd = leaf(x, cuda), None if r is None else leaf(r, cuda)
    y = gat_amd.dropout(xd, p, seed=seed, residual=rd)
    y.backward(dy.to(cuda))
    inv = 1.0 / (1.0 - p)
    a = torch.where(keep, x.double() * inv, 0.0)
    want = a if r is None else a + r.double()
    R.check(y, (want, 4 * R.U * (a.abs() + want.abs()) + R.u(dtype) * want.abs()), "y")
    gx = torch.where(keep, dy.double() * inv, 0.0)
    R.check(xd.grad, (gx, (4 * R.U + R.u(dtype)) * gx.abs()), "dx")
    if res:
        assert torch.equal(rd.grad.cpu(), dy)


def test_dropout_off_alignment_nan(cuda):
    import gat_amd
    x = torch.randn(50, 7, device=cuda)
    assert gat_amd.dropout(x, 0.4, training=False) is x and gat_amd.dropout(x, 0.0) is x
    assert torch.equal(gat_amd.dropout(x, 0.4, training=False, residual=x), x + x)
    for dtype in DTYPES:
        base = torch.randn(3001, generator=gen(1)).to(dtype).to(cuda)
        a = gat_amd.dropout(base[1:].view(100, 30), 0.5, seed=9)
        b = gat_amd.dropout(base[1:].clone().view(100, 30), 0.5, seed=9)
        c = gat_amd.dropout(base[1:].clone().view(30, 100).t(), 0.5, seed=9)     # its own [100, 30] rows
        assert torch.equal(a, b)
        assert torch.equal(c != 0, b != 0)
        bad = torch.full((64, 32), float("inf"), dtype=dtype, device=cuda)
        y = gat_amd.dropout(bad, 0.5, seed=3)
        assert not torch.isnan(y).any() and bool((y == 0).any()) and bool(torch.isinf(y).any())
    # draws differ from call to call, and follow torch's generator
    torch.manual_seed(5)
    d1, d2 = gat_amd.dropout(x, 0.5), gat_amd.dropout(x, 0.5)
    torch.manual_seed(5)
    assert torch.equal(d1, gat_amd.dropout(x, 0.5)) and not torch.equal(d1, d2)
    e = torch.zeros(0, 5, device=cuda, requires_grad=True)
    gat_amd.dropout(e, 0.5, seed=1).sum().backward()
    assert e.grad.shape == (0, 5)


def test_dropout_with_a_device_seed(cuda):
    """two uses of one seed tensor before any backward: each backward draws its own forward's mask"""
    import gat_amd
    seed = torch.tensor([1 << 40], device=cuda)
    x = torch.ones(200, 50, device=cuda, requires_grad=True)
    a, b = gat_amd.dropout(x, 0.5, seed=seed), gat_amd.dropout(x, 0.5, seed=seed)
    assert not torch.equal(a, b)
    (ga,), (gb,) = (torch.autograd.grad(t, x, torch.ones_like(t)) for t in (a, b))
    assert torch.equal(ga, a.detach()) and torch.equal(gb, b.detach())
    by_value = gat_amd.dropout(x, 0.5, seed=int(seed))
    assert torch.equal(by_value, b)


# ---- refusals, streams, graphs, all of them together -------------------------------------------
def test_refusals(cuda):
    import gat_amd
    z = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device=cuda)
    ids = torch.zeros(4, dtype=torch.long, device=cuda)
    for bad, error in (
            (lambda: gat_amd.linear_act(z(4, 8), z(3, 7)), ValueError),
            (lambda: gat_amd.linear_act(z(4, 8), z(0, 8)), ValueError),
            (lambda: gat_amd.linear_act(z(4, 0), z(3, 0)), ValueError),
            (lambda: gat_amd.linear_act(z(4, 8), z(3, 8), z(4)), ValueError),
            (lambda: gat_amd.linear_act(z(4, 8), z(3, 8), residual=z(4, 4)), ValueError),
            (lambda: gat_amd.linear_act(z(4, 8), z(3, 8), act="tanh"), ValueError),
            (lambda: gat_amd.linear_act(z(4, 8), z(3, 8, dtype=BF16)), TypeError),
            (lambda: gat_amd.linear_act(z(4, 8, dtype=torch.float64), z(3, 8, dtype=torch.float64)), TypeError),
            (lambda: gat_amd.group_norm_act(z(4, 8), 3, z(8), z(8)), ValueError),
            (lambda: gat_amd.group_norm_act(z(4, 8), 0, z(8), z(8)), ValueError),
            (lambda: gat_amd.group_norm_act(z(4, 8), 2, z(7), z(8)), ValueError),
            (lambda: gat_amd.group_norm_act(z(8), 2, z(8), z(8)), ValueError),
            (lambda: gat_amd.group_norm_act(z(4, 8), 2, z(8), z(8), eps=-1.0), ValueError),
            (lambda: gat_amd.group_norm_act(z(4, 0, 8), 2, z(8), z(8)), ValueError),
            (lambda: gat_amd.group_norm_act(z(2, 8200), 2, z(8200), z(8200)), ValueError),
            (lambda: gat_amd.group_norm_act(z(4, 8), 2, z(8, dtype=F16), z(8)), TypeError),
            (lambda: gat_amd.embedding(ids.int(), z(4, 8)), TypeError),
            (lambda: gat_amd.embedding(ids, z(8)), ValueError),
            (lambda: gat_amd.embedding(ids.cpu(), z(4, 8)), ValueError),
            (lambda: gat_amd.dropout(z(4, 8), 1.0), ValueError),
            (lambda: gat_amd.dropout(z(4, 8), -0.1), ValueError),
            (lambda: gat_amd.dropout(z(4, 8), 0.5, residual=z(8, 4)), ValueError),
            (lambda: gat_amd.dropout(z(4, 8), 0.5, seed=torch.zeros(1, device=cuda)), ValueError)):
        with pytest.raises(error):
            bad()
    x = z(4, 8).requires_grad_(True)
    (gx,) = torch.autograd.grad(gat_amd.linear_act(x, z(3, 8), act="gelu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


class Block:
    """embedding -> dropout -> linear (+ residual) -> group norm, forward and backward"""

    def __init__(self, cuda, dtype, n=700, seed=0):
        g = gen(seed)
        to = lambda t: t.to(dtype).to(cuda)
        self.ids = torch.randint(-1, 60, (n,), generator=g).to(cuda)
        self.table = to(torch.randn(60, 40, generator=g)).requires_grad_(True)
        self.w = to(torch.randn(48, 40, generator=g) / 6).requires_grad_(True)
        self.b = to(torch.randn(48, generator=g)).requires_grad_(True)
        self.res = to(torch.randn(n, 48, generator=g))
        self.gw, self.gb = (to(torch.randn(48, generator=g) + s).requires_grad_(True) for s in (1, 0))
        self.dy = to(torch.randn(n, 48, generator=g))
        self.seed = torch.tensor([77], device=cuda)
        self.leaves = [self.table, self.w, self.b, self.gw, self.gb]

    def __call__(self):
        import gat_amd
        h = gat_amd.embedding(self.ids, self.table, 2.0)
        h = gat_amd.dropout(h, 0.3, seed=self.seed)
        h = gat_amd.linear_act(h, self.w, self.b, "gelu", self.res)
        y = gat_amd.group_norm_act(h, 4, self.gw, self.gb, act="elu")
        return [y.detach(), *torch.autograd.grad(y, self.leaves, self.dy)]


def test_block_matches_64_bits(cuda):
    """the four in a row, f32: within 1e-5 of the largest value of each result (each operator's own bound is
    a few dozen f32 steps of its summands; four in a row with sums of 700 rows stay below 100 U = 6e-6)"""
    from gat_amd.glue import SEED_STEP, dropout_mask
    blk = Block(cuda, F32)
    got = blk()
    keep = dropout_mask(700, 40, 0.3, (77 + SEED_STEP) % (1 << 64), cuda).cpu()
    t, w, b, gw, gb = (p.detach().cpu().double().requires_grad_(True) for p in blk.leaves)
    ids = blk.ids.cpu()
    h = torch.where((ids >= 0)[:, None], t[ids.clamp(min=0)] * 2.0, torch.zeros((), dtype=torch.float64))
    h = torch.where(keep, h / 0.7, torch.zeros((), dtype=torch.float64))
    h = torch.nn.functional.gelu(h @ w.t() + b) + blk.res.cpu().double()
    y = torch.nn.functional.elu(torch.nn.functional.group_norm(h, 4, gw, gb, 1e-5))
    want = [y, *torch.autograd.grad(y, (t, w, b, gw, gb), blk.dy.cpu().double())]
    for i, (a, r) in enumerate(zip(got, want)):
        assert float((a.cpu().double() - r).abs().max()) < 1e-5 * float(r.abs().max()), i


@pytest.mark.parametrize("dtype", DTYPES)
def test_block_on_another_stream(cuda, dtype):
    blk = Block(cuda, dtype)
    want = blk()
    blk.seed.fill_(77)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = blk()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_block_captured_and_replayed(cuda, dtype):
    """replays equal eager runs from the same seeds, with eager work between them; two graphs share nothing"""
    blk, other = Block(cuda, dtype), Block(cuda, dtype, n=300, seed=1)
    for b in (blk, other):      # warm up on a side stream, as captures want it
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b()
        torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for b in (blk, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = b()
        graphs.append(graph)
        outs.append(out)
    for step in range(4):
        for b, graph, out in zip((blk, other), graphs, outs):
            b.seed.fill_(1000 + step)
            want = [t.clone() for t in b()]
            b.seed.fill_(1000 + step)
            for t in out:
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(out, want)), step
