"""The dense operators without a GPU: argument checks of the C entry points (which return before anything is
launched) and of the Python ones, struct layouts, and the 64-bit references the GPU tests use against
differences."""
import ctypes as C

import pytest
import torch

import dense_ref as R
from gat_amd import _lib


def rc(code):
    return code, _lib.lib().gatmi_last_error().decode()


def test_struct_layouts():
    assert C.sizeof(_lib.Linear) == 24
    assert C.sizeof(_lib.GroupNorm) == 56 and _lib.GroupNorm.weight.offset == 40


@pytest.mark.parametrize("fields,word", [
    (dict(dtype=3), "element type"), (dict(dtype=-1), "element type"), (dict(act=5), "activation"),
    (dict(in_features=0), "features"), (dict(out_features=65537), "features"), (dict(rows=-1), "rows"),
    (dict(rows=1 << 31), "rows")])
def test_linear_refusals(fields, word):
    lib = _lib.lib()
    d = _lib.Linear(4, 8, 8, 0, 0)
    for k, v in fields.items():
        setattr(d, k, v)
    for code in (lib.gatmi_linear_fwd(C.byref(d), 256, 256, None, None, 256, None, 256, 1 << 30, None),
                 lib.gatmi_linear_bwd(C.byref(d), 256, 256, None, 256, None, None, None, 256, 1 << 30, None)):
        code, msg = rc(code)
        assert code == 1 and word in msg
    assert lib.gatmi_linear_bwd_workspace_bytes(C.byref(d)) == 0


def test_linear_null_and_workspace():
    lib = _lib.lib()
    d = _lib.Linear(4, 8, 8, 0, 2)
    assert rc(lib.gatmi_linear_fwd(C.byref(d), None, 256, None, None, 256, None, None, 0, None))[0] == 1
    assert rc(lib.gatmi_linear_fwd(None, 256, 256, None, None, 256, None, None, 0, None))[0] == 1
    code, msg = rc(lib.gatmi_linear_bwd(C.byref(d), 256, 256, None, 256, 256, 256, 256, 256, 1 << 30, None))
    assert code == 1 and "slope" in msg
    code, msg = rc(lib.gatmi_linear_bwd(C.byref(d), 256, 256, 256, 256, 256, 256, 256, 256, 16, None))
    assert code == 4 and "workspace" in msg
    d.rows = 0
    assert lib.gatmi_linear_fwd(C.byref(d), None, None, None, None, None, None, None, 0, None) == 0
    d.rows = 1 << 20
    code, msg = rc(lib.gatmi_linear_fwd(C.byref(d), 256, 256, None, None, 256, None, None, 0, None))
    assert code == 4 and "workspace" in msg


@pytest.mark.parametrize("fields,word", [
    (dict(dtype=7), "element type"), (dict(act=-1), "activation"), (dict(groups=0), "groups"), (dict(width=0), "groups"),
    (dict(groups=1024, width=9), "channels"), (dict(batch=-1), "batch"), (dict(length=0), "length"),
    (dict(batch=1 << 31), "batch"), (dict(length=1 << 31), "length"), (dict(eps=-1.0), "eps")])
def test_group_norm_refusals(fields, word):
    lib = _lib.lib()
    d = _lib.GroupNorm(4, 1, 2, 8, 0, 0, 1e-5, 0, 256, 256)
    for k, v in fields.items():
        setattr(d, k, v)
    for code in (lib.gatmi_group_norm_fwd(C.byref(d), 256, 256, 256, 256, 256, 1 << 40, None),
                 lib.gatmi_group_norm_bwd(C.byref(d), 256, 256, 256, 256, 256, 256, 256, 256, 1 << 40, None)):
        code, msg = rc(code)
        assert code == 1 and word in msg
    assert lib.gatmi_group_norm_workspace_bytes(C.byref(d)) == 0


def test_group_norm_null_and_workspace():
    lib = _lib.lib()
    d = _lib.GroupNorm(4, 7, 2, 8, 0, 0, 1e-5, 0, 256, 256)
    assert rc(lib.gatmi_group_norm_fwd(C.byref(d), None, 256, 256, 256, 256, 1 << 40, None))[0] == 1
    assert rc(lib.gatmi_group_norm_fwd(C.byref(d), 256, 256, 256, None, 256, 1 << 40, None))[0] == 1
    assert rc(lib.gatmi_group_norm_fwd(C.byref(d), 256, 256, None, None, 256, 1 << 40, None))[0] == 1
    assert rc(lib.gatmi_group_norm_fwd(C.byref(d), 256, 256, 256, 256, 256, 16, None))[0] == 4
    assert rc(lib.gatmi_group_norm_bwd(C.byref(d), 256, 256, 256, 256, 256, 256, 256, 256, 16, None))[0] == 4
    assert rc(lib.gatmi_group_norm_bwd(C.byref(d), 256, 256, None, 256, 256, 256, 256, 256, 1 << 40, None))[0] == 1
    d.batch = 0
    assert lib.gatmi_group_norm_fwd(C.byref(d), None, None, None, None, None, 0, None) == 0


def test_embedding_refusals():
    lib = _lib.lib()
    for args in ((3, 4, 4, 4), (0, -1, 4, 4), (0, 1 << 31, 4, 4), (0, 4, -1, 4), (0, 4, 1 << 31, 4), (0, 4, 4, 0),
                 (0, 4, 4, 65537)):
        assert rc(lib.gatmi_embedding_fwd(*args, 1.0, 256, 256, 256, None))[0] == 1
        assert rc(lib.gatmi_embedding_bwd(*args, 1.0, 256, 256, 256, 256, 1 << 40, None))[0] == 1
    assert lib.gatmi_embedding_bwd_workspace_bytes(-1, 4, 4) == 0
    assert rc(lib.gatmi_embedding_fwd(0, 4, 4, 4, 1.0, None, 256, 256, None))[0] == 1
    assert rc(lib.gatmi_embedding_bwd(0, 4, 4, 4, 1.0, 256, 256, 256, 256, 16, None))[0] == 4
    assert lib.gatmi_embedding_fwd(0, 0, 4, 4, 1.0, None, None, None, None) == 0


def test_dropout_refusals():
    lib = _lib.lib()
    for args in ((3, 4, 4, 0.5), (0, -1, 4, 0.5), (0, 1 << 32, 4, 0.5), (0, 4, 0, 0.5), (0, 4, 1 << 31, 0.5),
                 (0, 4, 4, 1.0), (0, 4, 4, -0.1), (0, 4, 4, float("nan"))):
        assert rc(lib.gatmi_dropout(*args, 1, None, None, 256, None, 256, None))[0] == 1
    assert rc(lib.gatmi_dropout(0, 4, 4, 0.5, 1, None, None, None, None, 256, None))[0] == 1
    assert lib.gatmi_dropout(0, 0, 4, 0.5, 1, None, None, None, None, None, None) == 0


def test_python_entry_points_refuse_cpu_tensors():
    import gat_amd
    x = torch.zeros(4, 8)
    for call in (lambda: gat_amd.linear_act(x, torch.zeros(3, 8)),
                 lambda: gat_amd.group_norm_act(x, 2, torch.ones(8), torch.zeros(8)),
                 lambda: gat_amd.embedding(torch.zeros(4, dtype=torch.long), x), lambda: gat_amd.dropout(x, 0.5)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


@pytest.mark.parametrize("name", ["none", "elu", "silu", "gelu"])
def test_references_agree_with_differences(name):
    """the 64-bit gradients the GPU tests hold the kernels to, against central differences"""
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, w, b, res, dy = rnd(5, 6), rnd(4, 6), rnd(4), rnd(5, 4), rnd(5, 4)
    ref = R.Linear(x, w, b, res, name, dy, torch.float32)
    h = 1e-5
    for arg, grad in ((0, ref.dx[0]), (1, ref.dw[0]), (2, ref.db[0])):
        args = [x, w, b]
        v = rnd(*args[arg].shape)
        def at(t):
            moved = list(args)
            moved[arg] = args[arg] + t * v
            return float((R.Linear(*moved, res, name, None, torch.float32).y[0] * dy).sum())
        diff = (at(h) - at(-h)) / (2 * h)
        assert abs(diff - float((grad * v).sum())) < 1e-7 * (1 + abs(diff)) * 10
    args = [x, w[0], b[[0, 1, 2, 3, 0, 1]]]
    dyg = rnd(5, 6)
    gn = R.GroupNorm(args[0], 2, args[1], args[2], name, dyg, torch.float32)
    for arg, grad in ((0, gn.dx[0]), (1, gn.dw[0]), (2, gn.db[0])):
        v = rnd(*args[arg].shape)
        def at2(t):
            moved = list(args)
            moved[arg] = args[arg] + t * v
            return float((R.GroupNorm(moved[0], 2, moved[1], moved[2], name, None, torch.float32).y[0] * dyg).sum())
        diff = (at2(h) - at2(-h)) / (2 * h)
        assert abs(diff - float((grad * v).sum())) < 1e-6 * (1 + abs(diff))


@pytest.mark.parametrize("which", range(7))
def test_difference_cases_have_power(which):
    """a gradient that is off by 5% fails them"""
    import dense_diff as D
    op, kw, shapes = D.CASES[which]
    if op == "dropout":
        kw = dict(kw, keep=torch.rand(*shapes[0]) >= kw["p"])
    *_, want, bound = D.case(op, kw, shapes)
    assert want > 0 and bound < 0.05 * want, (want, bound)
