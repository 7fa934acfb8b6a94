"""Group norm over positions whose data a shifted sum of squares would not survive: rows far from all others, at the
places where a block of the kernel starts."""
import pytest
import torch

import dense_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,groups,dtype", [((256, 12000, 8), 1, torch.float32), ((256, 12000, 8), 2, torch.bfloat16),
                                                ((3, 20011, 48), 4, torch.float32), ((1, 3000, 257), 1, torch.float32)])
@pytest.mark.parametrize("far,mean", [(1000.0, 0.0), (-3000.0, 2.0)])
def test_group_norm_outlying_rows(cuda, shape, groups, dtype, far, mean):
    """the first rows of every thousand are of size `far` (sink nodes, padding in front of data): means and variances to
    the bound of any f32 sum of 256 steps, so the outliers' own values are right"""
    import gat_amd
    g = torch.Generator().manual_seed(7)
    x = torch.randn(*shape, generator=g) + mean
    for first in range(0, shape[1], 1000):
        x[:, first] = far * (1 + torch.rand(shape[0], shape[2], generator=g))
    x = x.to(dtype)
    c = shape[2]
    w, b = (torch.randn(c, generator=g) * 0.2 + 1).to(dtype), (torch.randn(c, generator=g) * 0.3).to(dtype)
    ref = R.GroupNorm(x, groups, w, b, "none", None, dtype)
    with torch.no_grad():
        y = gat_amd.group_norm_act(x.to(cuda), groups, w.to(cuda), b.to(cuda))
    R.check(y, ref.y, "y")


def test_group_norm_saved_statistics_of_outlying_rows(cuda):
    """the statistics themselves, from the C entry point"""
    import ctypes as C
    from gat_amd import _lib
    lib = _lib.lib()
    n, length, c, groups = 64, 48000, 8, 2
    g = torch.Generator().manual_seed(3)
    x = torch.randn(n, length, c, generator=g)
    x[:, ::1000] = 2000.0
    xd = x.to(cuda)
    one, zero = torch.ones(c, device=cuda), torch.zeros(c, device=cuda)
    y, stats = torch.empty_like(xd), torch.empty(2, n, groups, device=cuda)
    d = _lib.GroupNorm(n, length, groups, c // groups, 0, 0, 1e-5, 0, one.data_ptr(), zero.data_ptr())
    need = lib.gatmi_group_norm_workspace_bytes(C.byref(d))
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    code = lib.gatmi_group_norm_fwd(C.byref(d), xd.data_ptr(), y.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(),
                                    ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert code == 0
    v = x.double().view(n, length, groups, -1)
    var, mean = torch.var_mean(v, dim=(1, 3), unbiased=False)
    rstd = (var + 1e-5).rsqrt()
    # a variance of squares around means, all of one sign: at most 256 additions one after another
    assert float((stats[1].cpu().double() / rstd - 1).abs().max()) < 256 * R.U
    assert float((stats[0].cpu().double() - mean).abs().max()) < 256 * R.U * float(v.abs().mean((1, 3)).max())
