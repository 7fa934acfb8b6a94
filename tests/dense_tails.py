"""Activations in 64 bits with RELATIVE error bounds, for tests of the dense operators where an activation is
saturated: values and slopes that are small themselves, not next to something of size 1.  Used by the tests only.

With terms t_i whose sum is the value (or the slope), f32 arithmetic on functions that are good to a few steps is
off by at most c (1 + z^2) sum |t_i|: the argument of an exponential, of size z^2 / 2 at most here, is rounded once or
twice, which moves its result by up to z^2 U relative, and every function and operation adds its own.  c is 8 U for
f32 tensors (library functions of at most four steps, U = 2^-24).  16-bit tensors use v_exp / v_rcp forms, whose own
part is below 2^-17: the polynomial of the normal distribution's tail is within 2^-17.9 relative, exp(z) - 1 within
2^-18 where it takes over from its series."""
import torch

U = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def act(z, name):
    """(value, slope, sum of the terms' sizes of the value, of the slope) in float64"""
    if name == "elu":
        e = torch.exp(z.clamp(max=0))
        m = torch.expm1(z.clamp(max=0))
        up = z > 0
        return torch.where(up, z, m), torch.where(up, torch.ones_like(z), e), torch.where(up, z, m).abs(), torch.where(up, torch.ones_like(z), e)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * torch.sigmoid(-z)), (z * s).abs(), s * (1 + z.abs())
    p = 0.5 * torch.special.erfc(-z / 2 ** 0.5)
    g = z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    return z * p, p + g, (z * p).abs(), p + g.abs()


def own(z, dtype):
    """the relative error of the function itself, times the terms' sizes"""
    return 8 * U * (1 + z * z) if dtype == torch.float32 else 2.0 ** -17 + 4 * U * (1 + z * z)


def coding(slope, dtype, name):
    """what the slope's way through memory may cost: f32 tensors nothing; 16-bit ones half a step of 2^-15, and where
    the slope is below 2^-5 and has the sign of the activation's lower tail half a step of eleven bits, or of 2^-37"""
    if dtype == torch.float32:
        return 0.0 * slope
    tail = (slope if name == "elu" else -slope) >= 0
    return torch.where(tail & (slope.abs() < 2.0 ** -5), 2.0 ** -11 * slope.abs() + 2.0 ** -38, 2.0 ** -16)


def within(got, want, bound, name):
    """every element within its bound, or within a step of the type's subnormal numbers (two roundings of half a step)"""
    got = got.detach().cpu()
    f = torch.finfo(got.dtype)
    assert got.shape == want.shape, name
    room = bound + f.smallest_normal * f.eps
    off = (got.double() - want).abs()
    if not bool((off <= room).all()):
        at = int(torch.argmax((off / room).reshape(-1).nan_to_num(nan=float("inf"))))
        raise AssertionError(f"{name}: {int((~(off <= room)).sum())} of {off.numel()} outside; worst at {at}: got "
                             f"{float(got.reshape(-1)[at])!r}, want {float(want.reshape(-1)[at])!r} within "
                             f"{float(room.reshape(-1)[at]):.3g}")
