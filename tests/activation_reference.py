"""The activation operators from their definitions, in 64 bits on the CPU: what the tests compare the kernels with."""

import torch

GROUP = 32
U32 = 2.0**-24  # half a step of float32
RANGE = {torch.float32: (-126, 121), torch.bfloat16: (-126, 121), torch.float16: (-24, 9)}


def unit_roundoff(dtype):
    return torch.finfo(dtype).eps / 2


def smallest_half_step(dtype):
    """Half the spacing of the type's subnormals: what rounding may cost next to zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def power_of_two(k):
    """2^k in 64 bits, to the bit (`pow` on a GPU is off by a unit for some k)."""
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def groups_of(v):
    """(rows, groups, 32) of a matrix, padded with zeros."""
    rows, cols = v.shape
    g = -(-cols // GROUP)
    out = torch.zeros((rows, g * GROUP), dtype=v.dtype)
    out[:, :cols] = v
    return out.view(rows, g, GROUP)


def encode(x, dtype):
    """(codes, exponent bytes) of a 64-bit matrix, exactly by the definition."""
    v = groups_of(x.double())
    bad = ~torch.isfinite(v).all(dim=2)
    v = torch.where(bad.unsqueeze(2), torch.zeros_like(v), v)
    amax = v.abs().amax(dim=2)
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    k = torch.where(mantissa * 128 >= 127.5, exponent - 6, exponent - 7).clamp(*RANGE[dtype])
    codes = (v / power_of_two(k).unsqueeze(2)).round().clamp(-127, 127)
    e = k + 127
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    e = torch.where(bad, torch.full_like(e, 255), e)
    return codes.view(x.shape[0], -1).to(torch.int8), e.to(torch.uint8)


def units(exponents):
    """2^(e - 127) for every group."""
    return power_of_two(exponents.to(torch.int64) - 127)


def decode(codes, exponents, cols):
    """64-bit values of codes and exponent bytes."""
    e = exponents.to(torch.int64)
    unit = units(exponents)
    unit = torch.where(e == 0, torch.zeros_like(unit), unit)
    unit = torch.where(e == 255, torch.full_like(unit, float("nan")), unit)
    return codes.double()[:, :cols] * unit.repeat_interleave(GROUP, dim=1)[:, :cols]


def depth(n):
    """Most additions one term goes through when n terms are added by at least 32 lanes in order and a tree over them."""
    return n / 32 + 16
