"""Rotation by positions in 64 bits, and how far a kernel's results may be from it.

Bounds count roundings, with u = 2^-24, a half step of fp32 relative to 1.  Cosine and sine are off by at most 4 u: two for the
hardware's functions (2^-23 measured), one for the rounding of their argument, at most a half as half turns (pi 2^-26), and the
argument's own part, position * 2^-52 turns; `scaling` adds another u.  A product of two fp32 values and a fused sum add 2 u.  So a rotated
channel is off by at most 8 u scaling (|x| + |x'|).  Norms: the sum of squares is off by 12 u of itself (8 in a lane, 4 across),
half of which enters the root; that, the division, the root and two products make 10 u, taken as 16.  FWHT-128: seven sums of
growing terms and one product, 8 u of sum |y| / sqrt(128), beside the mean-square growth of what is there, at most sum of the
errors / sqrt(128).  The result's own rounding is h = finfo(dtype).eps / 2 of it, for fp16 at least 2^-25 (half a subnormal
step).
"""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U = 2.0 ** -24


def axes_of(sections, interleaved):
    """The axis of each pair."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [i % 3 if i % 3 < len(sections) and i < 3 * sections[i % 3] else 0 for i in range(64)]


def hadamard(device):
    h = torch.ones(1, 1, dtype=torch.float64, device=device)
    while h.shape[0] < 128:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    return h / math.sqrt(128.0)


def rotate(x, positions, rotary, weight=None, apply_hadamard=False):
    """(result, bound) in 64 bits of x [B, H, S, 128] with positions [axes, B, S]."""
    dtype, x = x.dtype, x.double()
    err = torch.zeros_like(x)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + rotary.eps) * weight.double()
        err = 16 * U * x.abs()
    pos = positions[torch.tensor(axes_of(rotary.mrope_section, rotary.interleaved), device=x.device)].permute(1, 2, 0)[:, None].double()
    freq = rotary.inv_freq.double()
    angle = pos * freq
    far = 2.0 ** -51 * angle.abs() * 2  # the angle's own rounding, here and there
    c, s = torch.cos(angle) * rotary.scaling, torch.sin(angle) * rotary.scaling
    a, b = x[..., :64], x[..., 64:]
    y = torch.cat((a * c - b * s, b * c + a * s), -1)
    size = (a.abs() + b.abs()) * abs(rotary.scaling)
    err = (err[..., :64] + err[..., 64:]) * abs(rotary.scaling) + size * (8 * U + far)
    err = torch.cat((err, err), -1)
    if apply_hadamard:
        h = hadamard(x.device)
        err = err @ h.abs() + 8 * U * (y.abs() @ h.abs())
        y = y @ h
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    return y, err * (1 + 2 * HALF[dtype]) + HALF[dtype] * y.abs() + least
