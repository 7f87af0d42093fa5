"""Rotary positions in 64 bits, as products of complex numbers, and how far a result may be off."""

from __future__ import annotations

import torch


def plain_turn(x, positions, frequencies, interleaved, magnitude=1.0, inverse=False):
    n = frequencies.numel()
    out = x.detach().double().cpu().clone()
    angle = positions.cpu().double()[:, None] * frequencies.cpu().double()
    by = torch.polar(torch.full_like(angle, magnitude), -angle if inverse else angle)[:, None]
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    turned = torch.complex(out[..., first], out[..., second]) * by
    out[..., first], out[..., second] = turned.real, turned.imag
    return out


def assert_turned(got, want, x, pairs, magnitude=1.0):
    """Half a step of the type, and in front of it, relative to m (|a| + |b|): sine and cosine rounded to 32 bits (2^-24
    each, doubled for a function that is off by one step and once more for the multiplication by m), two products and
    their sum (3 * 2^-24), the angle (2^-52 of up to 2^31 turns is 2^-21 turns; 2^-53 of them in the 64-bit result too).
    What is not turned is the same."""
    got, size = got.detach().double().cpu(), x.detach().double().cpu().abs()
    assert torch.equal(got[..., 2 * pairs:], want[..., 2 * pairs:])
    largest = 2 * size[..., :2 * pairs].amax(-1, keepdim=True) if pairs else 0.0
    eps = torch.finfo(x.dtype).eps / 2
    # float64 stays in 64 bits, with the angle's error alone
    steps = 2.0**-50 if x.dtype == torch.float64 else 7 * 2.0**-24
    allowed = eps * want.abs() * (1 + 2.0**-8) + abs(magnitude) * largest * (steps + 8 * 2.0**-21) + float(
        torch.finfo(x.dtype).smallest_normal) * torch.finfo(x.dtype).eps
    error = (got - want).abs()
    assert got.isfinite().all() and (error <= allowed).all(), float((error / allowed).max())
