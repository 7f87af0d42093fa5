"""Rotary positions in float32, bounded pair by pair: positions of up to 5,500 leave the angle no error that counts, so that
what is allowed is what the arithmetic of 32 bits takes."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu
from tests.rotary_common import plain_turn
from tests.test_gpu_rotary import SHAPES, _frequencies, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _assert_near(got, want, x, pairs, interleaved, magnitude):
    """Of each pair (a, b), relative to magnitude * (|a| + |b|), in units of 2^-24: an eighth of a turn rounded (0.8), a sine
    that is two steps off (2), its product with the magnitude (1), two products and a sum (2), the magnitude itself (1).
    The angle: three roundings of 2^-53 of at most 880 turns, and one of 5,500 radians in the 64-bit result, are below 0.01."""
    first, second = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else
                     (slice(0, pairs), slice(pairs, 2 * pairs)))
    size = x.double().abs()
    size = size[..., first] + size[..., second]
    got = got.double().cpu()
    for part in (first, second):
        error = (got[..., part] - want[..., part]).abs()
        assert (error <= 6.81 * 2.0**-24 * abs(magnitude) * size).all(), float((error / size).max() * 2.0**24 / abs(magnitude))
    assert torch.equal(got[..., 2 * pairs:], x.double()[..., 2 * pairs:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width, pairs", SHAPES)
@pytest.mark.parametrize("magnitude", [1.0, 1.2079])
def test_widths(interleaved, width, pairs, magnitude):
    query, key, positions = _inputs(23, 3, 2, width, torch.float32, width + pairs)
    f = _frequencies(pairs)
    grads = [torch.randn(t.shape, generator=torch.Generator().manual_seed(pairs)) for t in (query, key)]
    leaves = [t.cuda().requires_grad_() for t in (query, key)]
    out = autosage_amd.rotary_positions(*leaves, positions.cuda(), f.cuda(), interleaved=interleaved, magnitude=magnitude)
    back = torch.autograd.grad(out, leaves, [g.cuda() for g in grads])
    for x, y, g, z in zip((query, key), out, grads, back):
        _assert_near(y.detach(), plain_turn(x, positions, f, interleaved, magnitude), x, pairs, interleaved, magnitude)
        _assert_near(z, plain_turn(g, positions, f, interleaved, magnitude, inverse=True), g, pairs, interleaved, magnitude)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width, pairs", [(64, 32), (40, 9), (64, 8), (80, 40), (1001, 333)])
def test_strides(interleaved, width, pairs):
    query, key, positions = _inputs(300, 6, 2, width, torch.float32, 7)
    f = _frequencies(pairs)
    wide = torch.cat((query, key, key), 1).cuda()
    spread = torch.stack((wide, wide + 1), -1)[..., 0]
    for rows in (wide, spread, wide.transpose(0, 1).contiguous().transpose(0, 1)):
        got = autosage_amd.rotary_positions(rows[:, :6], rows[:, 6:8], positions.cuda(), f.cuda(), interleaved=interleaved)
        for x, y in zip((query, key), got):
            _assert_near(y, plain_turn(x, positions, f, interleaved), x, pairs, interleaved, 1.0)


def test_the_angle_far_away():
    """2^-51 of the turns is what the angle may be off: three roundings of 2^-53, of the position times 1 / (2 pi) times the
    frequency.  Frequencies of which a position's turns are known in integers: 2 pi / 7."""
    f = torch.tensor([2.0 * torch.pi / 7], dtype=torch.float64)
    ones = torch.tensor([1.0, 0.0]).expand(64, 1, 2)
    for power in (10, 20, 24, 28, 31, 40, 50):
        positions = 2**power + torch.arange(64)
        got, _ = autosage_amd.rotary_positions(ones.cuda(), None, positions.cuda(), f.cuda())
        angle = (positions % 7).double() * (2 * torch.pi / 7)
        want = torch.stack((angle.cos(), angle.sin()), -1)[:, None]
        # the frequency itself is 2 pi / 7 to half a step: one rounding more
        turns = positions.double() / 7
        allowed = 6.81 * 2.0**-24 + 2 * torch.pi * 4 * 2.0**-53 * turns[:, None, None]
        assert ((got.double().cpu() - want).abs() <= allowed).all(), power
