"""Rotary positions on the CPU."""

from __future__ import annotations

import math

import pytest
import torch

import autosage_amd
from autosage_amd import _native
from tests.rotary_common import assert_turned, plain_turn


def test_frequencies():
    f = autosage_amd.rotary_frequencies(8)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    assert torch.equal(autosage_amd.rotary_frequencies(8, scaling="linear", factor=4.0), f / 4)
    based = autosage_amd.rotary_frequencies(8, scaling="base", factor=4.0)
    assert based[0] == 1.0 and math.isclose(float(based[-1]), 0.001 / 4)
    assert torch.equal(autosage_amd.rotary_frequencies(8, base=500.0)[1:2], 500.0 ** torch.tensor([-0.25], dtype=torch.float64))
    # within 1,000 positions the pairs turn 159, 15.9, 1.59 and 0.159 times
    ramp = autosage_amd.rotary_frequencies(8, scaling="ramp", factor=4.0, original_length=1000, turns=(1.0, 16.0))
    kept = (1000 * f / (2 * math.pi) - 1) / 15
    assert ramp[0] == f[0] and ramp[3] == f[3] / 4
    for i in (1, 2):
        assert math.isclose(float(ramp[i]), float(f[i] * kept[i] + f[i] / 4 * (1 - kept[i])))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width, pairs", [(1, 0), (2, 1), (7, 3), (16, 8), (40, 10)])
def test_turn(dtype, interleaved, width, pairs):
    gen = torch.Generator().manual_seed(width)
    query, key = torch.randn(6, 3, width, generator=gen).to(dtype), torch.randn(6, 1, width, generator=gen).to(dtype)
    positions = torch.tensor([0, 1, 7, 123456, 2**31, -3])
    frequencies = autosage_amd.rotary_frequencies(2 * pairs) if pairs else torch.zeros(0, dtype=torch.float64)
    got = autosage_amd.rotary_positions(query, key, positions, frequencies, interleaved=interleaved, magnitude=1.25)
    for x, y in zip((query, key), got):
        assert_turned(y, plain_turn(x, positions, frequencies, interleaved, 1.25), x, pairs, 1.25)
    alone, none = autosage_amd.rotary_positions(query, None, positions.clone(), frequencies, interleaved=interleaved,
                                                magnitude=1.25)
    assert none is None and torch.equal(alone, got[0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_against_differences(interleaved):
    query = torch.randn(4, 2, 7, dtype=torch.float64, requires_grad=True)
    key = torch.randn(4, 1, 7, dtype=torch.float64, requires_grad=True)
    frequencies = autosage_amd.rotary_frequencies(6)

    def turn(q, k):
        return autosage_amd.rotary_positions(q, k, torch.tensor([5, 0, 9, 100]), frequencies, interleaved=interleaved,
                                             magnitude=0.7)

    assert torch.autograd.gradcheck(turn, (query, key))
    assert torch.autograd.gradgradcheck(turn, (query, key))


def test_products_depend_on_the_distance_alone():
    frequencies = autosage_amd.rotary_frequencies(16)
    q, k = torch.randn(1, 1, 16, dtype=torch.float64), torch.randn(1, 1, 16, dtype=torch.float64)

    def product(i, j):
        a, _ = autosage_amd.rotary_positions(q, None, torch.tensor([i]), frequencies)
        b, _ = autosage_amd.rotary_positions(k, None, torch.tensor([j]), frequencies)
        return float((a * b).sum())

    assert math.isclose(product(5, 3), product(1005, 1003), abs_tol=1e-9)


def test_refusals():
    q, k, p = torch.randn(4, 2, 8), torch.randn(4, 1, 8), torch.arange(4)
    f = autosage_amd.rotary_frequencies(8)
    turn, frequencies = autosage_amd.rotary_positions, autosage_amd.rotary_frequencies
    for error, call in [
        (ValueError, lambda: turn(q[0], k, p, f)),
        (ValueError, lambda: turn(q, k[0], p, f)),
        (TypeError, lambda: turn(q, k.half(), p, f)),
        (TypeError, lambda: turn(q.int(), None, p, f)),
        (ValueError, lambda: turn(q, k[:3], p, f)),
        (ValueError, lambda: turn(q, k[..., :6], p, f)),
        (ValueError, lambda: turn(q[..., :0], None, p, f[:0])),
        (TypeError, lambda: turn(q, k, p.float(), f)),
        (ValueError, lambda: turn(q, k, p[:3], f)),
        (ValueError, lambda: turn(q, k, p[None], f)),
        (TypeError, lambda: turn(q, k, p, f.half())),
        (ValueError, lambda: turn(q, k, p, f[None])),
        (ValueError, lambda: turn(q[..., :7], None, p, f)),
        (RuntimeError, lambda: turn(q, k, p, f.clone().requires_grad_())),
        (ValueError, lambda: turn(q, k.to("meta"), p, f)),
        (ValueError, lambda: turn(q, k, p.to("meta"), f)),
        (ValueError, lambda: frequencies(7)),
        (ValueError, lambda: frequencies(0)),
        (ValueError, lambda: frequencies(8, base=0.0)),
        (ValueError, lambda: frequencies(8, factor=2.0)),
        (ValueError, lambda: frequencies(8, scaling="other")),
        (ValueError, lambda: frequencies(8, scaling="ramp", factor=2.0)),
        (ValueError, lambda: frequencies(8, scaling="linear", original_length=5)),
        (ValueError, lambda: frequencies(8, scaling="ramp", original_length=5, turns=(3.0, 3.0))),
        (ValueError, lambda: frequencies(2, scaling="base", factor=2.0)),
    ]:
        with pytest.raises(error):
            call()
    with torch.no_grad():
        turn(q, k, p, f.clone().requires_grad_())


def test_no_tokens_and_names_of_both_packages():
    import autosage

    q, k = autosage.rotary_positions(torch.zeros(0, 3, 8), torch.zeros(0, 0, 8), torch.zeros(0, dtype=torch.long),
                                     autosage.rotary_frequencies(4))
    assert q.shape == (0, 3, 8) and k.shape == (0, 0, 8)
    assert {"rotary_positions", "rotary_frequencies", "paged_cache_resize"} <= set(autosage.__all__)


def test_native_argument_checks_come_before_any_launch():
    path = _native.package_library_path()
    if not path.exists():
        pytest.skip("HIP library not built")
    import ctypes

    lib = _native.open_library(path)
    two, fake = (ctypes.c_int64 * 2)(8, 4), 256

    def turn(query=fake, strides=two, out=fake, heads=2, key=fake, positions=fake, frequencies=fake, tokens=3, width=8,
             pairs=4, dtype=0):
        return lib.as_rotary_positions(query, strides, out, heads, key, two, fake, 1, positions, frequencies, tokens,
                                       width, pairs, 0, 0, 1.0, dtype, None)

    for status, call, message in [
        (1, lambda: turn(dtype=3), b"dtype must be"),
        (3, lambda: turn(tokens=-1), b"at most"),
        (3, lambda: turn(tokens=1 << 40), b"at most"),
        (1, lambda: turn(heads=65536), b"heads must lie"),
        (3, lambda: turn(width=0), b"width must lie"),
        (3, lambda: turn(width=1025), b"width must lie"),
        (1, lambda: turn(pairs=5), b"the pairs must fit"),
        (1, lambda: turn(pairs=-1), b"the pairs must fit"),
        (1, lambda: turn(query=None), b"null pointer"),
        (1, lambda: turn(strides=None), b"null pointer"),
        (1, lambda: turn(key=None), b"null pointer"),
        (1, lambda: turn(positions=None), b"null pointer"),
        (1, lambda: turn(frequencies=None), b"null pointer"),
        (1, lambda: turn(out=fake + 2), b"rows must be aligned"),
        (0, lambda: turn(tokens=0), b""),
    ]:
        assert call() == status, message
        assert lib.as_last_error().startswith(message), lib.as_last_error()


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32])
def test_frequencies_have_no_derivative(dtype):
    query = torch.randn(3, 2, 8)
    positions = torch.arange(3)
    frequencies = autosage_amd.rotary_frequencies(8).to(dtype)

    def turned(f):
        return autosage_amd.rotary_positions(query, None, positions, f)[0]

    with pytest.raises(RuntimeError, match="no gradient for frequencies"):
        turned(frequencies.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no derivative for frequencies"):
        torch.func.jvp(turned, (frequencies,), (torch.ones_like(frequencies),))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(frequencies, torch.ones_like(frequencies))
        with pytest.raises(RuntimeError, match="no derivative for frequencies"):
            turned(dual)
