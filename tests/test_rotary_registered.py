"""The registered operator of rotary positions, whose gradient torch finds by itself: its plan and its refusals, with the CPU
composition in the kernel's place."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from autosage_amd import rotary


@pytest.fixture(scope="module")
def operator():
    schema, impl = rotary.SCHEMAS["rotary_positions"]
    library = torch.library.Library("autosage_rotary_test", "DEF")
    library.define(schema)
    library.impl("rotary_positions", impl, "CPU")
    torch.library.register_autograd("autosage_rotary_test::rotary_positions", rotary._backward,
                                    setup_context=rotary._setup, lib=library)
    yield torch.ops.autosage_rotary_test.rotary_positions
    library._destroy()


@pytest.fixture(autouse=True)
def _kernel(monkeypatch):
    def kernel(query, key, positions, frequencies, interleaved, magnitude, inverse):
        # what the kernel reads through a pointer
        assert positions.dtype == torch.long and positions.is_contiguous()
        assert frequencies.dtype == torch.float64 and frequencies.is_contiguous()
        some = key if query is None else query
        turned = rotary._cpu_rotary(some if query is None else query, key, positions,
                                    -frequencies if inverse else frequencies, interleaved, magnitude)
        return None if query is None else turned[0], turned[1]

    monkeypatch.setattr(rotary, "rotary_positions_impl", kernel)


def _positions(kind):
    at = torch.tensor([5, 0, 9, 100, 7])
    return {"as they are": at, "32 bits": at.int(), "a column": torch.stack((at, at + 1), 1)[:, 0],
            "one for all": at[:1].expand(5), "a column of 32 bits": torch.stack((at, at + 1), 1).int()[:, 0]}[kind]


def _frequencies(kind):
    f = autosage_amd.rotary_frequencies(8)
    return {"as they are": f, "32 bits": f.float(), "a column": torch.stack((f, f / 2), 1)[:, 0],
            "one for all": f[1:2].expand(4)}[kind]


@pytest.mark.parametrize("at", ["as they are", "32 bits", "a column", "one for all", "a column of 32 bits"])
@pytest.mark.parametrize("angles", ["as they are", "32 bits", "a column", "one for all"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_the_gradient_takes_the_plan_of_the_forward_call(operator, at, angles, interleaved):
    positions, frequencies = _positions(at), _frequencies(angles)
    query = torch.randn(5, 3, 10, dtype=torch.float64, requires_grad=True)
    key = torch.randn(5, 1, 10, dtype=torch.float64, requires_grad=True)
    out = operator(query, key, positions, frequencies, interleaved, 0.5)
    want = autosage_amd.rotary_positions(query, key, positions, frequencies, interleaved=interleaved, magnitude=0.5)
    grads = [torch.randn(t.shape, dtype=t.dtype, requires_grad=True) for t in out]
    got = torch.autograd.grad(out, (query, key), grads, create_graph=True)
    same = torch.autograd.grad(want, (query, key), grads, create_graph=True)
    # linear: the gradient's gradient is a turn of what comes in
    again, more = (torch.autograd.grad(t, grads, (query.detach(), key.detach())) for t in (got, same))
    for a, b in zip((*out, *got, *again), (*want, *same, *more)):
        assert torch.allclose(a, b, rtol=0, atol=1e-13)


def test_positions_that_change_behind_the_call(operator):
    """A gradient is that of the call's own positions, or an error: never that of others."""
    for kind in ("as they are", "32 bits"):
        positions = _positions(kind).clone()
        query = torch.randn(5, 3, 8, dtype=torch.float64, requires_grad=True)
        out, _ = operator(query, None, positions, autosage_amd.rotary_frequencies(8))
        grad = torch.randn_like(out)
        want, = torch.autograd.grad(out, query, grad, retain_graph=True)
        positions.add_(1)
        try:
            got, = torch.autograd.grad(out, query, grad)
        except RuntimeError as error:
            assert "modified by an inplace operation" in str(error)
        else:
            assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32])
@pytest.mark.parametrize("trained", [False, True])
def test_frequencies_have_no_gradient(operator, dtype, trained):
    """Refused as by the public call, whether or not the rows are trained as well."""
    query = torch.randn(5, 3, 8, dtype=torch.float64, requires_grad=trained)
    frequencies = autosage_amd.rotary_frequencies(8).to(dtype).requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient for frequencies"):
        operator(query, None, _positions("as they are"), frequencies)
    with torch.no_grad():
        out, _ = operator(query, None, _positions("as they are"), frequencies)
    assert not out.requires_grad
    out, _ = operator(query, None, _positions("as they are"), frequencies.detach())
    assert out.requires_grad == trained
