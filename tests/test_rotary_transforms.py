"""torch.func's transforms of rotary positions, with the CPU composition in the kernel's place."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from autosage_amd import rotary
from tests.test_rotary_registered import _kernel  # noqa: F401


def _turn(query, key, positions, frequencies):
    """The public call of GPU tensors."""
    rotary._check(query, key, positions, frequencies)
    return rotary._turn(query, key, *rotary._plan(positions, frequencies), False, 1.25, False)


Q, K, P = torch.randn(5, 3, 10, dtype=torch.float64), torch.randn(5, 1, 10, dtype=torch.float64), torch.arange(5)
F = autosage_amd.rotary_frequencies(8)


@pytest.mark.parametrize("count", [0, 1, 3])
@pytest.mark.parametrize("dim", [0, 1, -1])
def test_batches_of_any_number(count, dim):
    """Rows, positions or frequencies of a batch, of none at all too: as a call each."""
    gen = torch.Generator().manual_seed(count)
    many = {"query": torch.randn(count, 5, 3, 10, generator=gen, dtype=torch.float64),
            "key": torch.randn(count, 5, 1, 10, generator=gen, dtype=torch.float64),
            "positions": torch.randint(0, 99, (count, 5), generator=gen),
            "frequencies": torch.rand(count, 4, generator=gen, dtype=torch.float64)}
    alone = {"query": Q, "key": K, "positions": P, "frequencies": F}
    for batched in (["query"], ["key"], ["query", "key"], ["positions"], ["frequencies"], ["query", "positions"],
                    ["key", "frequencies"]):
        def call(*args):
            return _turn(**{**alone, **dict(zip(batched, args))})

        out = torch.vmap(call, in_dims=dim)(*(many[name].movedim(0, dim) for name in batched))
        assert [t.shape for t in out] == [(count, 5, 3, 10), (count, 5, 1, 10)]
        for i in range(count):
            want = _turn(**{**alone, **{name: many[name][i] for name in batched}})
            assert all(torch.allclose(a[i], b, rtol=0, atol=1e-13) for a, b in zip(out, want))
        one = torch.vmap(lambda *args: _turn(**{**alone, "key": None, **dict(zip(batched, args))})[0], in_dims=dim)
        if "key" not in batched:
            assert torch.allclose(one(*(many[name].movedim(0, dim) for name in batched)), out[0], rtol=0, atol=1e-13)


@pytest.mark.parametrize("count", [0, 2])
@pytest.mark.parametrize("batched", ["rows", "positions"])
def test_gradients_of_batches(count, batched):
    rows, places = torch.randn(count, 5, 3, 10, dtype=torch.float64), torch.arange(5 * count).view(count, 5)

    def total(query, positions):
        return (_turn(query, None, positions, F)[0] ** 3).sum()

    dims = (0, None) if batched == "rows" else (None, 0)
    args = (rows, P) if batched == "rows" else (Q, places)
    each = torch.vmap(torch.func.grad(total), in_dims=dims)(*args)
    assert each.shape == (count, 5, 3, 10)
    for i in range(count):
        x = (rows[i] if batched == "rows" else Q).clone().requires_grad_()
        want, = torch.autograd.grad(total(x, P if batched == "rows" else places[i]), x)
        assert torch.allclose(each[i], want, rtol=0, atol=1e-12)
    # the batch inside of the gradient
    summed = torch.func.grad(lambda q: torch.vmap(total, in_dims=dims)(*((q, P) if batched == "rows" else (q, places))).sum())
    assert torch.allclose(summed(args[0]), each if batched == "rows" else each.sum(0), rtol=0, atol=1e-12)
