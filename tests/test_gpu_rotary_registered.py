"""The registered operator of rotary positions on the GPU: gradients of plans that it converts."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at", ["32 bits", "a column", "one for all"])
@pytest.mark.parametrize("angles", ["64 bits", "32 bits", "a column"])
def test_gradients_of_converted_plans(dtype, at, angles):
    """Those of the public call, whose plan is converted once in front of both directions."""
    gen = torch.Generator().manual_seed(1)
    positions = torch.randint(0, 5000, (70,), generator=gen).cuda()
    positions = {"32 bits": positions.int(), "a column": torch.stack((positions, positions + 1), 1)[:, 0],
                 "one for all": positions[:1].expand(70)}[at]
    f = autosage_amd.rotary_frequencies(48, device="cuda")
    f = {"64 bits": f, "32 bits": f.float(), "a column": torch.stack((f, f / 2), 1)[:, 0]}[angles]
    query, key = (torch.randn(70, heads, 64, generator=gen).to(dtype).cuda().requires_grad_() for heads in (6, 2))
    grads = [torch.randn(t.shape, generator=gen).to(dtype).cuda().requires_grad_() for t in (query, key)]
    own = torch.ops.autosage.rotary_positions(query, key, positions, f, True, 1.25)
    want = autosage_amd.rotary_positions(query, key, positions, f, interleaved=True, magnitude=1.25)
    found = []
    for out in (own, want):
        first = torch.autograd.grad(out, (query, key), grads, create_graph=True)
        found.append((*out, *first, *torch.autograd.grad(first, grads, (query.detach(), key.detach()))))
    assert all(torch.equal(a, b) for a, b in zip(*found))


@pytest.mark.parametrize("trained", [False, True])
def test_frequencies_have_no_gradient(trained):
    query = torch.randn(70, 6, 64, device="cuda", requires_grad=trained)
    frequencies = autosage_amd.rotary_frequencies(48, device="cuda").requires_grad_()
    positions = torch.arange(70, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient for frequencies"):
        torch.ops.autosage.rotary_positions(query, None, positions, frequencies)
    with torch.no_grad():
        out, _ = torch.ops.autosage.rotary_positions(query, None, positions, frequencies)
    assert torch.equal(out, autosage_amd.rotary_positions(query.detach(), None, positions, frequencies.detach())[0])


def test_batches_of_none():
    query, positions = torch.randn(0, 7, 3, 24, device="cuda"), torch.zeros(0, 7, dtype=torch.long, device="cuda")
    f, one = autosage_amd.rotary_frequencies(16, device="cuda"), torch.randn(7, 3, 24, device="cuda")
    rows = torch.vmap(lambda q: autosage_amd.rotary_positions(q, None, torch.arange(7, device="cuda"), f)[0])(query)
    places = torch.vmap(lambda p: autosage_amd.rotary_positions(one, one, p, f))(positions)
    assert rows.shape == (0, 7, 3, 24) and all(t.shape == (0, 7, 3, 24) and t.is_cuda for t in places)
