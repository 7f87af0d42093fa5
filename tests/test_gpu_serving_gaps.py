"""A serving step in which some sequences have no new token: rows are packed, queries belong to sequences."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu
from tests.paged_common import assert_attention, plain_attention
from tests.test_gpu_serving_step import GROUP, HEADS, WIDTH, Plain, Server, _rows

pytestmark = pytest.mark.gpu

PLACES = 4
CHANGES = [[1, 0, 1, 1], [0, 0, 0, 1], [1, 1, 1, 1], [0, 1, 1, 0], [0, 0, 0, 0], [1, 0, 0, 0]]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _step(server, change, rows):
    query, key, token_ptr, positions, _ = server.add(change, rows)
    own = query[(token_ptr[1:] - 1).clamp(0, rows.size(0) - 1)]
    out, lse = autosage_amd.paged_attention(own, *server.pages, server.page_ptr, server.table.view(-1), server.lengths,
                                            scale=WIDTH**-0.5, return_lse=True, **server.exponents)
    return out, lse, own, key, positions


def _start(quantised):
    gen = torch.Generator().manual_seed(4)
    server, plain = Server(PLACES, 20, quantised), Plain(PLACES, quantised)
    first = _rows(60, gen)
    _, key, token_ptr, _, _ = server.add(torch.tensor([30, 1, 20, 9]).cuda(), first.cuda())
    for b in range(PLACES):
        mine = slice(int(token_ptr[b]), int(token_ptr[b + 1]))
        plain.add(b, key[mine], first[mine, HEADS * (GROUP + 1):])
    return server, plain, gen


def _answers(plain, change, rows, own, key, positions):
    """The plain rows with the step's added, and the 64-bit results of the sequences that grew."""
    at = 0
    for b in range(PLACES):
        if change[b]:
            assert int(positions[at]) == plain.lengths[b]
            plain.add(b, key[at:at + 1], rows[at:at + 1, HEADS * (GROUP + 1):])
            at += 1
    assert positions[at:].tolist() == [-1] * (PLACES - at)
    grew = torch.tensor(change, dtype=torch.bool)
    return grew, tuple(t[grew] for t in plain_attention(plain, own.cpu(), WIDTH**-0.5))


@pytest.mark.parametrize("quantised", [False, True])
def test_every_sequence_is_answered_with_its_own_query(quantised):
    server, plain, gen = _start(quantised)
    for change in CHANGES:
        rows = _rows(PLACES, gen)
        out, lse, own, key, positions = _step(server, torch.tensor(change).cuda(), rows.cuda())
        packed = autosage_amd.rotary_positions(rows[:, :HEADS * GROUP].cuda(), None, positions, server.frequencies)[0]
        at = 0
        for b in range(PLACES):
            if change[b]:
                assert torch.equal(own[b], packed[at])
                at += 1
        grew, want = _answers(plain, change, rows, own, key, positions)
        assert server.lengths.tolist() == plain.lengths
        if grew.any():
            assert_attention(out.cpu()[grew], lse.cpu()[grew], want, dtype=torch.bfloat16, quantised=quantised, lse_bound=2e-4)


@pytest.mark.parametrize("quantised", [False, True])
def test_a_captured_step_whose_gaps_move(quantised):
    server, plain, gen = _start(quantised)
    change, rows = torch.zeros(PLACES, dtype=torch.long, device="cuda"), _rows(PLACES, gen).cuda()
    _step(server, change, rows)  # nothing grows
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse, own, key, positions = _step(server, change, rows)
    for now in CHANGES:
        fresh = _rows(PLACES, gen)
        rows.copy_(fresh)
        change.copy_(torch.tensor(now))
        graph.replay()
        torch.cuda.synchronize()
        grew, want = _answers(plain, now, fresh, own, key, positions)
        assert server.lengths.tolist() == plain.lengths
        if grew.any():
            assert_attention(out.cpu()[grew], lse.cpu()[grew], want, dtype=torch.bfloat16, quantised=quantised, lse_bound=2e-4)
