"""The operators of a serving loop together: pages for new tokens, rotary positions, the cache's write, attention."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu
from tests.paged4_common import E2M1, E8M0, quantised_pairs
from tests.paged_common import assert_attention, plain_attention
from tests.rotary_common import plain_turn

pytestmark = pytest.mark.gpu

HEADS, GROUP, WIDTH, PAGE, ROOM = 2, 4, 64, 16, 12


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


class Server:
    """A batch of places for sequences over a cache of 4-bit (or 16-bit) pages."""

    def __init__(self, places, pages, quantised):
        dev = {"device": "cuda"}
        self.quantised = quantised
        if quantised:
            self.pages = [torch.full((pages, HEADS, PAGE, WIDTH // 2), 255, dtype=torch.uint8, **dev).view(E2M1) for _ in range(2)]
            self.exponents = {kind + "_exponents": torch.full((pages, HEADS, PAGE, WIDTH // 32), 255, dtype=torch.uint8,
                                                              **dev).view(E8M0) for kind in ("key", "value")}
        else:
            self.pages = [torch.full((pages, HEADS, PAGE, WIDTH), float("nan"), dtype=torch.bfloat16, **dev) for _ in range(2)]
            self.exponents = {}
        self.table = torch.full((places, ROOM), -1, **dev)
        self.page_ptr = torch.arange(places + 1, **dev) * ROOM
        self.lengths = torch.zeros(places, dtype=torch.long, **dev)
        self.free, self.count = torch.arange(pages, **dev), torch.tensor([pages], **dev)
        self.frequencies = autosage_amd.rotary_frequencies(32, device="cuda")

    def add(self, change, rows):
        """Rows of new queries, keys and values, ``[tokens, GROUP * HEADS + 2 * HEADS, WIDTH]``; the turned queries."""
        before = self.lengths.clone()
        new, token_ptr, positions, slots = autosage_amd.paged_cache_resize(
            self.table, self.lengths, change, self.free, self.count, page_size=PAGE, tokens=rows.size(0))
        query, key = autosage_amd.rotary_positions(rows[:, :HEADS * GROUP], rows[:, HEADS * GROUP:HEADS * (GROUP + 1)],
                                                   positions, self.frequencies)
        autosage_amd.paged_cache_write(key, rows[:, HEADS * (GROUP + 1):], *self.pages, self.page_ptr,
                                       self.table.view(-1), token_ptr, before, **self.exponents)
        self.lengths.copy_(new)
        return query, key, token_ptr, positions, slots

    def step(self, change, rows):
        query, *_ = self.add(change, rows)
        return autosage_amd.paged_attention(query, *self.pages, self.page_ptr, self.table.view(-1), self.lengths,
                                            scale=WIDTH**-0.5, return_lse=True, **self.exponents)


class Plain:
    """The same with every sequence's rows in a list, in 64 bits from the turned rows on."""

    def __init__(self, places, quantised):
        self.heads, self.quantised = HEADS, quantised
        self.rows = {kind: [torch.zeros(0, HEADS, WIDTH, dtype=torch.float64) for _ in range(places)]
                     for kind in ("key", "value")}

    def add(self, b, key, value):
        for kind, x in (("key", key), ("value", value)):
            x = x.cpu()
            held = quantised_pairs(x)[0] if self.quantised else x.double()
            self.rows[kind][b] = torch.cat((self.rows[kind][b], held))

    @property
    def lengths(self):
        return [r.size(0) for r in self.rows["key"]]


def _rows(tokens, gen):
    return torch.randn(tokens, HEADS * (GROUP + 2), WIDTH, generator=gen).bfloat16()


@pytest.mark.parametrize("quantised", [False, True])
def test_sequences_come_answer_and_go(quantised):
    places, gen = 5, torch.Generator().manual_seed(1)
    server, plain = Server(places, 24, quantised), Plain(places, quantised)
    change = [40, 0, 100, 1, 17]
    for round_ in range(3):
        rows = _rows(sum(max(c, 0) for c in change) + 2, gen)
        for b, c in enumerate(change):  # what goes, goes first
            if c < 0:
                for kind in plain.rows:
                    plain.rows[kind][b] = plain.rows[kind][b][:max(0, len(plain.rows[kind][b]) + c)]
        _, key, token_ptr, positions, slots = server.add(torch.tensor(change).cuda(), rows.cuda())
        at = 0
        for b, c in enumerate(change):
            n = plain.lengths[b]
            if c > 0:
                assert positions[at:at + c].tolist() == list(range(n, n + c))
                entry = torch.arange(n, n + c).cuda()
                assert torch.equal(slots[at:at + c], server.table[b, entry // PAGE] * PAGE + entry % PAGE)
                turned = plain_turn(rows[at:at + c, HEADS * GROUP:HEADS * (GROUP + 1)], positions[at:at + c],
                                    server.frequencies, False)
                assert (key[at:at + c].double().cpu() - turned).abs().max() <= 2.0**-8 * turned.abs().max()
                plain.add(b, key[at:at + c], rows[at:at + c, HEADS * (GROUP + 1):])
                at += c
        assert server.lengths.tolist() == plain.lengths and positions[at:].tolist() == [-1, -1]
        held = sum(-(-n // PAGE) for n in plain.lengths)
        used = server.table[server.table >= 0].tolist()
        assert len(used) == held and int(server.count) == 24 - held
        assert sorted(used + server.free[:24 - held].tolist()) == list(range(24))
        for _ in range(2):
            rows = _rows(places, gen)
            query, key, _, positions, _ = server.add(torch.ones(places, dtype=torch.long).cuda(), rows.cuda())
            assert positions.tolist() == plain.lengths
            for b in range(places):
                plain.add(b, key[b:b + 1], rows[b:b + 1, HEADS * (GROUP + 1):])
            out, lse = autosage_amd.paged_attention(query, *server.pages, server.page_ptr, server.table.view(-1),
                                                    server.lengths, scale=WIDTH**-0.5, return_lse=True, **server.exponents)
            assert_attention(out, lse, plain_attention(plain, query.cpu(), WIDTH**-0.5), dtype=torch.bfloat16,
                             quantised=quantised, lse_bound=2e-4)
        change = [-(10**6), 33, -50, 5, 0] if round_ == 0 else [7, -3, -(10**6), 60, -18]


@pytest.mark.parametrize("quantised", [False, True])
def test_a_captured_step_and_a_batch_that_is_refused(quantised):
    """One graph of a whole step, replayed until pages run out; every replay against an eager step of another server."""
    places, gen = 4, torch.Generator().manual_seed(2)
    server, other = Server(places, 9, quantised), Server(places, 9, quantised)
    first = _rows(60, gen).cuda()
    for s in (server, other):
        s.add(torch.tensor([30, 0, 20, 10]).cuda(), first)
    one = torch.ones(places, dtype=torch.long, device="cuda")
    rows = _rows(places, gen).cuda()
    server.step(one, rows)
    other.step(one, rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = server.step(one, rows)
    refused = False
    for turn in range(40):
        rows.normal_()
        one.copy_(torch.tensor([1, 1, 1, -20 if turn == 30 else 1]))
        graph.replay()
        torch.cuda.synchronize()
        before = other.lengths.clone()
        want = other.step(one, rows)
        assert all(torch.equal(a, b) for a, b in zip(results, want))
        assert torch.equal(server.lengths, other.lengths) and torch.equal(server.table, other.table)
        refused = refused or bool((other.lengths == before).any())
        assert all(torch.isfinite(r).all() for r in results)
    assert refused
    for a, b in zip((*server.pages, *server.exponents.values()), (*other.pages, *other.exponents.values())):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_attention_over_edges_with_turned_rows_equals_attention_over_pages():
    """Nodes of a text that see all in front of them: rotary positions of the nodes in the graph's attention, tokens one at
    a time over 16-bit pages."""
    n, width = 40, 32
    gen = torch.Generator().manual_seed(3)
    rows = torch.randn(n, 3, width, generator=gen).cuda()
    frequencies = autosage_amd.rotary_frequencies(width, device="cuda")
    query, key = autosage_amd.rotary_positions(rows[:, :1], rows[:, 1:2], torch.arange(n).cuda(), frequencies,
                                               interleaved=True)
    crow = torch.arange(n + 1).cumsum(0).cuda()
    col = torch.cat([torch.arange(i + 1) for i in range(n)]).cuda()
    whole = autosage_amd.csr_attention_forward(crow, col, query[:, 0].contiguous(), key[:, 0].contiguous(),
                                               rows[:, 2].contiguous(), scale=width**-0.5)
    whole = whole[0] if isinstance(whole, tuple) else whole
    pages = [torch.zeros(3, 1, 16, width, device="cuda") for _ in range(2)]
    ptr, idx = torch.tensor([0, 3]).cuda(), torch.tensor([2, 0, 1]).cuda()
    for t in range(n):
        at = torch.tensor([t]).cuda()
        q, k = autosage_amd.rotary_positions(rows[t:t + 1, :1], rows[t:t + 1, 1:2], at, frequencies, interleaved=True)
        autosage_amd.paged_cache_write(k, rows[t:t + 1, 2:], *pages, ptr, idx, torch.tensor([0, 1]).cuda(), at)
        out = autosage_amd.paged_attention(q, *pages, ptr, idx, at + 1, scale=width**-0.5)
        # both are within a few fp32 roundings of the exact result
        assert torch.allclose(out[0, 0], whole[t], rtol=2.0**-20, atol=2e-5)
