"""Page lists on the GPU against plain Python."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu
from tests.paged_lists_common import assert_resized, batch, plain_resize, tensors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _resize(case, page_size):
    own = tensors(case, "cuda")
    table, lengths, change, free, count, tokens = own
    got = autosage_amd.paged_cache_resize(table, lengths, change, free, count, page_size=page_size, tokens=tokens)
    assert_resized(own, got, plain_resize(*case[:5], page_size, tokens))


@pytest.mark.parametrize("sequences, room, page_size", [(1, 1, 1), (1, 9, 4), (5, 6, 16), (20, 12, 3), (64, 5, 8),
                                                        (64, 40, 16), (300, 7, 5), (1023, 3, 16), (1024, 3, 16),
                                                        (1025, 3, 16), (5000, 3, 4)])
@pytest.mark.parametrize("spare", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("seed", range(3))
def test_resize(sequences, room, page_size, spare, seed):
    _resize(batch(sequences, room, page_size, seed, spare=spare), page_size)


@pytest.mark.parametrize("sequences, room, page_size, most", [(3, 700, 64, 40000), (40, 300, 16, 4000), (9, 5000, 1, 3000),
                                                              (3000, 8, 16, 60), (16384, 4, 16, 5), (1, 3000, 12, 36000)])
@pytest.mark.parametrize("spare", [0.6, 1.0])
def test_many_tokens(sequences, room, page_size, most, spare):
    _resize(batch(sequences, room, page_size, 5, spare=spare, grow=0.8, drop=0.1, most=most), page_size)


@pytest.mark.parametrize("sequences, room", [(9, 4000), (40, 819), (40, 820), (1024, 32), (1024, 33)])
def test_lists_with_room_for_many_pages(sequences, room):
    """Some of them end, while the others get a token or none."""
    _resize(batch(sequences, room, 4, 12, spare=0.7, grow=0.4, drop=0.3, most=1), 4)


@pytest.mark.parametrize("sequences, most", [(12, 16), (500, 3), (12, 3000)])
def test_everything_comes_and_goes(sequences, most):
    """All sequences grow, all shrink to nothing, and the pages go round; a drop undoes a growth."""
    case = batch(sequences, 200, 16, 6, grow=1.0, drop=0.0, spare=1.0, most=most)
    own = tensors(case, "cuda")
    table, lengths, change, free, count, tokens = own
    before = [t.clone() for t in own[:-1]]
    grown, *_ = autosage_amd.paged_cache_resize(table, lengths, change, free, count, page_size=16, tokens=tokens)
    back, *_ = autosage_amd.paged_cache_resize(table, grown, lengths - grown, free, count, page_size=16, tokens=0)
    assert torch.equal(back, lengths) and all(torch.equal(a, b) for a, b in zip(own[:-1], before))
    none, *_ = autosage_amd.paged_cache_resize(table, lengths, torch.full_like(lengths, -(2**62)), free, count,
                                               page_size=16, tokens=0)
    total = int(before[4]) + int(((lengths + 15) // 16).sum())
    assert not none.any() and (table == -1).all() and int(count) == total
    assert sorted(free[:total].tolist()) == list(range(total))


def test_numbers_that_do_not_fit():
    """As on the CPU, and the guards around the tensors stay."""
    guard = torch.full((3, 4), -5)
    guard[:, :2] = torch.tensor([[3, 4], [5, -1], [2**40, -1]])
    stack = torch.tensor([-9, 0, 1, 2, -9])
    for lengths, change, count in [([2**62, -9, 3], [2**62, 2**62, -(2**62)], 99), ([8, 4, 0], [-8, -1, 5], 3),
                                   ([8, 4, 9], [-(2**63), -4, -9], -4), ([8, 4, 3], [0, 4, 5], 2), ([2, 2, 2], [9, 0, 9], 3)]:
        results = []
        for device in ("cpu", "cuda"):
            whole, free = guard.to(device, copy=True), stack.to(device, copy=True)
            n, c, k = (torch.tensor(x, device=device) for x in (lengths, change, [count]))
            got = autosage_amd.paged_cache_resize(whole[:, :2], n, c, free[1:4], k, page_size=4, tokens=4)
            results.append([t.cpu() for t in (*got, whole, free, k)])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        assert (results[1][4][:, 2:] == -5).all() and (results[1][5][[0, 4]] == -9).all()


@pytest.mark.parametrize("sequences, most", [(6, 40), (2000, 30)])
def test_more_and_fewer_rows_than_tokens(sequences, most):
    case = batch(sequences, 20, 8, 7, spare=1.0, most=most)
    for tokens in (0, 1, case[5] // 2, case[5] + 5000):
        _resize((*case[:5], tokens), 8)


def test_the_registered_operator_32_bit_numbers_and_versions(monkeypatch):
    monkeypatch.setenv("AUTOSAGE_VALIDATE", "1")
    case = batch(9, 8, 4, 8)
    case[2][:] = [max(c, -999) for c in case[2]]
    own = tensors(case, "cuda")
    table, lengths, change, free, count, tokens = own
    versions = [t._version for t in (table, free, count)]
    free_room = torch.cat((free, free))  # validation: all that goes back has to fit
    got = torch.ops.autosage.paged_cache_resize(table, lengths.int(), change.int(), free_room, count, 4, tokens)
    assert_resized((table, lengths, change, free_room[:free.numel()], count, tokens), got,
                   plain_resize(*case[:5], 4, tokens))
    assert table._version > versions[0] and count._version > versions[2]
    count.fill_(10**6)
    with pytest.raises(ValueError, match="invalid free_count"):
        autosage_amd.paged_cache_resize(table, lengths, change, free, count, page_size=4, tokens=tokens)


@pytest.mark.parametrize("sequences, most", [(7, 9), (1500, 20)])
def test_capture_and_replay(sequences, most):
    """Two graphs of one batch, replayed in turn while the changes change; every replay against an eager call."""
    case = batch(sequences, 30, 8, 9, grow=1.0, drop=0.0, spare=3.0, most=most)
    table, lengths, change, free, count, tokens = own = tensors(case, "cuda")
    others = [t.clone() for t in own[:-1]]

    def step(table, lengths, change, free, count):
        got = autosage_amd.paged_cache_resize(table, lengths, change, free, count, page_size=8, tokens=tokens)
        lengths.copy_(got[0])
        return got

    step(*own[:-1])
    step(*others)
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step(*own[:-1]))
        graphs.append(graph)
    torch.cuda.synchronize()
    gen = torch.Generator(device="cuda").manual_seed(10)
    for turn in range(8):
        change.copy_(torch.randint(-most, most + 1, change.shape, generator=gen, device="cuda"))
        others[2].copy_(change)
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        want = step(*others)
        assert all(torch.equal(a, b) for a, b in zip(results[turn % 2], want))
        assert all(torch.equal(a, b) for a, b in zip(own[:-1], others))


def test_two_batches_on_two_streams():
    cases = [batch(n, 40, 8, 11 + n, spare=0.8, most=200) for n in (30, 1200)]
    wants = [plain_resize(*c[:5], 8, c[5]) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        owns = [tensors(c, "cuda") for c in cases]
        torch.cuda.synchronize()
        got = []
        for stream, (table, lengths, change, free, count, tokens) in zip(streams, owns):
            with torch.cuda.stream(stream):
                got.append(autosage_amd.paged_cache_resize(table, lengths, change, free, count, page_size=8, tokens=tokens))
        torch.cuda.synchronize()
        for own, g, want in zip(owns, got, wants):
            assert_resized(own, g, want)


def test_offsets_beyond_32_bits():
    """A table of more than 2^32 bytes whose last sequence grows."""
    room = 1 << 18
    table = torch.full((2100, room), -1, device="cuda")  # 4.4 GB
    lengths = torch.zeros(2100, dtype=torch.long, device="cuda")
    change = torch.zeros_like(lengths)
    change[-1] = 1000
    free, count = torch.arange(5000, device="cuda"), torch.tensor([5000], device="cuda")
    new, _, positions, slots = autosage_amd.paged_cache_resize(table, lengths, change, free, count, page_size=2, tokens=1000)
    pages = 4999 - torch.arange(500, device="cuda")
    assert int(new[-1]) == 1000 and torch.equal(table[-1, :500], pages) and int(count) == 4500
    assert torch.equal(slots, pages.repeat_interleave(2) * 2 + positions % 2)
    assert int((table != -1).sum()) == 500
