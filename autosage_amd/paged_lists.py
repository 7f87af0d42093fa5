"""Page lists of a batch whose sequences come, grow, shrink and go.

The paged cache (``autosage_amd.paged``) reads which pages a sequence has from a
list.  ``paged_cache_resize`` keeps these lists: it takes pages for new tokens from
a stack of free ones, gives back those of tokens that are dropped, and says where
the new tokens belong.  What it returns is what the other operators of the cache
and ``rotary_positions`` take, and everything stays on the device, so that a step
can be captured while its sequences change.

CPU tensors run the same steps one after another.  The reference has no
counterpart.
"""

from __future__ import annotations

import torch

from . import _env
from . import _native
from .ops import load_native, native_load_error

_INTEGERS = (torch.int32, torch.int64)
_MOST_TOKENS = 2**40  # larger lengths and changes count as this


def _require(condition: bool, error: type, message: str) -> None:
    if not condition:
        raise error(message)


def _check(page_table, lengths, change, free_pages, free_count, page_size: int, tokens: int) -> None:
    # everything at once; the conditions run one by one only where something is wrong
    if (page_table.dtype is torch.long and page_table.dim() == 2 and free_pages.dtype is torch.long
            and free_pages.dim() == 1 and free_count.dtype is torch.long and free_count.numel() == 1
            and lengths.dtype is torch.long and change.dtype is torch.long
            and lengths.shape == change.shape == page_table.shape[:1]
            and page_table.is_contiguous() and free_pages.is_contiguous()
            and page_table.device == lengths.device == change.device == free_pages.device == free_count.device
            and page_size >= 1 and tokens >= 0
            and page_table.size(1) * page_size <= _MOST_TOKENS // 2):
        return
    for name, t in (("page_table", page_table), ("free_pages", free_pages), ("free_count", free_count)):
        _require(t.dtype == torch.long, TypeError, f"{name} must use torch.long: it is changed in place")
    for name, t in (("lengths", lengths), ("change", change)):
        _require(t.dtype in _INTEGERS, TypeError, f"{name} must use integers")
    _require(page_table.ndim == 2, ValueError, "page_table must have shape [sequences, pages]")
    for name, t in (("lengths", lengths), ("change", change)):
        _require(t.shape == page_table.shape[:1], ValueError, f"{name} must contain one entry per sequence")
    _require(free_pages.ndim == 1, ValueError, "free_pages must be one-dimensional")
    _require(free_count.numel() == 1, ValueError, "free_count must contain one entry")
    _require(page_table.size(1) <= 1 or page_table.stride(1) == 1, ValueError,
             "the rows of page_table must be contiguous")
    _require(page_table.size(0) <= 1 or page_table.size(1) == 0 or page_table.stride(0) >= page_table.size(1),
             ValueError, "the rows of page_table must not share entries")
    _require(free_pages.numel() <= 1 or free_pages.stride(0) == 1, ValueError, "free_pages must be contiguous")
    for name, t in (("lengths", lengths), ("change", change), ("free_pages", free_pages), ("free_count", free_count)):
        _require(t.device == page_table.device, ValueError, f"{name} must be on the device of page_table")
    _require(page_size >= 1, ValueError, "page_size must be positive")
    _require(tokens >= 0, ValueError, "tokens must not be negative")
    _require(page_table.size(1) * page_size <= _MOST_TOKENS // 2, ValueError,
             "a list must have room for less than 2^39 tokens")


def _validate(page_table, lengths, change, free_pages, free_count, page_size: int) -> None:
    """``AUTOSAGE_VALIDATE=1``."""
    room = page_table.size(1)
    bad = ((lengths < 0) | (lengths > room * page_size)).any()
    _require(not bool(bad), ValueError, "invalid lengths: they must lie in [0, pages of a list * page_size]")
    count = int(free_count.reshape(-1)[0])
    _require(0 <= count <= free_pages.numel(), ValueError, "invalid free_count: it must lie in [0, size of free_pages]")
    lengths = lengths.long()
    after = (lengths + change.long().clamp(-_MOST_TOKENS, 0)).clamp_min(0)
    back = ((lengths + page_size - 1) // page_size - (after + page_size - 1) // page_size).sum()
    _require(count + int(back) <= free_pages.numel(), ValueError,
             "invalid free_count: the pages that go back pass the end of free_pages")


def _cpu_resize(page_table, lengths, change, free_pages, free_count, page_size: int, tokens: int):
    sequences, room = page_table.shape
    stack = free_pages.numel()
    count = min(max(int(free_count.reshape(-1)[0]), 0), stack)
    length = [min(max(int(n), 0), _MOST_TOKENS) for n in lengths]
    step = [min(max(int(n), -_MOST_TOKENS), _MOST_TOKENS) for n in change]
    held = [min(-(-n // page_size), room) for n in length]
    after = [max(n + c, 0) for n, c in zip(length, step)]
    back = [(b, e) for b in range(sequences) if step[b] < 0
            for e in range(min(-(-after[b] // page_size), held[b]), held[b])]
    for k, (b, e) in enumerate(back):
        at = count + len(back) - 1 - k
        if at < stack:
            free_pages[at] = page_table[b, e]
        page_table[b, e] = -1
    top = min(count + len(back), stack)
    needed = taken = 0
    served = []
    for b in range(sequences):
        pages = -(-after[b] // page_size)
        need = max(pages - held[b], 0) if step[b] > 0 and pages <= room else 0
        served.append(step[b] <= 0 or (pages <= room and (need == 0 or needed + need <= top)))
        if served[b] and need > 0:
            for k in range(need):
                page_table[b, held[b] + k] = free_pages[top - 1 - needed - k]
            taken = needed + need
        needed += need
    free_count.fill_(top - taken)
    new_lengths = torch.tensor([a if s else n for a, s, n in zip(after, served, length)], dtype=torch.long)
    token_ptr = torch.tensor([0] + [max(c, 0) for c in step], dtype=torch.long).cumsum(0)
    positions = torch.full((tokens,), -1, dtype=torch.long)
    slots = torch.full((tokens,), -1, dtype=torch.long)
    for b in range(sequences):
        first = int(token_ptr[b])
        n = min(max(step[b], 0), tokens - first)
        if served[b] and n > 0:
            position = torch.arange(length[b], length[b] + n)
            page = page_table[b, position // page_size]
            positions[first:first + n] = position
            slots[first:first + n] = torch.where(page < 0, -1, page * page_size + position % page_size)
    return new_lengths, token_ptr, positions, slots


def _long(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.long and t.is_contiguous() else t.to(torch.long).contiguous()


def paged_cache_resize_impl(page_table, lengths, change, free_pages, free_count, page_size, tokens):
    page_size, tokens = int(page_size), int(tokens)
    _check(page_table, lengths, change, free_pages, free_count, page_size, tokens)
    if _env.get("AUTOSAGE_VALIDATE") == "1":
        _validate(page_table, lengths, change, free_pages, free_count, page_size)
    if not page_table.is_cuda:
        return _cpu_resize(page_table, lengths, change, free_pages, free_count, page_size, tokens)
    if not load_native():
        raise RuntimeError(f"AutoSAGE CUDA extension is unavailable: {native_load_error()}")
    lib = _native.library()
    lengths, change = _long(lengths), _long(change)
    sequences, room = page_table.shape
    device = page_table.device
    new_lengths = torch.empty(sequences, dtype=torch.long, device=device)
    token_ptr = torch.empty(sequences + 1, dtype=torch.long, device=device)
    positions = torch.empty(tokens, dtype=torch.long, device=device)
    slots = torch.empty(tokens, dtype=torch.long, device=device)
    # the kernel writes behind torch's back
    torch.autograd.graph.increment_version([page_table, free_pages, free_count])
    ws_bytes = lib.as_paged_cache_resize_workspace_bytes(sequences)
    ws = _native._workspace(ws_bytes, device)
    with _native._on(device):
        status = lib.as_paged_cache_resize(
            page_table.data_ptr(), page_table.stride(0), room, lengths.data_ptr(), change.data_ptr(),
            free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(), page_size, new_lengths.data_ptr(),
            token_ptr.data_ptr(), positions.data_ptr(), slots.data_ptr(), sequences, tokens, ws.data_ptr(), ws_bytes,
            _native._stream(device))
    _native._raise(status, "autosage::paged_cache_resize")
    return new_lengths, token_ptr, positions, slots


def paged_cache_resize(page_table, lengths, change, free_pages, free_count, *, page_size: int, tokens: int):
    """(new_lengths, token_ptr, positions, slots) of sequences that grow or shrink;
    ``page_table``, ``free_pages`` and ``free_count`` are changed in place.

    Sequence ``b`` has ``lengths[b]`` tokens in the pages ``page_table[b, :ceil(lengths[b] /
    page_size)]``, pages of its own.  ``change[b]`` new tokens come, or, where it is negative, the last
    ``-change[b]`` go (all of them where there are fewer).  Pages are taken from the end of
    ``free_pages[:free_count]`` and go back there; entries of the table that a sequence
    gives up become -1, and so should be those that it never had.  All pages that go back
    do so first, and in the order in which the same growth would take them, so that a
    drop undoes a growth.

    Sequences are served in their order while the free pages last: the first one that
    needs more than are left, those behind it that need any, and one whose list has no
    room keep their length.  ``new_lengths`` says so.

    ``token_ptr`` ``[sequences + 1]`` holds the sums of the positive changes, also of sequences
    that are not served: where the rows of the new tokens stand in a call of
    ``paged_cache_write`` with ``start=lengths``.  ``tokens`` is the number of these rows (more are
    padding); ``positions`` says which token of its sequence each is, for
    ``rotary_positions``, and ``slots`` its page times ``page_size`` plus its place there.  Both are -1
    for padding and for sequences that are not served.

    Rows stand one behind the other and sequences without a new token have none, but
    ``paged_attention`` takes a query for every sequence: of queries that come as such rows
    ``query[(token_ptr[1:] - 1).clamp(0, tokens - 1)]`` answers the sequences that grew, and the
    results of all others belong to no query of theirs.

    ``page_table.view(-1)`` with ``page_ptr = arange(sequences + 1) * page_table.size(1)`` are the
    page lists of the cache's other calls."""
    return paged_cache_resize_impl(page_table, lengths, change, free_pages, free_count, page_size, tokens)


SCHEMAS = {
    "paged_cache_resize": (
        "paged_cache_resize(Tensor(a!) page_table, Tensor lengths, Tensor change, Tensor(b!) free_pages, "
        "Tensor(c!) free_count, int page_size, int tokens) -> (Tensor, Tensor, Tensor, Tensor)",
        paged_cache_resize_impl,
    ),
}

__all__ = ["paged_cache_resize"]
