"""Page lists step by step in plain Python, and batches of sequences for them."""

from __future__ import annotations

import random

import torch


def plain_resize(table, lengths, change, free, count, page_size, tokens):
    """(table, free, count, new lengths, token_ptr, positions, slots) as lists: pages go one at a time.

    Pages that go back are put on the stack from the last one of the last sequence to the first one of the first, and
    pages are popped in the order of the sequences."""
    table, free = [list(r) for r in table], list(free)
    room = len(table[0]) if table else 0
    pages = lambda n: -(-n // page_size)  # noqa: E731
    new_lengths = list(lengths)
    for b in reversed(range(len(lengths))):
        if change[b] < 0:
            new_lengths[b] = max(lengths[b] + change[b], 0)
            for e in reversed(range(pages(new_lengths[b]), pages(lengths[b]))):
                free[count] = table[b][e]
                count += 1
                table[b][e] = -1
    positions, slots, token_ptr = [], [], [0]
    refused = False
    for b, (n, c) in enumerate(zip(lengths, change)):
        token_ptr.append(token_ptr[-1] + max(c, 0))
        if c <= 0:
            continue
        need = pages(n + c) - pages(n)
        if pages(n + c) > room:
            positions += [-1] * c
            slots += [-1] * c
            continue
        if need > 0 and (refused or need > count):
            refused = True
            positions += [-1] * c
            slots += [-1] * c
            continue
        for e in range(pages(n), pages(n + c)):
            count -= 1
            table[b][e] = free[count]
        new_lengths[b] = n + c
        for p in range(n, n + c):
            positions.append(p)
            page = table[b][p // page_size]
            slots.append(-1 if page < 0 else page * page_size + p % page_size)
    positions = (positions + [-1] * tokens)[:tokens]
    slots = (slots + [-1] * tokens)[:tokens]
    return table, free, count, new_lengths, token_ptr, positions, slots


def batch(sequences, room, page_size, seed, *, spare=0.5, grow=0.5, drop=0.3, most=None):
    """(table, lengths, change, free, count, tokens): a batch of sequences with lists of ``room`` pages, some that grow (by
    ``most`` tokens at most), some that shrink, some of both to nothing, and a stack with a share ``spare`` of what they need."""
    rng = random.Random(seed)
    lengths = [rng.choice([0, 1, page_size, rng.randint(0, room * page_size)]) for _ in range(sequences)]
    change = []
    for n in lengths:
        x = rng.random()
        if x < grow:
            change.append(rng.choice([1, page_size, rng.randint(1, most or max(1, room * page_size // 2))]))
        elif x < grow + drop:
            change.append(-rng.choice([1, n + 3, max(1, n // 2), 2**61]))
        else:
            change.append(0)
    held = [-(-n // page_size) for n in lengths]
    need = sum(max(0, -(-(n + c) // page_size) - h) for n, c, h in zip(lengths, change, held) if c > 0)
    total = sum(held) + int(spare * need) + 2
    ids = list(range(total))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (room - h))
        at += h
    free = ids[at:] + [-7] * at  # what is behind the top may be anything
    tokens = sum(c for c in change if c > 0) + rng.randint(0, 3)
    return table, lengths, change, free, total - at, tokens


def tensors(case, device):
    table, lengths, change, free, count, tokens = case
    make = lambda x: torch.tensor(x, dtype=torch.long, device=device)  # noqa: E731
    return make(table).view(len(lengths), -1), make(lengths), make(change), make(free), make([count]), tokens


def assert_resized(own, got, want):
    table, _, _, free, count, _ = own
    for name, a, b in zip(("table", "free", "count", "lengths", "token_ptr", "positions", "slots"),
                          (table, free, count, *got), (*want[:2], [want[2]], *want[3:])):
        assert a.tolist() == b, name
