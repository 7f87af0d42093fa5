"""Caches of 4-bit numbers for the tests, with what they hold found by search, in 64 bits."""

from __future__ import annotations

import numpy as np
import torch

E2M1 = torch.float4_e2m1fn_x2
E8M0 = torch.float8_e8m0fnu
SIZES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantised_pairs(x: torch.Tensor):
    """(values in 64 bits, bytes of codes, exponents + 127) that a 4-bit cache holds for finite rows ``x`` of an even
    width: for each 32 numbers the smallest exponent that brings them to 6, found one after another, and the nearest of
    all sizes, ties to the even code."""
    width = x.shape[-1]
    rows = x.double().cpu().numpy().reshape(-1, width)
    values, codes = np.empty_like(rows), np.empty(rows.shape, dtype=np.uint8)
    exponents = np.empty((rows.shape[0], -(-width // 32)), dtype=np.uint8)
    for g in range(exponents.shape[1]):
        part = rows[:, 32 * g:32 * g + 32]
        largest = np.abs(part).max(1)
        e = np.full(rows.shape[0], -127)
        while (over := largest > np.ldexp(6.0, e)).any():
            e += over
        scaled = np.abs(part) / np.ldexp(1.0, e)[:, None]
        away = np.abs(scaled[..., None] - SIZES)
        near = away == away.min(-1, keepdims=True)
        code = np.argmax(near * np.where(np.arange(8) % 2 == 0, 2, 1), -1)  # of two the even one
        values[:, 32 * g:32 * g + 32] = np.copysign(np.ldexp(SIZES[code], e[:, None]), part)
        codes[:, 32 * g:32 * g + 32] = code + 8 * np.signbit(part)
        exponents[:, g] = e + 127
    packed = codes[:, ::2] | codes[:, 1::2] << 4
    return (torch.from_numpy(values.reshape(x.shape)), torch.from_numpy(packed.reshape(*x.shape[:-1], width // 2)),
            torch.from_numpy(exponents.reshape(*x.shape[:-1], -1)))


class Cache4:
    """A cache of 4-bit numbers, every place outside the sequences NaN; ``lengths``, ``heads`` and ``rows`` as of
    ``paged_common.Cache``, whose plain attention reads them."""

    def __init__(self, lengths, heads, key_width, value_width, page, dtype, *, seed=0, spare=2, room=0, interleaved=False,
                 offset=0):
        gen = torch.Generator().manual_seed(seed)
        self.lengths, self.heads, self.page, self.dtype = list(lengths), heads, page, dtype
        counts = [-(-n // page) + room for n in self.lengths]
        pages = sum(counts) + spare
        self.page_ptr = torch.tensor([0] + counts).cumsum(0)
        self.page_idx = torch.randperm(pages, generator=gen)[: sum(counts)]
        self.rows, self.pages, self.exponents = {}, {}, {}
        for index, (kind, width) in enumerate((("key", key_width), ("value", value_width))):
            half, groups = width // 2, -(-width // 32)
            if interleaved:  # heads and kinds of a page side by side, exponents behind the codes of a token
                both = torch.full((pages, page, heads, 2, half + groups), 255, dtype=torch.uint8)
                store = both[:, :, :, index, :half].transpose(1, 2)
                exponents = both[:, :, :, index, half:].transpose(1, 2)
            else:
                store = torch.full((pages * heads * page * half + offset,), 255, dtype=torch.uint8)[offset:].view(
                    pages, heads, page, half)
                exponents = torch.full((pages * heads * page * groups + offset,), 255, dtype=torch.uint8)[offset:].view(
                    pages, heads, page, groups)
            self.rows[kind] = []
            for b, length in enumerate(self.lengths):
                rows = torch.randn(length, heads, width, generator=gen)
                rows = (rows * torch.exp(0.5 * torch.randn(length, heads, 1, generator=gen))).to(dtype)
                if length > 0:
                    t = torch.arange(length)
                    where, place = self.page_idx[self.page_ptr[b] + t // page], t % page
                    rows, store[where, :, place], exponents[where, :, place] = quantised_pairs(rows)
                self.rows[kind].append(rows.double())
            self.pages[kind], self.exponents[kind] = store, exponents

    def args(self, device="cuda"):
        """(key_pages, value_pages, page_ptr, page_idx) and the exponents as keywords, with the layout kept."""

        def move(t, dtype):
            base = t._base if t._base is not None else t
            return base.to(device).as_strided(t.shape, t.stride(), t.storage_offset()).view(dtype)

        return ((move(self.pages["key"], E2M1), move(self.pages["value"], E2M1), self.page_ptr.to(device),
                 self.page_idx.to(device)),
                {kind + "_exponents": move(self.exponents[kind], E8M0) for kind in ("key", "value")})
