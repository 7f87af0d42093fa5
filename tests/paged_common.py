"""Caches, plain 64-bit results and error bounds for the paged-cache tests."""

from __future__ import annotations

import math
from fractions import Fraction

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn
STALE = float("nan")


def plain_buckets(relative, buckets: int, max_distance: int, bidirectional: bool) -> np.ndarray:
    """Buckets from the definition: d < E holds its own bucket, else E + the largest j (below n - E) with
    (d / E)^(n - E) >= (M / E)^j, in exact fractions."""
    side = buckets // 2 if bidirectional else buckets
    exact = side // 2
    rest = side - exact
    out = np.empty(len(relative), dtype=np.int64)
    known = {}
    for i, rel in enumerate(relative):
        rel = int(rel)
        d = abs(rel) if bidirectional else max(-rel, 0)
        if d not in known:
            if d < exact:
                known[d] = d
            elif side == 1:
                known[d] = 0
            else:
                left = Fraction(min(d, max_distance), exact) ** rest
                step = Fraction(max_distance, exact)
                j = 0
                while j + 1 < rest and left >= step ** (j + 1):
                    j += 1
                known[d] = exact + j
        out[i] = known[d] + (side if bidirectional and rel > 0 else 0)
    return out


def quantised_rows(x: torch.Tensor):
    """(values in 64 bits, exponents) that an 8-bit cache holds for finite rows ``x``, by search over all of e4m3's
    numbers: nearest, ties to the even code."""
    codes = torch.arange(127, dtype=torch.uint8).view(E4M3).double().numpy()
    rows = x.double().cpu().numpy().reshape(-1, x.shape[-1])
    values = np.empty_like(rows)
    exponents = np.empty(rows.shape[0], dtype=np.int64)
    for i, row in enumerate(rows):
        largest = np.abs(row).max()
        e = -126
        while largest > 448.0 * 2.0**e:
            e += 1
        exponents[i] = e
        scaled = np.abs(row) / 2.0**e
        near = np.searchsorted(codes, scaled)
        below = np.clip(near - 1, 0, 126)
        above = np.clip(near, 0, 126)
        to_below, to_above = scaled - codes[below], codes[above] - scaled
        pick = np.where(to_below < to_above, below, np.where(to_above < to_below, above,
                                                            np.where(below % 2 == 0, below, above)))
        values[i] = np.copysign(codes[pick] * 2.0**e, row)
    return torch.from_numpy(values.reshape(x.shape)), torch.from_numpy(exponents.reshape(x.shape[:-1]))


class Cache:
    """A cache whose every place outside the sequences holds NaN, with rows drawn on the CPU."""

    def __init__(self, lengths, heads, key_width, value_width, page, dtype, *, quantised=False, seed=0, spare=2, room=0,
                 interleaved=False, offset=0):
        gen = torch.Generator().manual_seed(seed)
        self.lengths = list(lengths)
        self.heads, self.page, self.dtype, self.quantised = heads, page, dtype, quantised
        counts = [-(-n // page) + room for n in self.lengths]
        pages = sum(counts) + spare
        self.page_ptr = torch.tensor([0] + counts).cumsum(0)
        self.page_idx = torch.randperm(pages, generator=gen)[: sum(counts)]
        held = E4M3 if quantised else dtype
        self.rows = {}
        self.pages, self.exponents = {}, {}
        shared = None
        if interleaved:
            assert key_width == value_width
            shared = torch.full((pages, 2, heads, page, key_width), STALE).to(held)
        for index, (kind, width) in enumerate((("key", key_width), ("value", value_width))):
            store = shared[:, index] if interleaved else torch.full((pages * heads * page * width + offset,), STALE).to(
                held)[offset:].view(pages, heads, page, width)
            exponents = torch.full((pages, heads, page), 127, dtype=torch.int8) if quantised else None
            self.rows[kind] = []
            for b, length in enumerate(self.lengths):
                rows = torch.randn(length, heads, width, generator=gen)
                rows = (rows * torch.exp(0.5 * torch.randn(length, heads, 1, generator=gen))).to(dtype)
                if length == 0:
                    self.rows[kind].append(rows.double())
                    continue
                t = torch.arange(length)
                where, place = self.page_idx[self.page_ptr[b] + t // page], t % page
                if quantised:
                    values, e = quantised_rows(rows)
                    scaled = torch.ldexp(values, -e[..., None]).float().to(E4M3)
                    store.view(torch.uint8)[where, :, place] = scaled.view(torch.uint8)
                    exponents[where, :, place] = e.to(torch.int8)
                    self.rows[kind].append(values)
                else:
                    store[where, :, place] = rows
                    self.rows[kind].append(rows.double())
            self.pages[kind], self.exponents[kind] = store, exponents

    def args(self, device="cuda"):
        """(key_pages, value_pages, page_ptr, page_idx) and the exponents as keywords, with the layout kept."""

        def move(t):
            if t is None or device == "cpu":
                return t
            base = t._base if t._base is not None else t
            return base.to(device).as_strided(t.shape, t.stride(), t.storage_offset())

        return ((move(self.pages["key"]), move(self.pages["value"]), self.page_ptr.to(device),
                 self.page_idx.to(device)),
                {"key_exponents": move(self.exponents["key"]), "value_exponents": move(self.exponents["value"])})


def plain_attention(cache: Cache, query, scale, *, window=None, table=None, max_distance=None, bidirectional=True):
    """(out, lse, bound) in 64 bits.  ``bound`` counts what fp32 arithmetic may be off before the last rounding,
    relative to A = sum p|v| / sum p: every score is off by (width + 8) * 2^-23 of scale * sum |q k| + |bias|, which
    changes p by as much relatively; p itself by 2^-21 (argument and value of exp2); n terms summed in fp32 by
    n * 2^-24, twice (numerator, denominator)."""
    heads_q = query.shape[1]
    group = heads_q // cache.heads
    out = torch.zeros(len(cache.lengths), heads_q, cache.rows["value"][0].shape[-1], dtype=torch.float64)
    lse = torch.full((len(cache.lengths), heads_q), -math.inf, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for b, length in enumerate(cache.lengths):
        first = max(0, length - window) if window else 0
        n = length - first
        if n <= 0:
            continue
        for h in range(heads_q):
            k = cache.rows["key"][b][first:, h // group]
            v = cache.rows["value"][b][first:, h // group]
            q = query[b, h].double()
            s = (k @ q) * scale
            size = (k.abs() @ q.abs()) * abs(scale)
            if table is not None:
                bucket = plain_buckets(np.arange(first - length + 1, 1), table.shape[0], max_distance, bidirectional)
                bias = table[:, h].double()[torch.from_numpy(bucket)]
                s, size = s + bias, size + torch.where(bias.isinf(), 0.0, bias.abs())
            top = s.max()
            if top == -math.inf:
                continue
            p = (s - top).exp()
            total = p.sum()
            out[b, h] = (p @ v) / total
            lse[b, h] = top + total.log()
            off = float(size.max()) * (q.numel() + 8) * 2.0**-23 + 2.0**-21 + n * 2.0**-24
            bound[b, h] = 2 * off * (p @ v.abs()) / total
    return out, lse, bound


# Weights rounded for the matrix units: two bf16 parts keep 2^-18 of a weight, two fp16 parts 2^-22, each doubled
# for the order of sums; float32 has none.
_WEIGHT = {torch.float32: 2.0**-22, torch.bfloat16: 2.0**-17, torch.float16: 2.0**-20}


def assert_attention(got, lse, want, *, dtype, quantised=False, lse_bound=None):
    """Every output within its bound plus half a step of its type; the lse within the bound of the scores."""
    out, want_lse, bound = want
    got = got.double().cpu()
    # an 8-bit cache is multiplied in bf16 parts whatever the queries are (three of them for float32)
    weight = _WEIGHT[dtype] if not quantised or dtype == torch.float32 else _WEIGHT[torch.bfloat16]
    # |out| <= A and bound >= 2 * 2^-21 A: the weights' rounding counts relative to A <= bound / 2^-20
    allowed = bound * (1 + weight * 2.0**20) + torch.finfo(dtype).eps / 2 * out.abs() * (1 + 2.0**-10)
    allowed = allowed + float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    error = (got - out).abs()
    assert got.isfinite().all(), "not finite"
    worst = float((error / allowed.clamp_min(1e-300)).max()) if error.numel() else 0.0
    assert worst <= 1.0, f"error over bound {worst}"
    if lse is not None:
        lse = lse.double().cpu()
        empty = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        assert (lse[~empty] - want_lse[~empty]).abs().max().item() <= lse_bound if (~empty).any() else True
    return worst
