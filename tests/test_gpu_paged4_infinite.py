"""Attention over 4-bit pages that hold infinite numbers (what is written from 3.5 * 2^126 on), against the CPU composition:
a score of -inf takes no weight, one of +inf makes its head NaN, and an infinite value makes its column infinite (NaN on the
GPU), and all others stay as they are.  Queries next to their type's largest number stay finite."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu
from tests.paged4_common import E2M1, E8M0

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HUGE = 3.2e38  # held as 2^128
# rows that fill the kernel's width, whole groups, parts of groups, parts of words, rows of single bytes
WIDTHS = [64, 128, 256, 32, 96, 160, 40, 72, 34, 130, 200, 6]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


class Held:
    """Rows of ordinary numbers in a cache of one sequence for each of ``lengths``, and places for others."""

    def __init__(self, lengths, heads, width, value_width, page, seed):
        self.gen = torch.Generator().manual_seed(seed)
        self.lengths, self.page = torch.tensor(lengths), page
        self.rows = [torch.randn(sum(lengths), heads, w, generator=self.gen) for w in (width, value_width)]

    def attend(self, query, device, **more):
        counts = (self.lengths + self.page - 1) // self.page
        ptr = torch.nn.functional.pad(counts.cumsum(0), (1, 0))
        span = torch.nn.functional.pad(self.lengths.cumsum(0), (1, 0))
        names, pages = {}, []
        for kind, rows in zip(("key", "value"), self.rows):
            heads, width = rows.shape[1:]
            pages.append(torch.full((int(ptr[-1]), heads, self.page, width // 2), 255, dtype=torch.uint8, device=device).view(E2M1))
            names[kind + "_exponents"] = torch.full((int(ptr[-1]), heads, self.page, -(-width // 32)), 255, dtype=torch.uint8,
                                                    device=device).view(E8M0)
        order = torch.arange(int(ptr[-1])).flip(0)
        lists = [t.to(device) for t in (ptr, order)]
        autosage_amd.paged_cache_write(*(r.to(device) for r in self.rows), *pages, *lists, span.to(device),
                                       torch.zeros_like(self.lengths).to(device), **names)
        return [t.cpu() for t in autosage_amd.paged_attention(
            query.to(device), *pages, *lists, self.lengths.to(device), return_lse=True, **names, **more)]


def _check(held, query, **more):
    """The CPU composition's results: both are rounded once (half a step each), after sums of some 2^-16 of the values
    (weights in bf16 parts, exponentials and sums in float32; values are below 8 but where they are infinite)."""
    out, lse = held.attend(query, "cuda", **more)
    want, want_lse = held.attend(query, "cpu", **more)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(lse.isnan(), want_lse.isnan())
    assert torch.equal(out.isinf(), want.isinf()) and torch.equal(out.isposinf(), want.isposinf())
    eps = torch.finfo(query.dtype).eps
    keep = want.isfinite()
    assert torch.allclose(out[keep].double(), want[keep].double(), rtol=eps, atol=8 * 2.0**-16)
    keep = want_lse.isfinite()
    assert torch.equal(lse[~keep & ~lse.isnan()], want_lse[~keep & ~lse.isnan()])
    assert torch.allclose(lse[keep], want_lse[keep], rtol=2.0**-20, atol=2e-4)
    return want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("width", WIDTHS)
def test_keys_whose_score_is_minus_infinity(dtype, page, width):
    """At a row's begin, in its last group, in both; one token, or all of them."""
    held = Held([40, 300, 17], 2, width, 64, page, seed=width)
    query = torch.randn(3, 4, width, generator=held.gen).to(dtype)
    last = (width - 1) // 32 * 32
    query[:, :, 0], query[:, :, last] = query[:, :, 0].abs() + 0.5, query[:, :, last].abs() + 0.5
    keys = held.rows[0]
    keys[7, :, 0] = -HUGE
    keys[50, :, last] = -HUGE
    keys[111, :, 0], keys[111, :, last] = -HUGE, -HUGE
    keys[340:, 1, 0] = -HUGE
    want = _check(held, query, scale=0.1)
    assert want.isfinite().all() and not want[2, 2:].any() and want[2, :2].any()
    _check(held, query, scale=0.1, max_length=300)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("width", WIDTHS)
def test_keys_whose_score_is_infinite(dtype, page, width):
    """Numbers of the query that fill one part of it (0.5), two or three (1/3), or are negative; a query's zero makes NaN."""
    held = Held([40, 300], 2, width, 64, page, seed=width)
    query = torch.randn(2, 8, width, generator=held.gen)
    # heads 0 to 3 have the first key head: +inf, -inf, -inf, NaN
    for head, first in enumerate((-0.5, 0.5, 1.0 / 3.0, 0.0)):
        query[:, head, 0] = first
    held.rows[0][5, 0, 0] = -HUGE
    held.rows[0][77, 0, 0] = -HUGE
    want = _check(held, query.to(dtype), scale=0.1)
    assert want[:, [0, 3]].isnan().all() and want[:, [1, 2, 4, 5, 6, 7]].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("width", WIDTHS)
def test_infinite_values(dtype, page, width):
    held = Held([40, 300], 2, 64, width, page, seed=width)
    query = torch.randn(2, 4, 64, generator=held.gen).to(dtype)
    plain, _ = held.attend(query, "cuda", scale=0.1)
    spoilt = list(held.rows)
    for sign in (1, -1):
        held.rows = [spoilt[0], spoilt[1].clone()]
        held.rows[1][7, 1, width - 1] = sign * HUGE  # the other numbers of its group become zeros
        out, lse = held.attend(query, "cuda", scale=0.1)
        want, want_lse = held.attend(query, "cpu", scale=0.1)
        assert torch.equal(out.isfinite(), want.isfinite()) and not want[0, 2:, width - 1].isfinite().any()
        assert int((~want.isfinite()).sum()) == 2 and torch.allclose(lse, want_lse, rtol=2.0**-20, atol=2e-4)
        assert torch.equal(out[1], plain[1]) and torch.equal(out[0, :2], plain[0, :2])
        keep = want.isfinite()
        assert torch.allclose(out[keep].double(), want[keep].double(), rtol=torch.finfo(dtype).eps, atol=8 * 2.0**-16)


@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("width", [64, 128, 96, 40, 256])
def test_the_largest_queries_stay_finite(page, width):
    """Numbers that bf16 would round to infinity, times keys of some 2^-122."""
    held = Held([40, 300], 2, width, 64, page, seed=width)
    held.rows[0][:, :, :32] *= 2.0**-122
    query = torch.randn(2, 4, width, generator=held.gen)
    query[:, :, :32] = 0.0
    query[:, :, 3], query[:, :, 7] = torch.finfo(torch.float32).max, -3.4e38
    want = _check(held, query, scale=0.02)
    assert want.isfinite().all()


@pytest.mark.parametrize("width", [64, 40, 200])
@pytest.mark.parametrize("dtype, bits", [(torch.float32, 0x7F800001), (torch.float32, -1), (torch.float16, 0x7C01),
                                         (torch.bfloat16, 0x7F81)])
def test_every_nan_of_a_query_stays_one(dtype, bits, width):
    """Also one whose only bits are those that a shorter type has not."""
    held = Held([40, 300], 1, width, 64, 16, seed=width)
    query = torch.randn(2, 3, width, generator=held.gen).to(dtype)
    query.view(torch.int32 if dtype == torch.float32 else torch.int16)[0, 1, 9] = bits
    assert query.isnan().sum() == 1
    out, lse = held.attend(query, "cuda", scale=0.1)
    assert out[0, 1].isnan().all() and lse[0, 1].isnan()
    assert int(out.isnan().sum()) == 64 and int(lse.isnan().sum()) == 1
