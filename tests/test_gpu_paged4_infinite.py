"""Attention over 4-bit pages that hold infinite numbers (what is written from 3.5 * 2^126 on), against the CPU composition:
a score of -inf takes no weight, one of +inf makes its head NaN, and an infinite value makes its column infinite."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu
from tests.paged4_common import E2M1, E8M0

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16]
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
