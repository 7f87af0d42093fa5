"""A query head's result does not depend on the other heads of the call, to the last bit."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu
from tests.paged4_common import Cache4
from tests.paged_common import Cache

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _cache(kind, lengths, width, page, dtype, seed):
    if kind == "4 bits":
        return Cache4(lengths, 1, width, width, page, dtype, seed=seed)
    return Cache(lengths, 1, width, width, page, dtype, quantised=kind == "8 bits", seed=seed)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["as they are", "8 bits", "4 bits"])
@pytest.mark.parametrize("width, page", [(64, 16), (128, 8), (200, 8), (40, 5), (6, 8)])
def test_other_heads_change_nothing(dtype, kind, width, page):
    """Heads whose scores rise at other tokens, that are infinite, NaN or zeros: the running maximum is each head's own."""
    lengths = [40, 700, 1300]
    for seed in range(6):
        cache = _cache(kind, lengths, width, page, dtype, seed)
        args, exponents = cache.args()
        count = torch.tensor(lengths).cuda()
        gen = torch.Generator().manual_seed(seed)
        query = torch.randn(3, 5, width, generator=gen)
        others = {"more": query * 3, "less": query / 16, "new": torch.randn(3, 5, width, generator=gen),
                  "infinite": query.clone(), "NaN": query * float("nan"), "zeros": query * 0}
        others["infinite"][..., width // 2] = float("inf")
        for bound in (None, 1300):
            def attend(q):
                return autosage_amd.paged_attention(q.to(dtype).cuda(), *args, count, scale=0.25, max_length=bound,
                                                    return_lse=True, **exponents)

            want, want_lse = attend(query)
            assert want.isfinite().all()
            for name, other in others.items():
                other[:, 1], other[:, 4] = query[:, 1], query[:, 4]
                out, lse = attend(other)
                for head in (1, 4):
                    assert torch.equal(out[:, head], want[:, head]), (seed, bound, name)
                    assert torch.equal(lse[:, head], want_lse[:, head]), (seed, bound, name)
