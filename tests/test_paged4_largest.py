"""4-bit pages of numbers that round past the largest of their type: the bounds that the write names."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.paged4_common import E2M1, E8M0


def _back(rows, dtype, device):
    tokens, _, width = rows.shape
    pages = [torch.zeros(1, 1, tokens, width // 2, dtype=torch.uint8, device=device).view(E2M1) for _ in range(2)]
    names = {kind + "_exponents": torch.zeros(1, 1, tokens, -(-width // 32), dtype=torch.uint8, device=device).view(E8M0)
             for kind in ("key", "value")}
    span = [torch.tensor(x, device=device) for x in ([0, 1], [0], [0, tokens], [0])]
    autosage_amd.paged_cache_write(rows.to(device), rows.to(device), *pages, *span, **names)
    key, value = autosage_amd.paged_cache_read(*pages, *span, tokens, dtype=dtype, **names)
    assert torch.equal(key, value)
    return key.cpu()


def _check(device):
    # neighbours in float16: the largest that stays, the smallest that does not
    below, above = torch.tensor(57344.0).half().view(torch.int16) - 1, torch.tensor(57344.0).half()
    rows = torch.stack((below.view(torch.float16), above, torch.tensor(65504.0).half(), torch.tensor(49152.0).half()))
    got = _back(rows[:, None, None].expand(4, 1, 2).contiguous(), torch.float16, device)[:, 0, 0]
    assert got.tolist() == [49152.0, float("inf"), float("inf"), 49152.0]
    assert _back(rows[:, None, None].expand(4, 1, 2).contiguous(), torch.bfloat16, device)[:, 0, 0].tolist() == [
        49152.0, 65536.0, 65536.0, 49152.0]
    border = 3.5 * 2.0**126
    for dtype in (torch.float32, torch.bfloat16):
        rows = torch.tensor([border * (1 - 2.0**-8), border, torch.finfo(dtype).max, -border], dtype=dtype)
        for out in (dtype, torch.float32):
            got = _back(rows[:, None, None].expand(4, 1, 2).contiguous(), out, device)[:, 0, 0]
            assert got.tolist() == [3 * 2.0**126, float("inf"), float("inf"), -float("inf")]


def test_bounds_on_the_cpu():
    _check("cpu")


@pytest.mark.gpu
def test_bounds_on_the_gpu():
    from tests.gpu_common import require_gpu

    require_gpu()
    _check("cuda")
