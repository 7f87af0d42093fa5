"""The learned position bias on the CPU: buckets, gradients and refusals."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import autosage
import autosage_amd
from autosage_amd.position import bucket_borders, position_buckets
from tests.paged_common import plain_buckets


@pytest.mark.parametrize("buckets, max_distance, bidirectional", [
    (32, 128, True), (32, 128, False), (2, 5, False), (3, 2, False), (2, 7, True), (4, 3, True), (64, 4096, True),
    (128, 65, False), (256, 100000, False), (10, 6, True), (9, 1000, False), (32, 17, False)])
def test_buckets_are_those_of_the_definition(buckets, max_distance, bidirectional):
    relative = np.unique(np.concatenate([np.arange(-300, 301), [-max_distance - 1, -max_distance, 1 - max_distance,
                                                               max_distance, 10**9, -(10**9), 2**40, -(2**40)]]))
    got = position_buckets(torch.from_numpy(relative), buckets, max_distance, bidirectional)
    assert np.array_equal(got.numpy(), plain_buckets(relative, buckets, max_distance, bidirectional))
    borders = bucket_borders(buckets, max_distance, bidirectional)
    assert borders[0] == 0 and list(borders) == sorted(borders)
    assert len(borders) == (buckets // 2 if bidirectional else buckets)


def _graph():
    crow = torch.tensor([0, 3, 3, 5, 9])
    col = torch.tensor([0, 1, 3, 2, 0, 3, 3, 1, 0])
    rows = [0, 0, 0, 2, 2, 3, 3, 3, 3]
    return crow, col, rows


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("with_positions", [False, True])
def test_bias_is_the_table_entry_of_every_edge(dtype, index, with_positions):
    crow, col, rows = _graph()
    table = torch.randn(6, 3, generator=torch.Generator().manual_seed(0)).to(dtype)
    positions = torch.tensor([7, -40, 3, 0]) if with_positions else None
    at = positions if with_positions else torch.arange(4)
    bucket = plain_buckets([int(at[c] - at[r]) for c, r in zip(col, rows)], 6, 9, True)
    got = autosage_amd.csr_position_bias(crow.to(index), col.to(index), table, max_distance=9,
                                         positions=None if positions is None else positions.to(index))
    assert torch.equal(got, table[torch.from_numpy(bucket)].t())


def test_gradient_against_differences_on_the_cpu():
    crow, col, _ = _graph()
    table = torch.randn(6, 3, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda t: autosage_amd.csr_position_bias(crow, col, t, max_distance=9), (table,))


def test_a_graph_without_edges():
    table = torch.randn(4, 2)
    assert autosage_amd.csr_position_bias(torch.zeros(4, dtype=torch.long), torch.zeros(0, dtype=torch.long), table,
                                          max_distance=9).shape == (2, 0)


def test_refusals():
    crow, col, _ = _graph()
    table = torch.randn(6, 3)

    def call(**changes):
        args = {"crow": crow, "col": col, "table": table, "max_distance": 9, **changes}
        return autosage_amd.csr_position_bias(args.pop("crow"), args.pop("col"), args.pop("table"), **args)

    for error, changes in [
        (TypeError, {"crow": crow.float()}), (TypeError, {"col": col.float()}), (TypeError, {"table": table.long()}),
        (ValueError, {"crow": crow[None]}), (ValueError, {"table": table[0]}), (ValueError, {"table": table[:, :0]}),
        (ValueError, {"table": table[:5]}), (ValueError, {"table": table[:1], "bidirectional": False}),
        (ValueError, {"table": torch.randn(258, 1)}), (ValueError, {"max_distance": 1}),
        (ValueError, {"max_distance": 2**31}), (ValueError, {"table": table, "max_distance": 3, "bidirectional": False}),
        (ValueError, {"positions": torch.arange(3)}), (TypeError, {"positions": torch.rand(4)}),
        (ValueError, {"crow": torch.zeros(0, dtype=torch.long)}),
        (ValueError, {"crow": torch.zeros(1, dtype=torch.long)}),
    ]:
        with pytest.raises(error):
            call(**changes)
    call()


def test_the_names_are_public_in_both_packages():
    for name in ("csr_position_bias", "paged_cache_write", "paged_cache_read", "paged_attention"):
        assert name in autosage.__all__ and name in autosage_amd.__all__
        assert getattr(autosage, name) is getattr(autosage_amd, name)
