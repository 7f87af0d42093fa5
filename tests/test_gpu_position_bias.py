"""The learned position bias on the GPU against the definition: every value exactly, gradients within their sums."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import autosage_amd
from autosage_amd.position import position_buckets
from tests.gpu_common import case_graph, require_gpu, to_dev
from tests.paged_common import plain_buckets

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _plain(crow, col, buckets, max_distance, bidirectional, positions):
    rows = np.repeat(np.arange(len(crow) - 1), np.diff(crow))
    at = np.arange(len(crow) - 1) if positions is None else positions
    return torch.from_numpy(plain_buckets(at[col] - at[rows], buckets, max_distance, bidirectional))


def _check(crow, col, heads, buckets, max_distance, dtype, bidirectional=True, positions=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    table = torch.randn(buckets, heads, generator=gen).to(dtype)
    bucket = _plain(crow, col, buckets, max_distance, bidirectional, positions)
    d_crow, d_col, d_positions = to_dev(crow, col, positions)
    d_table = table.cuda().requires_grad_()
    out = autosage_amd.csr_position_bias(d_crow, d_col, d_table, max_distance=max_distance,
                                         bidirectional=bidirectional, positions=d_positions)
    assert out.dtype == dtype and torch.equal(out.detach().cpu(), table.t()[:, bucket])
    with torch.no_grad():
        again = autosage_amd.csr_position_bias(d_crow, d_col, d_table, max_distance=max_distance,
                                               bidirectional=bidirectional, positions=d_positions)
    assert torch.equal(again, out)
    grad = torch.randn(heads, len(col), generator=gen).to(dtype)
    got, = torch.autograd.grad(out, d_table, grad.cuda())
    want = torch.zeros(buckets, heads, dtype=torch.float64).index_add_(0, bucket, grad.double().t())
    size = torch.zeros_like(want).index_add_(0, bucket, grad.double().abs().t())
    # at most 64 terms in a row in fp32, the rest in fp64, one rounding to the type
    allowed = size * 64 * 2.0**-24 + want.abs() * torch.finfo(dtype).eps / 2 * 1.001 + 1e-30
    if dtype == torch.float16:
        allowed = allowed + 2.0**-25
    assert got.dtype == dtype and bool(((got.double().cpu() - want).abs() <= allowed).all())
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, degree, hubs, empty", [(1, 1, 0, 0.0), (7, 3, 0, 0.3), (64, 1, 0, 0.0), (700, 20, 3, 0.4),
                                                       (5000, 9, 2, 0.9)])
@pytest.mark.parametrize("heads, buckets, max_distance, bidirectional", [
    (1, 32, 128, True), (5, 32, 128, False), (8, 2, 5, False), (3, 64, 4096, True), (16, 128, 300, True),
    (2, 256, 2000, False), (4, 10, 6, True)])
def test_bias_and_gradient(dtype, rows, degree, hubs, empty, heads, buckets, max_distance, bidirectional):
    crow, col = case_graph(rows, degree, seed=rows, hubs=hubs, hub_degree=min(rows, 600) if hubs else 0, empty=empty)
    _check(crow, col, heads, buckets, max_distance, dtype, bidirectional)


@pytest.mark.parametrize("nnz", [1, 63, 64, 65, 255, 257, 1023, 1025, 4097, 16385, 70001])
def test_edge_counts_around_the_blocks(nnz):
    rng = np.random.default_rng(nnz)
    n = 300
    crow = np.zeros(n + 1, dtype=np.int64)
    crow[1:] = np.sort(rng.integers(0, nnz + 1, n))
    crow[-1] = nnz
    col = rng.integers(0, n, nnz)
    for dtype, heads in ((torch.float32, 3), (torch.bfloat16, 5)):
        _check(crow, col, heads, 32, 100, dtype)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_positions_of_their_own(index):
    crow, col = case_graph(900, 12, seed=3, empty=0.2)
    positions = np.random.default_rng(0).integers(-5000, 5000, 900)
    _check(crow, col, 4, 32, 128, torch.float32, positions=positions)
    _check(crow, col, 4, 32, 128, torch.float32, bidirectional=False, positions=positions)
    d_crow, d_col, d_positions = to_dev(crow, col, positions)
    table = torch.randn(32, 4, device="cuda")
    a = autosage_amd.csr_position_bias(d_crow, d_col, table, max_distance=128, positions=d_positions)
    b = autosage_amd.csr_position_bias(d_crow.to(index), d_col.to(index), table, max_distance=128,
                                       positions=d_positions.to(index))
    assert torch.equal(a, b)


def test_far_positions_and_every_border():
    """One row of keys at every distance around the borders, and at distances beyond 32 bits."""
    near = np.arange(-2100, 2101)
    far = np.array([2**31 - 1, 2**31, 2**31 + 1, 2**40, 2**61])
    positions = np.concatenate([[0], near, far, -far])
    n = len(positions)
    crow = np.concatenate([[0], np.full(n, n - 1)]).astype(np.int64)
    col = np.arange(1, n)
    for buckets, distance, both in ((64, 2000, True), (32, 128, False), (200, 1999, False), (8, 2**31 - 1, True)):
        _check(crow, col, 2, buckets, distance, torch.float32, both, positions)


@pytest.mark.parametrize("far", [False, True])
def test_many_nodes_with_positions(far):
    """Enough nodes for the 32-bit copy of the positions, which one position beyond 32 bits rules out."""
    n, degree = 600_000, 4
    rng = np.random.default_rng(11)
    crow = np.arange(n + 1, dtype=np.int64) * degree
    col = rng.integers(0, n, n * degree)
    positions = rng.permutation(n) - 100_000
    if far:
        positions[n // 3] = 2**33
    rel = positions[col] - np.repeat(positions, degree)
    bucket = torch.from_numpy(plain_buckets(np.clip(rel, -3000, 3000), 32, 2000, True))
    table = torch.randn(32, 2)
    d_crow, d_col, d_positions = to_dev(crow, col, positions)
    out = autosage_amd.csr_position_bias(d_crow, d_col, table.cuda(), max_distance=2000, positions=d_positions)
    assert torch.equal(out.cpu(), table.t()[:, bucket])


def test_a_table_with_strides_and_a_gradient_that_is_expanded():
    crow, col = case_graph(400, 7, seed=5)
    d_crow, d_col = to_dev(crow, col)
    base = torch.randn(4, 32, device="cuda", requires_grad=True)
    out = autosage_amd.csr_position_bias(d_crow, d_col, base.t(), max_distance=64)
    out.sum().backward()  # an expanded gradient of ones
    bucket = _plain(crow, col, 32, 64, True, None)
    assert torch.equal(base.grad.cpu(), torch.bincount(bucket, minlength=32).float().expand(4, 32))


def test_second_gradient():
    crow, col = case_graph(50, 4, seed=6)
    d_crow, d_col = to_dev(crow, col)
    table = torch.randn(8, 2, device="cuda", requires_grad=True)
    weights = torch.randn(2, len(col), device="cuda")
    out = autosage_amd.csr_position_bias(d_crow, d_col, table, max_distance=9)
    first, = torch.autograd.grad((out * out * weights).sum(), table, create_graph=True)
    second, = torch.autograd.grad((first * first).sum(), table)
    cpu = table.detach().cpu().double().requires_grad_()
    out = autosage_amd.csr_position_bias(torch.from_numpy(crow), torch.from_numpy(col), cpu, max_distance=9)
    first, = torch.autograd.grad((out * out * weights.cpu().double()).sum(), cpu, create_graph=True)
    want, = torch.autograd.grad((first * first).sum(), cpu)
    assert torch.allclose(second.double().cpu(), want, rtol=1e-4, atol=1e-4)


def test_the_registered_operators():
    crow, col = case_graph(500, 9, seed=12)
    d_crow, d_col = to_dev(crow, col)
    table = torch.randn(32, 3, device="cuda", requires_grad=True)
    weights = torch.randn(3, len(col), device="cuda")
    gradients = []
    for out in (autosage_amd.csr_position_bias(d_crow, d_col, table, max_distance=90),
                torch.ops.autosage.csr_position_bias(d_crow, d_col, None, table, 90, True)[0]):
        first, = torch.autograd.grad((out * out * weights).sum(), table, create_graph=True)
        gradients.append((out, first, *torch.autograd.grad((first * first).sum(), table)))
    assert all(torch.equal(a, b) for a, b in zip(*gradients))


def test_the_same_bits_every_time():
    crow, col = case_graph(20000, 30, seed=7, hubs=4, hub_degree=5000)
    one = _check(crow, col, 4, 32, 1000, torch.float32)
    for _ in range(3):
        assert torch.equal(_check(crow, col, 4, 32, 1000, torch.float32), one)


def test_offsets_beyond_32_bits():
    """More than 2^32 biases: rows of 512 neighbours each, nine heads in 16 bits; the gradient of ones counts edges."""
    n, degree, heads = (1 << 20) + 3, 512, 9
    crow = torch.arange(n + 1, device="cuda") * degree
    step = torch.arange(degree, device="cuda") * 3 - 700
    col = ((torch.arange(n, device="cuda")[:, None] + step) % n).view(-1)
    table = torch.randn(32, heads, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = autosage_amd.csr_position_bias(crow, col, table, max_distance=600)
    assert out.numel() > 2**32
    count = torch.zeros(32, dtype=torch.long)
    for a in range(0, n, 1 << 18):
        b = min(a + (1 << 18), n)
        rel = col.view(n, degree)[a:b] - torch.arange(a, b, device="cuda")[:, None]
        bucket = position_buckets(rel.flatten(), 32, 600, True)
        count += torch.bincount(bucket, minlength=32).cpu()
        for h in (0, heads - 1):
            assert torch.equal(out[h, a * degree:b * degree], table.detach()[bucket, h])
    grad, = torch.autograd.grad(out, table, torch.ones_like(out))
    assert torch.equal(grad.cpu(), count.double().bfloat16()[:, None].expand(32, heads))


def test_empty_graph_and_refusals():
    none = torch.zeros(0, dtype=torch.long, device="cuda")
    crow = torch.zeros(5, dtype=torch.long, device="cuda")
    table = torch.randn(8, 3, device="cuda", requires_grad=True)
    out = autosage_amd.csr_position_bias(crow, none, table, max_distance=9)
    assert out.shape == (3, 0)
    out.sum().backward()
    assert table.grad.shape == (8, 3) and not table.grad.any()
    with pytest.raises(TypeError):
        autosage_amd.csr_position_bias(crow, none, table.double(), max_distance=9)
    with pytest.raises(ValueError):
        autosage_amd.csr_position_bias(crow, none.cpu(), table, max_distance=9)


def test_capture_of_a_training_step():
    crow, col = case_graph(3000, 20, seed=8, hubs=2, hub_degree=900)
    d_crow, d_col = to_dev(crow, col)
    table = torch.randn(32, 4, device="cuda", requires_grad=True)
    grad = torch.randn(4, len(col), device="cuda")

    def step():
        out = autosage_amd.csr_position_bias(d_crow, d_col, table, max_distance=128)
        return out.detach(), torch.autograd.grad(out, table, grad)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        with torch.no_grad():
            table.mul_(1.5)
            grad.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_another_stream():
    crow, col = case_graph(3000, 20, seed=9)
    d_crow, d_col = to_dev(crow, col)
    table = torch.randn(32, 4, device="cuda")
    want = autosage_amd.csr_position_bias(d_crow, d_col, table, max_distance=128)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = autosage_amd.csr_position_bias(d_crow, d_col, table, max_distance=128)
    side.synchronize()
    assert torch.equal(got, want)


def test_columns_beyond_the_rows(monkeypatch):
    """Without positions a graph need not be square, also where it is validated; with them it has to be."""
    crow, col = torch.tensor([0, 2, 3]), torch.tensor([0, 9, 2**40])
    table = torch.randn(8, 2)
    want = autosage_amd.csr_position_bias(crow, col, table, max_distance=20)
    for validate in ("0", "1"):
        monkeypatch.setenv("AUTOSAGE_VALIDATE", validate)
        got = autosage_amd.csr_position_bias(crow.cuda(), col.cuda(), table.cuda(), max_distance=20)
        assert torch.equal(got.cpu(), want)
    with pytest.raises(ValueError, match="CSR"):
        autosage_amd.csr_position_bias(crow.cuda(), -col.cuda(), table.cuda(), max_distance=20)
    with pytest.raises(ValueError, match="CSR"):
        autosage_amd.csr_position_bias(crow.cuda(), col.cuda(), table.cuda(), max_distance=20,
                                       positions=torch.arange(2).cuda())


def test_the_registered_operator_is_validated(monkeypatch):
    crow, col = torch.tensor([0, 2, 3]).cuda(), torch.tensor([0, -1, 1]).cuda()
    table = torch.randn(8, 2, device="cuda", requires_grad=True)
    monkeypatch.setenv("AUTOSAGE_VALIDATE", "1")
    with pytest.raises(ValueError, match="CSR"):
        torch.ops.autosage.csr_position_bias(crow, col, None, table, 9, True)
    torch.ops.autosage.csr_position_bias(crow, col.abs(), None, table, 9, True)


def test_forward_mode():
    """Tangents of the table, and of the gradient that comes back."""
    crow, col = case_graph(60, 5, seed=13)
    cpu, gpu = (torch.from_numpy(crow), torch.from_numpy(col)), to_dev(crow, col)
    gen = torch.Generator().manual_seed(14)
    table, tangent = torch.randn(8, 2, generator=gen), torch.randn(8, 2, generator=gen)
    weights, change = torch.randn(2, len(col), generator=gen), torch.randn(2, len(col), generator=gen)
    fw = torch.autograd.forward_ad
    results = []
    for graph, device in ((cpu, "cpu"), (gpu, "cuda")):
        own = table.clone().to(device).requires_grad_()
        with fw.dual_level():
            dual = fw.make_dual(own, tangent.to(device))
            out = autosage_amd.csr_position_bias(*graph, dual, max_distance=9)
            first, = torch.autograd.grad((out * out).sum(), own)
            back, = torch.autograd.grad(autosage_amd.csr_position_bias(*graph, own, max_distance=9), own,
                                        fw.make_dual(weights.to(device), change.to(device)))
            results.append([*fw.unpack_dual(out), *fw.unpack_dual(first), *fw.unpack_dual(back)])
    for a, b in zip(*results):
        assert a is not None and torch.allclose(a, b.cpu(), rtol=1e-5, atol=1e-5)
    assert torch.equal(results[0][1], results[1][1].cpu())
    with fw.dual_level():
        for grad in (False, True):
            dual = fw.make_dual(table.cuda().requires_grad_(grad), tangent.cuda())
            with pytest.raises(RuntimeError):
                torch.ops.autosage.csr_position_bias(*gpu, None, dual, 9, True)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.ops.autosage.csr_position_bias_backward(torch.zeros(4, dtype=torch.uint8, device="cuda"),
                                                          fw.make_dual(weights[:, :4].cuda(), change[:, :4].cuda()), 8)


def test_function_transforms():
    """torch.func over the GPU's function and the CPU's composition: derivatives, batches of tables and of graphs."""
    crow, col = case_graph(40, 4, seed=15)
    gen = torch.Generator().manual_seed(16)
    table, tables = torch.randn(6, 2, generator=gen), torch.randn(3, 6, 2, generator=gen)
    weights = torch.randn(2, len(col), generator=gen)
    positions = torch.randint(-20, 20, (3, 40), generator=gen)
    f = torch.func
    results = []
    for device in ("cpu", "cuda"):
        graph = [torch.from_numpy(a).to(device) for a in (crow, col)]
        w, t, ts, at = (x.to(device) for x in (weights, table, tables, positions))

        def bias(table, positions=None):
            return autosage_amd.csr_position_bias(*graph, table, max_distance=9, positions=positions)

        def loss(table):
            return (bias(table) ** 3 * w).sum()

        results.append([f.grad(loss)(t), f.vmap(bias)(ts), f.vmap(bias, in_dims=1)(ts.transpose(0, 1)),
                        f.vmap(f.grad(loss))(ts), f.jacrev(bias)(t), f.jacfwd(bias)(t), f.hessian(loss)(t),
                        f.jacrev(f.jacrev(loss))(t), f.jvp(bias, (t,), (ts[0],))[1], f.vmap(bias)(ts, at),
                        f.vmap(f.grad(lambda a, p: (bias(a, p) ** 2 * w).sum()))(ts, at), f.vjp(bias, t)[1](w)[0],
                        f.vmap(f.vjp(bias, t)[1])(torch.stack([w, 2 * w]))[0]])
    for a, b in zip(*results):
        # sums of a few dozen numbers of both devices in float32, in different orders
        assert a.shape == b.shape and torch.allclose(a, b.cpu(), rtol=1e-4, atol=1e-4)


def test_batches_of_more_heads_than_one_call_takes():
    crow, col = case_graph(6, 2, seed=17)
    gen = torch.Generator().manual_seed(18)
    tables, weights = torch.randn(2, 4, 40000, generator=gen), torch.randn(40000, len(col), generator=gen)
    results = []
    for device in ("cpu", "cuda"):
        graph = [torch.from_numpy(a).to(device) for a in (crow, col)]
        ts, w = tables.to(device), weights.to(device)

        def bias(table):
            return autosage_amd.csr_position_bias(*graph, table, max_distance=9)

        results.append([torch.func.vmap(bias)(ts), torch.func.vmap(torch.func.grad(lambda t: (bias(t) * w).sum()))(ts)])
    assert torch.equal(results[0][0], results[1][0].cpu())
    # sums of at most a dozen numbers of a few units in float32
    assert torch.allclose(results[0][1], results[1][1].cpu(), rtol=1e-5, atol=1e-5)
