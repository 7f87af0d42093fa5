"""Rotary positions on the GPU against 64-bit results."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu
from tests.rotary_common import assert_turned, plain_turn

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _inputs(tokens, heads, key_heads, width, dtype, seed, furthest=5000):
    gen = torch.Generator().manual_seed(seed)
    query = torch.randn(tokens, heads, width, generator=gen).to(dtype)
    key = torch.randn(tokens, key_heads, width, generator=gen).to(dtype)
    positions = torch.randint(-furthest // 10, furthest, (tokens,), generator=gen)
    return query, key, positions


def _frequencies(pairs):
    return autosage_amd.rotary_frequencies(2 * pairs) if pairs else torch.zeros(0, dtype=torch.float64)


def _check(query, key, positions, frequencies, interleaved, magnitude=1.0, move=lambda t: t.cuda()):
    got = autosage_amd.rotary_positions(move(query), move(key), positions.cuda(), frequencies.cuda(),
                                        interleaved=interleaved, magnitude=magnitude)
    for x, y in zip((query, key), got):
        assert y.is_contiguous() and y.shape == x.shape and y.dtype == x.dtype
        assert_turned(y, plain_turn(x, positions, frequencies, interleaved, magnitude), x, frequencies.numel(), magnitude)
    return got


SHAPES = [(1, 0), (2, 1), (3, 1), (7, 3), (8, 4), (16, 8), (15, 7), (18, 9), (24, 12), (33, 5), (40, 10), (64, 32), (72, 36),
          (80, 16), (80, 9), (100, 50), (128, 64), (128, 1), (128, 31), (130, 64), (200, 99), (256, 128), (255, 100),
          (300, 0), (1024, 512), (1001, 333), (1024, 1), (1023, 1), (1023, 511)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width, pairs", SHAPES)
def test_widths(dtype, interleaved, width, pairs):
    query, key, positions = _inputs(9, 3, 2, width, dtype, width + pairs)
    _check(query, key, positions, _frequencies(pairs), interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens, heads, key_heads", [(1, 1, 1), (1, 64, 8), (2, 1, 0), (3, 0, 5), (17, 13, 13), (33, 7, 1),
                                                      (257, 32, 8), (5000, 2, 1)])
@pytest.mark.parametrize("width, pairs", [(128, 64), (40, 9)])
def test_tokens_and_heads(dtype, interleaved, tokens, heads, key_heads, width, pairs):
    query, key, positions = _inputs(tokens, heads, key_heads, width, dtype, tokens)
    _check(query, key, positions, _frequencies(pairs), interleaved, magnitude=1.125)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(dtype, interleaved):
    query, key, _ = _inputs(8, 4, 2, 64, dtype, 5)
    positions = torch.tensor([0, 1, 10**6, 10**6 + 1, 2**31 - 1, 2**31, -(2**31), 123456789])
    _check(query, key, positions, _frequencies(32), interleaved)
    _check(query, key, positions, autosage_amd.rotary_frequencies(64, scaling="ramp", factor=8.0, original_length=4096),
           interleaved, magnitude=1.2079)


def test_float32_is_exact_at_every_angle():
    """Angles from one pair: positions 0 to 60,000 at frequencies that pass through all of the circle."""
    positions = torch.arange(60000)
    ones = torch.zeros(60000, 1, 2)
    ones[..., 0] = 1.0
    for frequency in (0.1, 1.0, 2.0 * torch.pi / 8, 3.0e-5):
        f = torch.tensor([frequency], dtype=torch.float64)
        got, _ = autosage_amd.rotary_positions(ones.cuda(), None, positions.cuda(), f.cuda())
        want = plain_turn(ones, positions, f, False)
        # one step of sine and cosine, and the angle's 2^-52 of 10^4 turns
        assert (got.double().cpu() - want).abs().max() <= 2.0**-23 + 2.0**-36


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width, pairs", [(64, 32), (40, 9), (64, 8)])
def test_strided_rows(dtype, interleaved, width, pairs):
    """Slices of one projection, heads in another order, rows that begin anywhere, rows that are not contiguous."""
    query, key, positions = _inputs(21, 6, 2, width, dtype, 7)
    frequencies = _frequencies(pairs)
    wide = torch.cat((query, key, key), 1).cuda()
    got = autosage_amd.rotary_positions(wide[:, :6], wide[:, 6:8], positions.cuda(), frequencies.cuda(),
                                        interleaved=interleaved)
    want = _check(query, key, positions, frequencies, interleaved)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    def turned(t):
        return t.cuda().transpose(0, 1).contiguous().transpose(0, 1)

    def shifted(t):
        room = torch.zeros(t.size(0), t.size(1), t.size(2) + 3, dtype=t.dtype, device="cuda")
        room[..., 1:-2] = t.cuda()
        return room[..., 1:-2]

    def spread(t):
        room = torch.zeros(*t.shape, 2, dtype=t.dtype, device="cuda")
        room[..., 0] = t.cuda()
        return room[..., 0]

    def repeated(t):
        return t[:1].cuda().expand(t.size(0), -1, -1)

    for move in (turned, shifted, spread):
        assert all(torch.equal(a, b) for a, b in zip(_check(query, key, positions, frequencies, interleaved, move=move), want))
    _check(query[:1].expand(21, -1, -1), key[:1].expand(21, -1, -1), positions, frequencies, interleaved, move=repeated)
    every = torch.stack((positions, positions), 1).cuda()[:, 0]  # positions that are not contiguous, and 32-bit ones
    for p in (every, positions.int().cuda()):
        got = autosage_amd.rotary_positions(wide[:, :6], wide[:, 6:8], p, frequencies.cuda(), interleaved=interleaved)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width, pairs", [(64, 32), (40, 9)])
def test_gradients(dtype, interleaved, width, pairs):
    query, key, positions = _inputs(30, 5, 2, width, dtype, 9)
    frequencies = _frequencies(pairs)
    gen = torch.Generator().manual_seed(10)
    grads = [torch.randn(t.shape, generator=gen).to(dtype) for t in (query, key)]
    leaves = [t.cuda().requires_grad_() for t in (query, key)]
    out = autosage_amd.rotary_positions(*leaves, positions.cuda(), frequencies.cuda(), interleaved=interleaved,
                                        magnitude=0.75)
    got = torch.autograd.grad(out, leaves, [g.cuda() for g in grads], retain_graph=True)
    for g, y in zip(grads, got):
        assert_turned(y, plain_turn(g, positions, frequencies, interleaved, 0.75, inverse=True), g, pairs, 0.75)
    # one result alone, one input alone, gradients that are expanded, the registered operator
    alone = torch.autograd.grad(out[1], leaves, grads[1].cuda(), allow_unused=True, retain_graph=True)
    assert alone[0] is None and torch.equal(alone[1], got[1])
    total = torch.autograd.grad(out[0].sum() + out[1].sum(), leaves, retain_graph=True)
    ones = torch.ones_like(query)
    assert_turned(total[0], plain_turn(ones, positions, frequencies, interleaved, 0.75, inverse=True), ones, pairs, 0.75)
    half = autosage_amd.rotary_positions(leaves[0], key.cuda(), positions.cuda(), frequencies.cuda(),
                                         interleaved=interleaved, magnitude=0.75)
    assert torch.equal(torch.autograd.grad(half[0], leaves[0], grads[0].cuda())[0], got[0])
    assert torch.equal(half[1], out[1])
    named = torch.ops.autosage.rotary_positions(*leaves, positions.cuda(), frequencies.cuda(), interleaved, 0.75)
    again = torch.autograd.grad(named, leaves, [g.cuda() for g in grads])
    assert all(torch.equal(a, b) for a, b in zip((*named, *again), (*out, *got)))
    single, empty = torch.ops.autosage.rotary_positions(leaves[0], None, positions.cuda(), frequencies.cuda(), interleaved,
                                                        0.75)
    assert empty.numel() == 0 and torch.equal(torch.autograd.grad(single, leaves[0], grads[0].cuda())[0], got[0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(interleaved):
    """Linear: the difference of two calls is the call of the difference; <g, J d> = <J^T g, d>."""
    query, key, positions = _inputs(11, 3, 1, 24, torch.float32, 11)
    frequencies = _frequencies(8).cuda()
    q = query.cuda().requires_grad_()

    def turn(x):
        return autosage_amd.rotary_positions(x, None, positions.cuda(), frequencies, interleaved=interleaved)[0]

    step, g = torch.randn_like(q), torch.randn_like(q)
    slope = (turn(q + step) - turn(q - step)).double() / 2
    grad = torch.autograd.grad(turn(q), q, g)[0]
    # 792 products each off by a few 2^-24 of numbers below 10
    with torch.no_grad():
        off = abs(float((slope * g.double()).sum() - (grad.double() * step.double()).sum()))
    assert off <= 792 * 100 * 2.0**-22


def test_second_gradients_forward_mode_and_transforms():
    query, key, positions = _inputs(7, 3, 2, 24, torch.float32, 12)
    q, k, p, f = query.cuda(), key.cuda(), positions.cuda(), _frequencies(8).cuda()

    def turn(q, k):
        return autosage_amd.rotary_positions(q, k, p, f, magnitude=1.5)

    want = turn(q, k)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    with torch.autograd.forward_ad.dual_level():
        out = turn(torch.autograd.forward_ad.make_dual(q, dq), torch.autograd.forward_ad.make_dual(k, dk))
        tangents = [torch.autograd.forward_ad.unpack_dual(t).tangent for t in out]
        one = torch.autograd.forward_ad.unpack_dual(turn(torch.autograd.forward_ad.make_dual(q, dq), k)[0]).tangent
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.ops.autosage.rotary_positions(torch.autograd.forward_ad.make_dual(q, dq), None, p, f)
    assert all(torch.equal(a, b) for a, b in zip(tangents, turn(dq, dk))) and torch.equal(one, tangents[0])
    x = q.clone().requires_grad_()
    grad, = torch.autograd.grad(turn(x, k)[0], x, dq, create_graph=True)
    # the gradient does not depend on x, but on what comes in
    g = dq.clone().requires_grad_()
    grad, = torch.autograd.grad(turn(x, k)[0], x, g, create_graph=True)
    assert torch.equal(torch.autograd.grad(grad, g, q)[0], want[0])
    loss = torch.func.grad(lambda a: (turn(a, k)[0] * dq).sum())(q)
    assert torch.equal(loss, torch.autograd.grad(turn(x, k)[0], x, dq)[0])
    batch = torch.stack((q, dq))
    many = torch.vmap(lambda a: turn(a, k))(batch)
    assert torch.equal(many[0], torch.stack((want[0], turn(dq, k)[0]))) and torch.equal(many[1][1], want[1])
    alone = torch.vmap(lambda a: autosage_amd.rotary_positions(a, None, p, f)[0], in_dims=2, out_dims=2)(
        torch.stack((q, dq), 2))
    assert torch.equal(alone[:, :, 1], autosage_amd.rotary_positions(dq, None, p, f)[0])
    places = torch.stack((p, p + 5))
    moved = torch.vmap(lambda at: autosage_amd.rotary_positions(q, k, at, f))(places)
    assert torch.equal(moved[0][1], autosage_amd.rotary_positions(q, k, p + 5, f)[0])
    _, push = torch.func.jvp(lambda a: turn(a, k)[0], (q,), (dq,))
    assert torch.equal(push, turn(dq, k)[0])


def test_infinite_and_nan_rows():
    """They stay in their pair, and what is not turned stays as it is."""
    query, key, positions = _inputs(5, 2, 1, 24, torch.bfloat16, 13)
    query[1, 0, 3], query[2, 1, 20], query[3, 0, 9] = float("nan"), float("inf"), float("inf")
    got, _ = autosage_amd.rotary_positions(query.cuda(), None, positions.cuda(), _frequencies(8).cuda())
    want = query.clone()
    odd = ~got.isfinite().cpu()
    assert odd[1, 0, 3] and odd[1, 0, 11] and odd[3, 0, 9] and odd[3, 0, 1] and got[2, 1, 20] == float("inf")
    assert int(odd.sum()) == 5 and torch.equal(got[..., 16:].cpu().nan_to_num(1.0), want[..., 16:].nan_to_num(1.0))


def test_refusals():
    query, key, positions = _inputs(5, 2, 1, 24, torch.float32, 14)
    f = _frequencies(8).cuda()
    q, p = query.cuda(), positions.cuda()
    with pytest.raises(TypeError, match="native rotary positions"):
        autosage_amd.rotary_positions(q.double(), None, p, f)
    with pytest.raises(ValueError, match="on the device"):
        autosage_amd.rotary_positions(q, None, positions, f)
    with pytest.raises(ValueError, match="at most 1024"):
        autosage_amd.rotary_positions(torch.zeros(5, 1, 1025, device="cuda"), None, p, f)
    with pytest.raises(RuntimeError, match="no gradient for frequencies"):
        autosage_amd.rotary_positions(q, None, p, f.clone().requires_grad_())
    none = autosage_amd.rotary_positions(q[:0], q[:0], p[:0], f)
    assert none[0].shape == (0, 2, 24)


def test_offsets_beyond_32_bits():
    tokens, heads, width = 70000, 256, 128  # 2.3e9 elements
    query = torch.zeros(tokens, heads, width, dtype=torch.bfloat16, device="cuda")
    rows = torch.randn(3, heads, width, generator=torch.Generator().manual_seed(15)).bfloat16()
    at = torch.tensor([0, 33000, tokens - 1])
    query[at.cuda()] = rows.cuda()
    positions = torch.arange(tokens)
    got, _ = autosage_amd.rotary_positions(query, None, positions.cuda(), _frequencies(64).cuda())
    assert_turned(got[at.cuda()], plain_turn(rows, at, _frequencies(64), False), rows, 64)
    assert int(got.count_nonzero()) <= rows.numel()


def test_capture_and_replay_of_a_training_step():
    """Forward and gradients in a graph, eager steps of other leaves between the replays."""
    query, key, positions = _inputs(300, 8, 2, 64, torch.bfloat16, 16)
    f = _frequencies(32).cuda()
    q, k, p = query.cuda().requires_grad_(), key.cuda().requires_grad_(), positions.cuda()
    grads = torch.randn_like(q), torch.randn_like(k)

    def step(q, k):
        out = autosage_amd.rotary_positions(q, k, p, f)
        return (*(t.detach() for t in out), *torch.autograd.grad(out, (q, k), grads))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(q, k)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(q, k)
    for turn in range(4):
        with torch.no_grad():
            q.normal_()
            k.normal_()
            p.random_(0, 10000)
            grads[0].normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = step(q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_())
        assert all(torch.equal(a, b) for a, b in zip(results, want))


def test_another_stream():
    query, key, positions = _inputs(3000, 8, 2, 64, torch.bfloat16, 17)
    q, k, p, f = query.cuda(), key.cuda(), positions.cuda(), _frequencies(32).cuda()
    want = autosage_amd.rotary_positions(q, k, p, f)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(autosage_amd.rotary_positions(q, k, p, f))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))
