"""Rotary positions: queries and keys turned by the angle of their position.

The first ``2n`` numbers of a row are ``n`` pairs, each turned by the row's position times
the pair's frequency.  The product of a query with a key then depends on how far
apart they are and on nothing else of their positions, so that keys can be turned
once, when they are written to a cache (``paged_cache_write``), and attention
(``paged_attention``, or the attention over the edges of a graph with a position for every node)
needs no term for the distance.

The reference's attention has no positions.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _native
from .ops import load_native, native_load_error
from .position import has_tangent

MAX_WIDTH = 1024
_DTYPES = {torch.float32: 0, **_native.DTYPES_16}
_TwoStrides = ctypes.c_int64 * 2
_NO_GRADIENT = "rotary_positions has no gradient for frequencies"


def rotary_frequencies(dims: int, *, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, turns: tuple[float, float] = (1.0, 32.0),
                       device=None) -> torch.Tensor:
    """The angles between one position and the next of the ``dims / 2`` pairs, ``base ** (-2 i / dims)``
    radians, in float64, for ``rotary_positions``.

    ``scaling`` stretches them for contexts that are ``factor`` times as long as those a model was
    trained for: ``"linear"`` divides every one by ``factor``; ``"base"`` takes ``base * factor ** (dims /
    (dims - 2))``, which leaves the first and divides the last by ``factor``; ``"ramp"`` leaves pairs that turn
    ``turns[1]`` times or more within ``original_length`` positions, divides those that turn ``turns[0]`` times or
    less, and mixes both in between, by how often a pair turns.  (A ``magnitude`` of ``0.1 * log(factor) +
    1`` in ``rotary_positions`` belongs to it.)"""
    dims = int(dims)
    if dims < 2 or dims % 2 != 0:
        raise ValueError("dims must be positive and even")
    if not (base > 0 and math.isfinite(base) and factor > 0 and math.isfinite(factor)):
        raise ValueError("base and factor must be positive")
    if scaling not in (None, "linear", "base", "ramp"):
        raise ValueError("scaling must be None, 'linear', 'base' or 'ramp'")
    if scaling is None and factor != 1.0:
        raise ValueError("a factor belongs to a scaling")
    if (scaling == "ramp") != (original_length is not None):
        raise ValueError("original_length belongs to scaling='ramp'")
    if scaling == "base":
        if dims == 2:
            raise ValueError("scaling='base' needs two pairs or more")
        base = base * factor ** (dims / (dims - 2))
    frequencies = float(base) ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if scaling == "linear":
        frequencies = frequencies / factor
    if scaling == "ramp":
        few, many = turns
        if not (original_length > 0 and 0 <= few < many):
            raise ValueError("original_length must be positive and turns ascend from 0 or more")
        kept = ((original_length * frequencies / (2 * math.pi) - few) / (many - few)).clamp(0.0, 1.0)
        frequencies = frequencies * kept + frequencies / factor * (1.0 - kept)
    return frequencies if device is None else frequencies.to(device)


def _require(condition: bool, error: type, message: str) -> None:
    if not condition:
        raise error(message)


def _check(query, key, positions, frequencies) -> None:
    if (query.dim() == 3 and (key is None or (key.dim() == 3 and key.dtype is query.dtype
                                              and key.size(0) == query.size(0) and key.size(2) == query.size(2)
                                              and key.device == query.device))
            and query.is_floating_point() and query.size(2) >= 1 and not has_tangent(frequencies)
            and positions.dtype is torch.long and positions.shape == query.shape[:1]
            and frequencies.dtype is torch.float64 and frequencies.dim() == 1
            and 2 * frequencies.size(0) <= query.size(2) and not frequencies.requires_grad
            and positions.device == frequencies.device == query.device):
        return
    _require(query.ndim == 3 and (key is None or key.ndim == 3), ValueError,
             "query and key must have shape [tokens, heads, width]")
    _require(query.is_floating_point() and (key is None or key.dtype == query.dtype), TypeError,
             "query and key must both use the same floating-point dtype")
    _require(key is None or (key.size(0) == query.size(0) and key.size(2) == query.size(2)), ValueError,
             "query and key must have the same tokens and width")
    _require(query.size(2) >= 1, ValueError, "a row has at least one number")
    _require(positions.dtype in (torch.int32, torch.int64), TypeError, "positions must use integers")
    _require(positions.shape == query.shape[:1], ValueError, "positions must contain one entry per token")
    _require(frequencies.dtype in (torch.float32, torch.float64), TypeError,
             "frequencies must use float64 (or float32)")
    _require(frequencies.ndim == 1 and 2 * frequencies.size(0) <= query.size(2), ValueError,
             "frequencies must contain one entry per pair, and the pairs fit the width")
    for name, t in (("key", key), ("positions", positions), ("frequencies", frequencies)):
        _require(t is None or t.device == query.device, ValueError, f"{name} must be on the device of query")
    _require(not (torch.is_grad_enabled() and frequencies.requires_grad), RuntimeError, _NO_GRADIENT)
    _require(not has_tangent(frequencies), RuntimeError, "rotary_positions has no derivative for frequencies")


def _cpu_turn(x, cos, sin, interleaved: bool):
    pairs = cos.size(-1)
    wide = x[..., :2 * pairs].to(torch.promote_types(x.dtype, torch.float32))
    cos, sin = cos.to(wide.dtype), sin.to(wide.dtype)
    a, b = (wide[..., ::2], wide[..., 1::2]) if interleaved else (wide[..., :pairs], wide[..., pairs:])
    turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1 if interleaved else -2).flatten(-2)
    return torch.cat((turned.to(x.dtype), x[..., 2 * pairs:]), -1)


def _cpu_rotary(query, key, positions, frequencies, interleaved, magnitude):
    angle = positions.double()[:, None, None] * frequencies.double()
    cos, sin = angle.cos() * magnitude, angle.sin() * magnitude
    return (_cpu_turn(query, cos, sin, interleaved),
            None if key is None else _cpu_turn(key, cos, sin, interleaved))


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.size(-1) == 1 or t.stride(-1) == 1 else t.contiguous()


def rotary_positions_impl(query, key, positions, frequencies, interleaved, magnitude, inverse):
    """(query, key) turned, either of which may be None."""
    some = key if query is None else query
    _require(some.dtype in _DTYPES, TypeError, "native rotary positions support float32, bfloat16 and float16")
    tokens, _, width = some.shape
    _require(width <= MAX_WIDTH, ValueError, f"the width must be at most {MAX_WIDTH}")
    lib = _native.library()
    ins = [None if t is None else _rows(t) for t in (query, key)]
    outs = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (query, key)]
    args = []
    for t, out in zip(ins, outs):
        args += ([None, None, None, 0] if t is None else
                 [t.data_ptr(), _TwoStrides(t.stride(0), t.stride(1)), out.data_ptr(), t.size(1)])
    with _native._on(some.device):
        status = lib.as_rotary_positions(
            *args, positions.data_ptr(), frequencies.data_ptr(), tokens, width, frequencies.size(0), int(interleaved),
            int(inverse), magnitude, _DTYPES[some.dtype], _native._stream(some.device))
    _native._raise(status, "autosage::rotary_positions")
    return outs[0], outs[1]


# Inside torch.func's transforms tensors are wrapped, and only functions with rules for
# them reach the kernel.
_transforms_active = getattr(torch._C, "_are_functorch_transforms_active", lambda: False)


def _turn(query, key, positions, frequencies, interleaved, magnitude, inverse):
    given = [t for t in (query, key) if t is not None]
    if _transforms_active() or has_tangent(*given):
        return _RotaryTransformed.apply(query, key, positions, frequencies, interleaved, magnitude, inverse)
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        return _Rotary.apply(query, key, positions, frequencies, interleaved, magnitude, inverse)
    return rotary_positions_impl(query, key, positions, frequencies, interleaved, magnitude, inverse)


def _turn_back(ctx, grad_query, grad_key):
    positions, frequencies = ctx.saved_tensors
    if grad_query is None and grad_key is None:
        return None, None
    interleaved, magnitude, inverse = ctx.how
    return _turn(grad_query, grad_key, positions, frequencies, interleaved, magnitude, not inverse)


# The public function's gradient: the other way round, with the other sign, and so itself
# differentiable.
class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, positions, frequencies, interleaved, magnitude, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, frequencies)
        ctx.how = interleaved, magnitude, inverse
        return rotary_positions_impl(query, key, positions, frequencies, interleaved, magnitude, inverse)

    @staticmethod
    def backward(ctx, grad_query, grad_key):
        wanted = [g if need else None for g, need in zip((grad_query, grad_key), ctx.needs_input_grad)]
        return (*_turn_back(ctx, *wanted), None, None, None, None, None)


# The same for every other derivative and torch.func's transforms: torch asks for the context in a
# call of its own there, which costs the host time that the class above saves.
class _RotaryTransformed(torch.autograd.Function):
    @staticmethod
    def forward(query, key, positions, frequencies, interleaved, magnitude, inverse):
        return rotary_positions_impl(query, key, positions, frequencies, interleaved, magnitude, inverse)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.save_for_backward(*inputs[2:4])
        ctx.save_for_forward(*inputs[2:4])
        ctx.how = inputs[4:]

    @staticmethod
    def backward(ctx, grad_query, grad_key):
        return (*_turn_back(ctx, grad_query, grad_key), None, None, None, None, None)

    @staticmethod
    def jvp(ctx, query, key, *_):
        return _turn(query, key, *ctx.saved_tensors, *ctx.how)

    @staticmethod
    def vmap(info, in_dims, *inputs):
        rows, rest = inputs[:2], inputs[2:]
        if info.batch_size == 0:
            none = [None if x is None else (x.expand(0, *x.shape) if d is None else x.movedim(d, 0)).clone()
                    for x, d in zip(rows, in_dims)]
            return tuple(none), tuple(None if x is None else 0 for x in none)
        if in_dims[2] is None and in_dims[3] is None:
            # the batch's heads side by side
            flat = [x if d is None else x.movedim(d, 1).flatten(1, 2) for x, d in zip(rows, in_dims)]
            if all(x is None or x.size(1) <= 65535 for x in flat):
                out = _RotaryTransformed.apply(*flat, *rest)
                return (tuple(x if d is None else x.unflatten(1, (info.batch_size, -1)) for x, d in zip(out, in_dims)),
                        tuple(None if d is None else 1 for d in in_dims[:2]))
        results = [_RotaryTransformed.apply(*(x if d is None else x.select(d, i) for x, d in zip(inputs, in_dims)))
                   for i in range(info.batch_size)]
        return (tuple(None if parts[0] is None else torch.stack(parts) for parts in zip(*results)),
                tuple(None if x is None else 0 for x in results[0]))


def _registered(query, key, positions, frequencies, interleaved=False, magnitude=1.0, inverse=False):
    if has_tangent(query, key):
        raise RuntimeError("the registered operator of rotary positions has no forward-mode derivative: "
                           "call autosage_amd.rotary_positions")
    _check(query, key, positions, frequencies)
    out = rotary_positions_impl(query, key, *_plan(positions, frequencies), bool(interleaved), float(magnitude),
                                bool(inverse))
    return out[0], query.new_empty(0) if key is None else out[1]


SCHEMAS = {
    # the key's result is empty where there is no key
    "rotary_positions": (
        "rotary_positions(Tensor query, Tensor? key, Tensor positions, Tensor frequencies, bool interleaved=False, "
        "float magnitude=1.0, bool inverse=False) -> (Tensor, Tensor)",
        _registered,
    ),
}


def _setup(ctx, inputs, output) -> None:
    # the operator itself runs without a history, where nothing shows that there will be one
    _require(not ctx.needs_input_grad[3], RuntimeError, _NO_GRADIENT)
    ctx.set_materialize_grads(False)
    # as the kernel reads them, which is not how they may have been given
    ctx.save_for_backward(*_plan(*inputs[2:4]))
    ctx.how = (*inputs[4:], *(False, 1.0, False)[len(inputs) - 4:])  # arguments that are the default may be left out
    ctx.with_key = inputs[1] is not None


def _backward(ctx, grad_query, grad_key):
    positions, frequencies = ctx.saved_tensors
    grads = _turn_back(ctx, grad_query, grad_key if ctx.with_key else None)
    return (*grads, None, None, None, None, None)


def register_autograd() -> None:
    """Attaches the gradient to the registered operator."""
    torch.library.register_autograd("autosage::rotary_positions", _backward, setup_context=_setup)


def _plan(positions, frequencies):
    return (positions if positions.dtype == torch.long and positions.is_contiguous() else
            positions.to(torch.long).contiguous(),
            frequencies if frequencies.dtype == torch.float64 and frequencies.is_contiguous() else
            frequencies.to(torch.float64).contiguous())


def rotary_positions(query, key, positions, frequencies, *, interleaved: bool = False, magnitude: float = 1.0):
    """(query, key) with the first ``2 * len(frequencies)`` numbers of every row turned by ``positions[token] *
    frequencies[i]`` radians for pair ``i``, and multiplied by ``magnitude``: ``(a, b)`` becomes ``(a cos - b sin, a
    sin + b cos)``.  The rest of a row stays as it is.

    ``query`` is ``[tokens, heads, width]`` and ``key``, which may be None, ``[tokens, key heads, width]``, of the same
    dtype (on the GPU float32, bfloat16 or float16, and a width of at most 1,024), and may be slices of one projection.
    Pairs are ``(x[i], x[i + n])``, or with ``interleaved`` ``(x[2 i], x[2 i + 1])``.  ``frequencies``
    (``rotary_frequencies``) are float64; ``positions`` one integer per token, the ``positions`` of
    ``paged_cache_resize`` or the numbers of a graph's nodes.

    The angle is computed and reduced in float64, off by less than 2^-51 of the turns, so that a
    position of a million is as good as one of ten: float32 does not show it up to 2^24 turns. Beyond, the
    error grows with them (2^-20 of a turn at 2^31, and positions beyond 2^53 are rounded themselves).
    The pairs are turned in float32 and rounded once.  Both results are new, contiguous tensors with
    gradients of every order, forward-mode derivatives and rules for ``torch.func``'s transforms; a derivative for
    ``frequencies`` is refused."""
    _check(query, key, positions, frequencies)
    interleaved, magnitude = bool(interleaved), float(magnitude)
    if not query.is_cuda:
        return _cpu_rotary(query, key, positions, frequencies, interleaved, magnitude)
    if not load_native():
        raise RuntimeError(f"AutoSAGE CUDA extension is unavailable: {native_load_error()}")
    return _turn(query, key, *_plan(positions, frequencies), interleaved, magnitude, False)


__all__ = ["rotary_frequencies", "rotary_positions"]
