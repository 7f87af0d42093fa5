"""Learned bias of the distance between two nodes, by buckets.

Attention over the edges of a CSR graph knows which keys a query sees, not how
far they are.  ``csr_position_bias`` gives every edge and head a learned number
for the distance between its two nodes, to be added to the edge scores in front
of the row softmax; ``paged_attention`` adds the same numbers when the tokens of
a sequence are answered one at a time.

With ``n`` buckets for one side of the query and ``E = n // 2``, distances below
``E`` have a bucket each and bucket ``E + j`` begins where
``(d / E) ** (n - E)`` reaches ``(max_distance / E) ** j``; the last bucket holds
everything farther.  The borders are found in integers, so that no logarithm's
last bit decides a bucket.  The reference's attention has no positions.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native
from .ops import load_native, native_load_error, validate_if_requested

MAX_BUCKETS = 256
_MAX_HEADS = 65535
# node ids that are positions may be any: rows of a part of a graph see columns of all of it
_MAX_NODES = 2**62
_DTYPES = {torch.float32: 0, **_native.DTYPES_16}


@functools.lru_cache(maxsize=256)
def bucket_borders(buckets: int, max_distance: int, bidirectional: bool = True) -> tuple[int, ...]:
    """The smallest distance of each bucket of one side of the query (half of
    ``buckets`` with ``bidirectional``, else all of them)."""
    if not 2 <= buckets <= MAX_BUCKETS:
        raise ValueError(f"the number of buckets must lie in [2, {MAX_BUCKETS}]")
    if bidirectional and buckets % 2 != 0:
        raise ValueError("a bidirectional bias needs an even number of buckets")
    side = buckets // 2 if bidirectional else buckets
    exact = side // 2
    if not max(exact, 1) < max_distance < 2**31:
        raise ValueError(f"max_distance must lie in ({max(exact, 1)}, 2^31)")
    if side == 1:
        return (0,)
    rest = side - exact
    borders = list(range(exact + 1))
    for j in range(1, rest):
        # the smallest d with d^rest >= exact^(rest - j) * max_distance^j
        goal = exact ** (rest - j) * max_distance**j
        low, high = borders[-1], max_distance
        while low < high:
            middle = (low + high) // 2
            if middle**rest >= goal:
                high = middle
            else:
                low = middle + 1
        borders.append(low)
    return tuple(borders)


@functools.lru_cache(maxsize=256)
def border_array(buckets: int, max_distance: int, bidirectional: bool):
    """``bucket_borders`` as the C array of the native calls (host memory)."""
    borders = bucket_borders(buckets, max_distance, bidirectional)
    return (ctypes.c_int32 * len(borders))(*borders)


def position_buckets(relative: torch.Tensor, buckets: int, max_distance: int, bidirectional: bool) -> torch.Tensor:
    """The bucket of every (key position - query position)."""
    borders = torch.tensor(bucket_borders(buckets, max_distance, bidirectional), device=relative.device)
    distance = relative.abs() if bidirectional else (-relative).clamp_min(0)
    found = torch.searchsorted(borders, distance, right=True) - 1
    return found + (relative > 0).long() * (buckets // 2) if bidirectional else found


def _check(crow, col, positions, table) -> None:
    if crow.ndim != 1 or col.ndim != 1 or crow.numel() < 1:
        raise ValueError("crow and col must be one-dimensional")
    if crow.dtype not in (torch.int32, torch.int64) or col.dtype not in (torch.int32, torch.int64):
        raise TypeError("crow and col must use integer indices")
    if table.ndim != 2 or table.size(1) < 1:
        raise ValueError("table must have shape [buckets, heads]")
    if not table.is_floating_point():
        raise TypeError("table must use a floating-point dtype")
    if not (crow.device == col.device == table.device):
        raise ValueError("crow, col, and table must be on the same device")
    if col.numel() > 0 and crow.numel() < 2:
        raise ValueError("edges without rows")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must use integers")
        if positions.ndim != 1 or positions.numel() != crow.numel() - 1:
            raise ValueError("positions must contain one entry per node")
        if positions.device != crow.device:
            raise ValueError("positions and crow must be on the same device")


def _long(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or (t.dtype == torch.long and t.is_contiguous()) else t.to(torch.long).contiguous()


def csr_position_bias_impl(crow, col, positions, table, max_distance, bidirectional, keep=True):
    """(bias [heads, edges], the edges' buckets: one byte each, none without ``keep``)."""
    _check(crow, col, positions, table)
    if table.dtype not in _DTYPES:
        raise TypeError("the native position bias supports float32, bfloat16 and float16 tables")
    buckets, heads = table.shape
    borders = border_array(buckets, max_distance, bool(bidirectional))
    crow, col, positions, table = _long(crow), _long(col), _long(positions), table.contiguous()
    validate_if_requested(crow, col, _MAX_NODES if positions is None else None)
    nnz = col.numel()
    out = torch.empty(heads, nnz, dtype=table.dtype, device=table.device)
    # whole words: the last one may reach behind the edges
    found = torch.empty((nnz + 3) // 4 * 4 if keep else 0, dtype=torch.uint8, device=table.device)
    if nnz == 0:
        return out, found
    n = crow.numel() - 1
    lib = _native.library()
    ws_bytes = lib.as_csr_position_bias_workspace_bytes(n, nnz, int(positions is not None))
    ws = _native._workspace(ws_bytes, table.device) if ws_bytes else None
    with _native._on(table.device):
        status = lib.as_csr_position_bias(
            crow.data_ptr(), col.data_ptr(), _native._ptr(positions), table.data_ptr(), out.data_ptr(),
            found.data_ptr() if keep else None, n, nnz, heads, buckets, borders, int(bool(bidirectional)),
            _DTYPES[table.dtype], _native._ptr(ws), ws_bytes, _native._stream(table.device))
    _native._raise(status, "autosage::csr_position_bias")
    return out, found


def csr_position_bias_backward_impl(found, grad, buckets):
    """dL/dtable [buckets, heads] from the edges' buckets and dL/dbias [heads, edges]."""
    if grad.ndim != 2 or grad.size(0) < 1 or found.ndim != 1 or found.numel() != (grad.size(1) + 3) // 4 * 4:
        raise ValueError("grad must have shape [heads, edges], with a bucket for every edge")
    if grad.dtype not in _DTYPES or found.dtype != torch.uint8:
        raise TypeError("the native position bias supports float32, bfloat16 and float16 gradients, and uint8 buckets")
    if grad.device != found.device:
        raise ValueError("grad and the buckets must be on the same device")
    found, grad = found.contiguous(), grad.contiguous()
    heads, nnz = grad.shape
    table = torch.empty(buckets, heads, dtype=grad.dtype, device=grad.device)
    lib = _native.library()
    ws = _native._workspace(lib.as_csr_position_bias_backward_workspace_bytes(nnz, heads, buckets), grad.device)
    with _native._on(grad.device):
        status = lib.as_csr_position_bias_backward(
            found.data_ptr(), grad.data_ptr(), table.data_ptr(), nnz, heads, buckets, _DTYPES[grad.dtype],
            ws.data_ptr(), ws.numel(), _native._stream(grad.device))
    _native._raise(status, "autosage::csr_position_bias (backward)")
    return table


def has_tangent(*tensors) -> bool:
    """Whether one of the tensors carries a forward-mode derivative."""
    # without a level nothing has one; asking each tensor would take 0.3 us
    if getattr(forward_ad, "_current_level", 0) < 0:
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _refuse_tangent(t) -> None:
    if has_tangent(t):
        raise RuntimeError("the registered operators of the position bias have no forward-mode derivative: "
                           "call autosage_amd.csr_position_bias")


def _registered(crow, col, positions, table, max_distance, bidirectional):
    _refuse_tangent(table)
    return csr_position_bias_impl(crow, col, positions, table, max_distance, bidirectional)


def _registered_backward(found, grad, buckets):
    _refuse_tangent(grad)
    return csr_position_bias_backward_impl(found, grad, buckets)


SCHEMAS = {
    # the bias, and the edges' buckets for its gradient
    "csr_position_bias": (
        "csr_position_bias(Tensor crow, Tensor col, Tensor? positions, Tensor table, int max_distance, "
        "bool bidirectional) -> (Tensor, Tensor)",
        _registered,
    ),
    "csr_position_bias_backward": (
        "csr_position_bias_backward(Tensor found, Tensor grad, int buckets) -> Tensor",
        _registered_backward,
    ),
}


# Inside torch.func's transforms (grad, vmap, jvp and what they make up) tensors are
# wrapped, and only functions with rules for them reach the kernels.
_transforms_active = getattr(torch._C, "_are_functorch_transforms_active", lambda: False)


def _bucket_sums(found, grad, buckets):
    """dL/dtable, with a history where it is differentiated itself."""
    if (torch.is_grad_enabled() and grad.requires_grad) or _transforms_active() or has_tangent(grad):
        return _BucketSums.apply(grad, found, buckets)
    return csr_position_bias_backward_impl(found, grad, buckets)


# The public function's gradients: the dispatcher's own wrapping of an operator's
# gradient takes some 100 us a training step, these 50, the kernels 20 (720,000
# edges, 5 heads).
class _PositionBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, crow, col, positions, max_distance, bidirectional):
        out, found = csr_position_bias_impl(crow, col, positions, table, max_distance, bidirectional)
        ctx.save_for_backward(found)
        ctx.buckets = table.size(0)
        return out

    @staticmethod
    def backward(ctx, grad):
        return _bucket_sums(ctx.saved_tensors[0], grad, ctx.buckets), None, None, None, None, None


# The same for every other derivative and torch.func's transforms: torch asks for the
# context in a call of its own where more than the gradient is defined, which costs
# the host time that the class above saves.
class _PositionBiasTransformed(torch.autograd.Function):
    @staticmethod
    def forward(table, crow, col, positions, max_distance, bidirectional):
        return csr_position_bias_impl(crow, col, positions, table, max_distance, bidirectional)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _setup(ctx, (None, None, None, inputs[0]), output)
        ctx.save_for_forward(output[1])
        ctx.edges = output[0].size(1)

    @staticmethod
    def backward(ctx, grad, _):
        # apply also unwraps what a transform that is over has saved
        grad_table = None if grad is None else _BucketSums.apply(grad, ctx.saved_tensors[0], ctx.buckets)
        return grad_table, None, None, None, None, None

    @staticmethod
    def jvp(ctx, table, *_):
        return _lookup(table, ctx.saved_tensors[0], ctx.edges), None

    @staticmethod
    def vmap(info, in_dims, *inputs):
        table = inputs[0]
        if in_dims[1:4] != (None, None, None) or info.batch_size * table.size(-1) > _MAX_HEADS:
            return _one_by_one(_PositionBiasTransformed, info, in_dims, inputs)
        # the tables' heads side by side
        table = table.movedim(in_dims[0], 1)
        out, found = _PositionBiasTransformed.apply(table.flatten(1), *inputs[1:])
        return (out.unflatten(0, table.shape[1:]), found), (0, None)


class _BucketSums(torch.autograd.Function):
    @staticmethod
    def forward(grad, found, buckets):
        return csr_position_bias_backward_impl(found, grad, buckets)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.save_for_backward(inputs[1])
        ctx.save_for_forward(inputs[1])
        ctx.edges, ctx.buckets = inputs[0].size(1), inputs[2]

    @staticmethod
    def backward(ctx, grad_table):
        return _lookup(grad_table, ctx.saved_tensors[0], ctx.edges), None, None

    @staticmethod
    def jvp(ctx, grad, *_):
        return _BucketSums.apply(grad, ctx.saved_tensors[0], ctx.buckets)

    @staticmethod
    def vmap(info, in_dims, grad, found, buckets):
        if in_dims[1] is None:
            rows = grad.movedim(in_dims[0], 0)
            if info.batch_size * rows.size(1) <= _MAX_HEADS:
                return _BucketSums.apply(rows.flatten(0, 1), found, buckets).unflatten(1, rows.shape[:2]), 1
        return _one_by_one(_BucketSums, info, in_dims, (grad, found, buckets))


def _one_by_one(function, info, in_dims, inputs):
    """The vmap rule of calls that differ in more than their tables: one call each."""
    results = [function.apply(*(x if d is None else x.select(d, i) for x, d in zip(inputs, in_dims)))
               for i in range(info.batch_size)]
    if isinstance(results[0], tuple):
        return tuple(torch.stack(parts) for parts in zip(*results)), (0,) * len(results[0])
    return torch.stack(results), 0


def _lookup(table, found, edges):
    """The bias of edges whose buckets are known: linear in the table, and the transpose of the sums."""
    return table.t()[:, found[:edges].long()]


def _setup(ctx, inputs, output) -> None:
    ctx.buckets = inputs[3].size(0)
    ctx.save_for_backward(output[1])
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)


def _backward(ctx, grad, _):
    wanted = grad is not None and ctx.needs_input_grad[3]
    grad_table = _bucket_sums(ctx.saved_tensors[0], grad, ctx.buckets) if wanted else None
    return None, None, None, grad_table, None, None


def _sums_setup(ctx, inputs, output) -> None:
    ctx.save_for_backward(inputs[0])
    ctx.edges = inputs[1].size(1)


def _sums_backward(ctx, grad_table):
    return None, _lookup(grad_table, ctx.saved_tensors[0], ctx.edges), None


def register_autograd() -> None:
    """Attaches the gradients to the registered operators."""
    torch.library.register_autograd("autosage::csr_position_bias", _backward, setup_context=_setup)
    torch.library.register_autograd("autosage::csr_position_bias_backward", _sums_backward, setup_context=_sums_setup)


def _cpu_position_bias(crow, col, positions, table, max_distance, bidirectional) -> torch.Tensor:
    crow, col = crow.long(), col.long()
    rows = torch.repeat_interleave(torch.arange(crow.numel() - 1, device=col.device), crow[1:] - crow[:-1])
    relative = col - rows if positions is None else positions.long()[col] - positions.long()[rows]
    return table.t()[:, position_buckets(relative, table.size(0), max_distance, bidirectional)]


def csr_position_bias(crow, col, table, *, max_distance: int, bidirectional: bool = True,
                      positions=None) -> torch.Tensor:
    """The learned bias of every edge: ``out[h, e] = table[bucket, h]`` for the
    bucket of the position of ``col[e]`` minus that of the edge's row.

    ``table`` is ``[buckets, heads]``, float32, bfloat16 or float16; the result
    is ``[heads, edges]`` of its dtype, one row for each head's scores, with a
    gradient for ``table`` (the sum over each bucket's edges, in a fixed order).
    Node ids are positions (and columns may then lie beyond the rows) unless
    ``positions`` (one integer per node, within +-2^62) gives them.  With ``bidirectional`` half of the buckets are for keys behind the
    query; without it a key behind the query counts as distance 0."""
    _check(crow, col, positions, table)
    max_distance = int(max_distance)
    bucket_borders(table.size(0), max_distance, bool(bidirectional))
    if not table.is_cuda:
        return _cpu_position_bias(crow, col, positions, table, max_distance, bool(bidirectional))
    if not load_native():
        raise RuntimeError(f"AutoSAGE CUDA extension is unavailable: {native_load_error()}")
    crow, col, positions = _long(crow), _long(col), _long(positions)
    if _transforms_active() or has_tangent(table):
        return _PositionBiasTransformed.apply(table, crow, col, positions, max_distance, bool(bidirectional))[0]
    if torch.is_grad_enabled() and table.requires_grad:
        return _PositionBias.apply(table, crow, col, positions, max_distance, bool(bidirectional))
    return csr_position_bias_impl(crow, col, positions, table, max_distance, bool(bidirectional), keep=False)[0]


__all__ = ["bucket_borders", "csr_position_bias", "position_buckets"]
