"""Keys and values in pages, and attention of one new token over them.

A sequence that is answered token by token keeps the keys and values of its
tokens.  Here they lie in pages, ``[pages, heads, page_size, width]``, and a CSR
list says whose they are: sequence ``b`` has the pages
``page_idx[page_ptr[b]:page_ptr[b + 1]]`` in the order of its tokens.  A list may
be longer than the sequence needs so far (``page_ptr = arange(B + 1) * W`` makes
a table of ``W`` entries a sequence).

* ``paged_cache_write`` puts the rows of new tokens into their pages: as they
  are, as 8-bit numbers (``torch.float8_e4m3fn``) with one power of two for
  each token and head, or as 4-bit ones (``torch.float4_e2m1fn_x2``) with one
  for each 32 numbers of a row;
* ``paged_cache_read`` gives the rows of any run of tokens back;
* ``paged_attention`` is the attention of every sequence's last token over all
  tokens of the sequence, or over a window of the last ones.

On the GPU the three are native kernels on the current stream; nothing waits for
the device, so they can be captured into a graph and replayed while page lists,
lengths and tokens change in place.  CPU tensors run a torch composition.  The
reference computes attention over whole graphs and has no counterpart.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _env
from . import _native
from .ops import load_native, native_load_error
from .position import border_array, bucket_borders, has_tangent, position_buckets

E4M3 = torch.float8_e4m3fn
E2M1 = torch.float4_e2m1fn_x2  # two numbers in a byte
E8M0 = torch.float8_e8m0fnu
GROUP = 32  # numbers of a row of E2M1 that share an exponent
MAX_WIDTH = 256
_ROW_DTYPES = {torch.float32: 0, **_native.DTYPES_16}
_DTYPES = {**_ROW_DTYPES, E4M3: 3, E2M1: 5}
_CODED = (E4M3, E2M1)
_INTEGERS = (torch.int32, torch.int64)


def _require(condition: bool, error: type, message: str) -> None:
    if not condition:
        raise error(message)


def _check_rows(name: str, t: torch.Tensor) -> None:
    _require(t.size(-1) == 1 or t.stride(-1) == 1, ValueError, f"the rows of {name} must be contiguous")


def _width(pages: torch.Tensor) -> int:
    """Numbers in a row."""
    return pages.size(3) * 2 if pages.dtype is E2M1 else pages.size(3)


def _exponent_shape(pages: torch.Tensor) -> tuple:
    shape = tuple(pages.shape[:3])
    return (*shape, (pages.size(3) + GROUP // 2 - 1) // (GROUP // 2)) if pages.dtype is E2M1 else shape


# Each check asks for everything at once (a call of a few tokens is bound by the
# host: 10 us of checks one by one, 3 together); only where something is wrong do
# the conditions run one by one and name the first that fails.


def _check_cache(key_pages, value_pages, page_ptr, page_idx, key_exponents, value_exponents) -> None:
    dtype = key_pages.dtype
    key_shape, value_shape = key_pages.shape, value_pages.shape
    widest = MAX_WIDTH // 2 if dtype is E2M1 else MAX_WIDTH
    if (dtype in _DTYPES and value_pages.dtype is dtype and len(key_shape) == 4 and len(value_shape) == 4
            and key_shape[:3] == value_shape[:3] and key_pages.numel() > 0 and value_pages.numel() > 0
            and 1 < key_shape[3] <= widest and 1 < value_shape[3] <= widest
            and key_pages.stride(3) == 1 and value_pages.stride(3) == 1
            and page_ptr.dtype is torch.long and page_idx.dtype is torch.long and page_ptr.dim() == 1
            and page_idx.dim() == 1 and page_ptr.numel() >= 1
            and key_pages.get_device() == value_pages.get_device() == page_ptr.get_device() == page_idx.get_device()):
        if dtype not in _CODED:
            if key_exponents is None and value_exponents is None:
                return
        elif (key_exponents is not None and value_exponents is not None
                and key_exponents.dtype is value_exponents.dtype is (torch.int8 if dtype is E4M3 else E8M0)
                and key_exponents.shape == _exponent_shape(key_pages)
                and value_exponents.shape == _exponent_shape(value_pages)
                and (dtype is E4M3 or (key_exponents.stride(3) == 1 and value_exponents.stride(3) == 1))
                and key_exponents.get_device() == value_exponents.get_device() == key_pages.get_device()):
            return
    _require(key_pages.ndim == 4 and value_pages.ndim == 4 and key_pages.shape[:3] == value_pages.shape[:3],
             ValueError, "key_pages and value_pages must have shape [pages, heads, page_size, width]")
    _require(key_pages.dtype in _DTYPES and value_pages.dtype == key_pages.dtype, TypeError,
             "key_pages and value_pages must both use float32, bfloat16, float16, float8_e4m3fn or float4_e2m1fn_x2")
    _require(min(key_pages.shape) >= 1 and min(value_pages.shape) >= 1, ValueError,
             "a cache has at least one page, head, token and number")
    _require(_width(key_pages) <= MAX_WIDTH and _width(value_pages) <= MAX_WIDTH, ValueError,
             f"key and value widths must be at most {MAX_WIDTH}")
    _check_rows("key_pages", key_pages)
    _check_rows("value_pages", value_pages)
    coded = key_pages.dtype in _CODED
    for name, exponents, pages in (("key_exponents", key_exponents, key_pages),
                                   ("value_exponents", value_exponents, value_pages)):
        _require((exponents is not None) == coded, ValueError,
                 "key_exponents and value_exponents belong to float8_e4m3fn and float4_e2m1fn_x2 pages, and to no others")
        if coded:
            few = pages.dtype == E2M1
            _require(exponents.dtype == (E8M0 if few else torch.int8), TypeError,
                     f"{name} must use {'float8_e8m0fnu' if few else 'int8'}")
            _require(exponents.shape == _exponent_shape(pages), ValueError,
                     f"{name} must have shape [pages, heads, page_size" + (", width / 32 rounded up]" if few else "]"))
            if few:
                _check_rows(name, exponents)
            _require(exponents.device == key_pages.device, ValueError, f"{name} must be on the pages' device")
    for name, t in (("page_ptr", page_ptr), ("page_idx", page_idx)):
        _require(t.dtype in _INTEGERS, TypeError, f"{name} must use integers")
        _require(t.ndim == 1, ValueError, f"{name} must be one-dimensional")
    _require(page_ptr.numel() >= 1, ValueError, "page_ptr must contain one entry more than there are sequences")
    _require(value_pages.device == key_pages.device and page_ptr.device == key_pages.device
             and page_idx.device == key_pages.device, ValueError, "the cache must be on one device")


def _check_tokens(key_pages, page_ptr, token_ptr, start) -> None:
    if (token_ptr.dtype is torch.long and start.dtype is torch.long and token_ptr.dim() == 1 and start.dim() == 1
            and token_ptr.numel() == page_ptr.numel() == start.numel() + 1
            and token_ptr.get_device() == start.get_device() == key_pages.get_device()):
        return
    for name, t, more in (("token_ptr", token_ptr, 0), ("start", start, 1)):
        _require(t.dtype in _INTEGERS, TypeError, f"{name} must use integers")
        _require(t.ndim == 1 and t.numel() + more == page_ptr.numel(), ValueError,
                 f"{name} must contain one entry per sequence" + ("" if more else ", and one more"))
        _require(t.device == key_pages.device, ValueError, f"{name} must be on the cache's device")


def _check_new_rows(key, value, key_pages, value_pages) -> None:
    if (key.dim() == 3 and value.dim() == 3 and key.dtype is value.dtype and key.dtype in _ROW_DTYPES
            and (key_pages.dtype is key.dtype or key_pages.dtype in _CODED)
            and key.shape == (value.size(0), key_pages.size(1), _width(key_pages))
            and value.shape == (key.size(0), value_pages.size(1), _width(value_pages))
            and key.get_device() == value.get_device() == key_pages.get_device()):
        return
    for name, t, pages in (("key", key, key_pages), ("value", value, value_pages)):
        _require(t.ndim == 3 and t.size(1) == pages.size(1) and t.size(2) == _width(pages), ValueError,
                 f"{name} must have shape [tokens, heads, width] with the heads and width of {name}_pages")
        _require(t.device == pages.device, ValueError, f"{name} must be on the cache's device")
    _require(key.size(0) == value.size(0), ValueError, "key and value must have the same number of tokens")
    _require(key.dtype == value.dtype and key.dtype in _ROW_DTYPES and key_pages.dtype in (key.dtype, *_CODED),
             TypeError, "key and value must both use the dtype of the pages (float32, bfloat16 or float16 for "
             "float8_e4m3fn and float4_e2m1fn_x2 pages)")


def _no_gradient(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad()")
    if has_tangent(*tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative")


class _CacheStruct(ctypes.Structure):
    """``as_paged_cache`` of ``include/autosage_hip.h``."""

    _fields_ = [
        ("key_pages", ctypes.c_void_p), ("value_pages", ctypes.c_void_p),
        ("key_exponents", ctypes.c_void_p), ("value_exponents", ctypes.c_void_p),
        ("page_ptr", ctypes.c_void_p), ("page_idx", ctypes.c_void_p),
        ("page_idx_len", ctypes.c_int64), ("sequences", ctypes.c_int64), ("pages", ctypes.c_int64),
        ("page_size", ctypes.c_int64), ("heads", ctypes.c_int64), ("key_width", ctypes.c_int64),
        ("value_width", ctypes.c_int64),
        ("key_strides", ctypes.c_int64 * 3), ("value_strides", ctypes.c_int64 * 3),
        ("key_exponent_strides", ctypes.c_int64 * 3), ("value_exponent_strides", ctypes.c_int64 * 3),
        ("dtype", ctypes.c_int32),
    ]


# The same as 64-bit words, which ctypes fills three times as fast.
_CacheWords = ctypes.c_int64 * (ctypes.sizeof(_CacheStruct) // 8)
_NO_STRIDES = (0, 0, 0)


def _cache_struct(key_pages, value_pages, page_ptr, page_idx, key_exponents, value_exponents):
    pages, heads, page_size, width = key_pages.shape
    widths = (2 * width, 2 * value_pages.size(3)) if key_pages.dtype is E2M1 else (width, value_pages.size(3))
    key_strides, value_strides = key_pages.stride(), value_pages.stride()
    if key_exponents is None:
        key_e = value_e = 0
        key_e_strides = value_e_strides = _NO_STRIDES
    else:
        key_e, value_e = key_exponents.data_ptr(), value_exponents.data_ptr()
        key_e_strides, value_e_strides = key_exponents.stride()[:3], value_exponents.stride()[:3]
    return _CacheWords(
        key_pages.data_ptr(), value_pages.data_ptr(), key_e, value_e, page_ptr.data_ptr(), page_idx.data_ptr(),
        page_idx.numel(), page_ptr.numel() - 1, pages, page_size, heads, *widths,
        *key_strides[:3], *value_strides[:3], *key_e_strides, *value_e_strides, _DTYPES[key_pages.dtype])


_TwoStrides = ctypes.c_int64 * 2


def _long(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.long and t.is_contiguous() else t.to(torch.long).contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.size(-1) == 1 or t.stride(-1) == 1 else t.contiguous()


def _validate_lists(key_pages, page_ptr, page_idx, first, last) -> None:
    """``AUTOSAGE_VALIDATE=1``: every list is inside ``page_idx``, and holds ids of pages where tokens ``first`` to
    ``last - 1`` are (what else a list has room for may be anything)."""
    pages, page_size = key_pages.size(0), key_pages.size(2)
    counts = page_ptr[1:] - page_ptr[:-1]
    bad = (page_ptr[0] < 0) | (counts < 0).any() | (page_ptr[-1] > page_idx.numel())
    _require(not bool(bad), ValueError,
             "invalid page lists: page_ptr must not be negative, not descend and end inside page_idx")
    entry = torch.arange(int(page_ptr[0]), int(page_ptr[-1]), device=page_ptr.device)
    sequence = torch.searchsorted(page_ptr, entry, right=True) - 1
    at = (entry - page_ptr[sequence]) * page_size
    used = page_idx[entry[(at + page_size > first[sequence]) & (at < last[sequence])]]
    _require(not bool(((used < 0) | (used >= pages)).any()), ValueError,
             "invalid page lists: page ids must lie in [0, pages)")
    _require(not bool((last > counts * page_size).any()), ValueError,
             "invalid page lists: a sequence has more tokens than its pages hold")


def _page_lists(page_ptr, page_idx):
    """(begin, number of entries) of every sequence's list, inside ``page_idx`` whatever ``page_ptr`` holds: as the
    kernels do."""
    begin = page_ptr[:-1].clamp(0, page_idx.numel())
    return begin, torch.maximum(page_ptr[1:].clamp_max(page_idx.numel()), begin) - begin


def _places(page_ptr, page_idx, token_ptr, start, tokens: int, pages: int, page_size: int):
    """(which of the call's tokens have a place, their pages, their places there)."""
    at = torch.arange(tokens, device=start.device)
    sequence = torch.searchsorted(token_ptr, at, right=True) - 1
    known = (sequence >= 0) & (sequence < start.numel())
    at, sequence = at[known], sequence[known]
    # bounds beyond which a sum would pass 64 bits; no sequence has pages there
    mine = (at < token_ptr[sequence + 1]) & (token_ptr[sequence] >= -(2**62)) & (start[sequence] < 2**62)
    at, sequence = at[mine], sequence[mine]
    position = start[sequence] + (at - token_ptr[sequence])
    entry = position // page_size
    begin, room = _page_lists(page_ptr, page_idx)
    has_page = (position >= 0) & (entry < room[sequence])
    at, position, entry, sequence = at[has_page], position[has_page], entry[has_page], sequence[has_page]
    page = page_idx[begin[sequence] + entry]
    inside = (page >= 0) & (page < pages)
    return at[inside], page[inside], position[inside] % page_size


def _validate_call(key_pages, page_ptr, page_idx, token_ptr, start, tokens: int, writes: bool) -> None:
    if _env.get("AUTOSAGE_VALIDATE") != "1":
        return
    counts = token_ptr[1:] - token_ptr[:-1]
    bad = (token_ptr[0] < 0) | (counts < 0).any() | (token_ptr[-1] > tokens) | (start < 0).any()
    _require(not bool(bad), ValueError,
             "invalid tokens: token_ptr must not be negative, not descend and end inside the tokens, start not be "
             "negative")
    last = torch.where(counts > 0, start.clamp_max(2**62) + counts, 0)  # the sum stays below 2^63
    _validate_lists(key_pages, page_ptr, page_idx, start, last)
    if writes:
        pages, page_size = key_pages.size(0), key_pages.size(2)
        _, page, place = _places(page_ptr, page_idx, token_ptr, start, tokens, pages, page_size)
        _require(torch.unique(page * page_size + place).numel() == page.numel(), ValueError,
                 "invalid page lists: two tokens of one call have the same place")


def _need_native() -> ctypes.CDLL:
    if not load_native():
        raise RuntimeError(f"AutoSAGE CUDA extension is unavailable: {native_load_error()}")
    return _native.library()


# ---------------------------------------------------------------------------
# 8-bit and 4-bit numbers


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, exponents): 2^e is the smallest power of two, not below 2^-126,
    that brings a row's largest finite magnitude to 448; what is not finite is
    held as NaN."""
    x = x.float()
    finite = x.isfinite()
    mantissa, exponent = torch.frexp(torch.where(finite, x.abs(), 0.0).amax(-1, keepdim=True))
    exponent = torch.where(mantissa == 0, -126, exponent - 9 + (mantissa > 0.875).to(torch.int32)).clamp_min(-126)
    # two steps: 2^-e itself may be beyond float32
    half = exponent // 2
    codes = torch.where(finite, torch.ldexp(torch.ldexp(x, -half), half - exponent), float("nan")).to(E4M3)
    return codes, exponent.squeeze(-1).to(torch.int8)


def _values(codes: torch.Tensor, exponents: torch.Tensor) -> torch.Tensor:
    half = exponents.to(torch.int32)[..., None] // 2
    return torch.ldexp(torch.ldexp(codes.float(), half), exponents.to(torch.int32)[..., None] - half)


def _quantise_pairs(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, two in a byte, exponents + 127) of 4-bit numbers, as bytes: 2^e is the smallest power of two, not below
    2^-127, that brings the largest magnitude of 32 numbers to 6; a group with a number that is not finite is held as
    NaN (255)."""
    width = x.size(-1)
    x = torch.nn.functional.pad(x.float(), (0, -width % GROUP)).unflatten(-1, (-1, GROUP))
    finite = x.isfinite().all(-1, keepdim=True)
    x = torch.where(finite, x, 0.0)
    mantissa, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))
    exponent = torch.where(mantissa == 0, -127, exponent - 3 + (mantissa > 0.75).to(torch.int32)).clamp_min(-127)
    size = torch.ldexp(x.abs(), -exponent)
    # half to the even code
    code = ((size > 0.25).int() + (size >= 0.75) + (size > 1.25) + (size >= 1.75) + (size > 2.5) + (size >= 3.5)
            + (size > 5.0) + 8 * x.signbit()).to(torch.uint8).flatten(-2)[..., :width]
    return code[..., ::2] | code[..., 1::2] << 4, torch.where(finite, exponent + 127, 255).squeeze(-1).to(torch.uint8)


def _pair_values(codes: torch.Tensor, exponents: torch.Tensor) -> torch.Tensor:
    sizes = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    numbers = torch.cat((sizes, -sizes))[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    exponent = exponents.repeat_interleave(GROUP, -1)[..., :numbers.size(-1)].int()
    return torch.where(exponent == 255, float("nan"), torch.ldexp(numbers, exponent - 127))


def _put_rows(rows: torch.Tensor, pages: torch.Tensor, exponents: Optional[torch.Tensor], page, place) -> None:
    if exponents is None:
        pages[page, :, place] = rows
        return
    codes, scale = (_quantise_pairs if pages.dtype == E2M1 else _quantise)(rows)
    pages.view(torch.uint8)[page, :, place] = codes.view(torch.uint8)
    exponents.view(scale.dtype)[page, :, place] = scale


def _held_rows(pages: torch.Tensor, exponents: Optional[torch.Tensor], *index) -> torch.Tensor:
    """What the places of an index hold, in float32 where they are coded."""
    if exponents is None:
        return pages[index]
    codes = pages.view(torch.uint8)[index]
    if pages.dtype == E2M1:
        return _pair_values(codes, exponents.view(torch.uint8)[index])
    return _values(codes.view(E4M3), exponents[index])


# ---------------------------------------------------------------------------
# Write


def paged_cache_write_impl(key, value, key_pages, value_pages, page_ptr, page_idx, token_ptr, start,
                           key_exponents=None, value_exponents=None) -> None:
    _check_cache(key_pages, value_pages, page_ptr, page_idx, key_exponents, value_exponents)
    _check_tokens(key_pages, page_ptr, token_ptr, start)
    _check_new_rows(key, value, key_pages, value_pages)
    for t in (key_pages, value_pages, key_exponents, value_exponents):
        if t is not None and 0 in t.stride():
            _require(all(s > 0 for s, n in zip(t.stride(), t.shape) if n > 1), ValueError,
                     "pages and exponents that are written must not hold a place twice")
    _no_gradient("paged_cache_write", key, value, key_pages, value_pages)
    page_ptr, page_idx, token_ptr, start = _long(page_ptr), _long(page_idx), _long(token_ptr), _long(start)
    tokens = key.size(0)
    _validate_call(key_pages, page_ptr, page_idx, token_ptr, start, tokens, True)
    if tokens == 0 or page_ptr.numel() == 1:
        return
    if not key.is_cuda:
        at, page, place = _places(page_ptr, page_idx, token_ptr, start, tokens, key_pages.size(0),
                                  key_pages.size(2))
        for rows, pages, exponents in ((key, key_pages, key_exponents), (value, value_pages, value_exponents)):
            _put_rows(rows[at], pages, exponents, page, place)
        return
    lib = _need_native()
    key, value = _rows(key), _rows(value)
    # the kernel writes behind torch's back: a graph that saved the pages has to see that they changed
    torch.autograd.graph.increment_version([t for t in (key_pages, value_pages, key_exponents, value_exponents)
                                            if t is not None])
    cache = _cache_struct(key_pages, value_pages, page_ptr, page_idx, key_exponents, value_exponents)
    with _native._on(key.device):
        status = lib.as_paged_cache_write(
            ctypes.byref(cache), key.data_ptr(), _TwoStrides(key.stride(0), key.stride(1)), value.data_ptr(),
            _TwoStrides(value.stride(0), value.stride(1)), token_ptr.data_ptr(), start.data_ptr(), tokens,
            _DTYPES[key.dtype], _native._stream(key.device))
    _native._raise(status, "autosage::paged_cache_write")


def paged_cache_write(key, value, key_pages, value_pages, page_ptr, page_idx, token_ptr, start, *,
                      key_exponents=None, value_exponents=None) -> None:
    """Writes the rows of new tokens into the pages of their sequences, in place.

    ``key`` ``[tokens, heads, key width]`` and ``value`` ``[tokens, heads, value
    width]`` hold the tokens of sequence ``b`` at ``token_ptr[b]:token_ptr[b +
    1]``; the first of them is token ``start[b]`` of its sequence.  Rows in front of
    ``token_ptr[0]`` and behind ``token_ptr[-1]`` are padding.  Pages of ``torch.float8_e4m3fn`` come with
    ``key_exponents`` and ``value_exponents`` (int8, ``[pages, heads,
    page_size]``): a row is held as codes and the exponent of the smallest power
    of two that brings its largest magnitude to 448, so that scaling is exact
    and every number is off by at most 1/16 of itself or half the smallest
    code; infinities and NaN become NaN.  That 1/16 may pass the largest number
    of a type: what is 63,488 or more may be held as 65,536, which a read in
    float16 gives as infinity (and 3.3e38 as 2^128, infinite in every type).

    Pages of ``torch.float4_e2m1fn_x2`` (``[pages, heads, page_size, width / 2]``, two numbers in a byte,
    the first in its low bits; widths are even) come with exponents of ``torch.float8_e8m0fnu``,
    ``[pages, heads, page_size, ceil(width / 32)]``, contiguous in the last dimension: one
    power of two for each 32 neighbouring numbers of a row, the smallest that brings the largest of
    them to 6; the numbers divided by it are rounded to 0, 1/2, 1, 3/2, 2, 3, 4 or 6, half to
    the even code. A number is off by at most a fifth of itself, or a quarter of its group's power
    of two where that is more. That may pass the largest number of a type: what is 57,344 or more
    may be held as 65,536, which a read in float16 gives as infinity (and 2.98e38, 3.5 * 2^126, as 2^128, infinite
    in every type). A group with a number that is not finite is NaN as a whole.

    A token whose place has no page is not written.  Two tokens of one call must
    not share a place (``AUTOSAGE_VALIDATE=1`` checks it, with the lists)."""
    paged_cache_write_impl(key, value, key_pages, value_pages, page_ptr, page_idx, token_ptr, start, key_exponents,
                           value_exponents)


# ---------------------------------------------------------------------------
# Read


def paged_cache_read_impl(key_pages, value_pages, page_ptr, page_idx, token_ptr, start, tokens, dtype=None,
                          key_exponents=None, value_exponents=None):
    _check_cache(key_pages, value_pages, page_ptr, page_idx, key_exponents, value_exponents)
    _check_tokens(key_pages, page_ptr, token_ptr, start)
    tokens = int(tokens)
    _require(tokens >= 0, ValueError, "tokens must not be negative")
    coded = key_pages.dtype in _CODED
    if dtype is None:
        dtype = torch.bfloat16 if coded else key_pages.dtype
    _require(dtype in _ROW_DTYPES and (coded or dtype == key_pages.dtype), TypeError,
             "dtype must be the dtype of the pages (float32, bfloat16 or float16 for float8_e4m3fn and "
             "float4_e2m1fn_x2 pages)")
    _no_gradient("paged_cache_read", key_pages, value_pages)
    page_ptr, page_idx, token_ptr, start = _long(page_ptr), _long(page_idx), _long(token_ptr), _long(start)
    _validate_call(key_pages, page_ptr, page_idx, token_ptr, start, tokens, False)
    heads, device = key_pages.size(1), key_pages.device
    shapes = [(tokens, heads, _width(pages)) for pages in (key_pages, value_pages)]
    if tokens == 0 or page_ptr.numel() == 1 or not key_pages.is_cuda:
        out = [torch.zeros(shape, dtype=dtype, device=device) for shape in shapes]
        if tokens > 0 and page_ptr.numel() > 1:
            at, page, place = _places(page_ptr, page_idx, token_ptr, start, tokens, key_pages.size(0),
                                      key_pages.size(2))
            for rows, pages, exponents in zip(out, (key_pages, value_pages), (key_exponents, value_exponents)):
                rows[at] = _held_rows(pages, exponents, page, slice(None), place).to(dtype)
        return out[0], out[1]
    lib = _need_native()
    key, value = (torch.empty(shape, dtype=dtype, device=device) for shape in shapes)
    cache = _cache_struct(key_pages, value_pages, page_ptr, page_idx, key_exponents, value_exponents)
    with _native._on(device):
        status = lib.as_paged_cache_read(ctypes.byref(cache), key.data_ptr(), value.data_ptr(), token_ptr.data_ptr(),
                                         start.data_ptr(), tokens, _DTYPES[dtype], _native._stream(device))
    _native._raise(status, "autosage::paged_cache_read")
    return key, value


def paged_cache_read(key_pages, value_pages, page_ptr, page_idx, token_ptr, start, tokens: int, *,
                     dtype: Optional[torch.dtype] = None, key_exponents=None, value_exponents=None):
    """(key, value) of a run of tokens of every sequence, ``[tokens, heads,
    width]``: those of sequence ``b`` are its tokens from ``start[b]`` on and
    stand at ``token_ptr[b]:token_ptr[b + 1]``.  ``tokens`` is the number of
    rows of the result; rows of no sequence, and tokens without a page, are
    zeros.  ``float8_e4m3fn`` and ``float4_e2m1fn_x2`` pages give the numbers they
    stand for in ``dtype`` (default bfloat16, which holds them exactly unless they
    are below its smallest number; infinite where they are beyond its largest),
    other pages their own dtype."""
    return paged_cache_read_impl(key_pages, value_pages, page_ptr, page_idx, token_ptr, start, tokens, dtype,
                                 key_exponents, value_exponents)


# ---------------------------------------------------------------------------
# Attention


def _check_attention(query, key_pages, lengths, page_ptr, window, bias_table, max_distance, max_length,
                     bidirectional) -> None:
    heads = key_pages.size(1)
    if (bias_table is None and max_distance is None and window is None and query.dim() == 3
            and query.size(0) == page_ptr.numel() - 1 == lengths.numel() and query.size(2) == _width(key_pages)
            and query.size(1) >= 1 and query.size(1) % heads == 0 and query.dtype in _ROW_DTYPES
            and (key_pages.dtype is query.dtype or key_pages.dtype in _CODED)
            and lengths.dtype is torch.long and lengths.dim() == 1
            and query.get_device() == lengths.get_device() == key_pages.get_device()
            and (max_length is None or max_length >= 0)):
        return
    _require(query.ndim == 3 and query.size(0) == page_ptr.numel() - 1 and query.size(2) == _width(key_pages)
             and query.size(1) >= 1 and query.size(1) % heads == 0, ValueError,
             "query must have shape [sequences, query heads, key width] with a multiple of the cache's heads")
    _require(query.dtype in _ROW_DTYPES and key_pages.dtype in (query.dtype, *_CODED), TypeError,
             "query must use the dtype of the pages (float32, bfloat16 or float16 for float8_e4m3fn and "
             "float4_e2m1fn_x2 pages)")
    _require(query.device == key_pages.device, ValueError, "query must be on the cache's device")
    _require(lengths.dtype in _INTEGERS, TypeError, "lengths must use integers")
    _require(lengths.ndim == 1 and lengths.numel() == query.size(0), ValueError,
             "lengths must contain one entry per sequence")
    _require(lengths.device == query.device, ValueError, "lengths must be on the cache's device")
    _require(window is None or int(window) >= 1, ValueError, "window must be positive")
    _require(max_length is None or int(max_length) >= 0, ValueError, "max_length must not be negative")
    if bias_table is None:
        _require(max_distance is None, ValueError, "max_distance belongs to a bias_table")
        return
    _require(max_distance is not None, ValueError, "a bias_table needs max_distance")
    _require(bias_table.ndim == 2 and bias_table.size(1) == query.size(1), ValueError,
             "bias_table must have shape [buckets, query heads]")
    _require(bias_table.dtype == query.dtype, TypeError, "bias_table must use the dtype of query")
    _require(bias_table.device == query.device, ValueError, "bias_table must be on the cache's device")
    bucket_borders(bias_table.size(0), int(max_distance), bool(bidirectional))


def _cpu_attention(query, key_pages, value_pages, page_ptr, page_idx, lengths, scale, window, bias_table, max_distance,
                   bidirectional, max_length, key_exponents, value_exponents):
    """One sequence after another, in float32."""
    sequences, heads_q, _ = query.shape
    heads, page_size = key_pages.size(1), key_pages.size(2)
    group = heads_q // heads
    out = torch.zeros(sequences, heads_q, _width(value_pages), dtype=torch.float32)
    lse = torch.full((sequences, heads_q), float("-inf"))
    begins, rooms = _page_lists(page_ptr, page_idx)
    for b in range(sequences):
        length = max(0, int(lengths[b]))
        first = max(0, length - window) if window else 0
        mine = page_idx[int(begins[b]):int(begins[b] + rooms[b])]
        short = length > mine.numel() * page_size or (max_length is not None and length > max_length)
        skipped = first // page_size
        mine = mine[skipped: -(-length // page_size)]
        if short or bool(((mine < 0) | (mine >= key_pages.size(0))).any()):
            out[b], lse[b] = float("nan"), float("nan")
            continue
        if length == 0:
            continue
        rows = []
        for pages, exponents in ((key_pages, key_exponents), (value_pages, value_exponents)):
            held = _held_rows(pages, exponents, mine).float()
            held = held.transpose(0, 1).reshape(heads, -1, held.size(-1))
            held = held[:, first - skipped * page_size:length - skipped * page_size]
            rows.append(held.repeat_interleave(group, 0))
        scores = (rows[0] @ query[b].float()[:, :, None]).squeeze(-1) * scale
        if bias_table is not None:
            away = torch.arange(first - length + 1, 1)
            bucket = position_buckets(away, bias_table.size(0), max_distance, bidirectional)
            scores = scores + bias_table.float()[bucket].t()
        top = scores.amax(-1, keepdim=True)
        weights = (scores - torch.where(top == float("-inf"), 0.0, top)).exp()
        total = weights.sum(-1, keepdim=True)
        result = (weights[:, None] @ rows[1]).squeeze(1) / total
        out[b] = torch.where(total == 0, 0.0, result)
        lse[b] = (top + total.log()).squeeze(-1)
    return out.to(query.dtype), lse


def _attention(query, key_pages, value_pages, page_ptr, page_idx, lengths, scale=1.0, window=None,
                         bias_table=None, max_distance=None, bidirectional=True, max_length=None, key_exponents=None,
                         value_exponents=None, return_lse=False):
    """(out, lse); no lse unless ``return_lse``."""
    _check_cache(key_pages, value_pages, page_ptr, page_idx, key_exponents, value_exponents)
    _check_attention(query, key_pages, lengths, page_ptr, window, bias_table, max_distance, max_length, bidirectional)
    _no_gradient("paged_attention", query, key_pages, value_pages, bias_table)
    page_ptr, page_idx, lengths = _long(page_ptr), _long(page_idx), _long(lengths)
    if _env.get("AUTOSAGE_VALIDATE") == "1":
        first = torch.zeros_like(lengths) if window is None else (lengths - int(window)).clamp_min(0)
        _validate_lists(key_pages, page_ptr, page_idx, first, lengths)
        _require(not bool((lengths < 0).any()), ValueError, "invalid lengths: they must not be negative")
        _require(max_length is None or not bool((lengths > int(max_length)).any()), ValueError,
                 "invalid lengths: one is beyond max_length")
    if not query.is_cuda:
        out, lse = _cpu_attention(query, key_pages, value_pages, page_ptr, page_idx, lengths, float(scale), window,
                                  bias_table, max_distance, bool(bidirectional), max_length, key_exponents,
                                  value_exponents)
        return out, lse if return_lse else None
    lib = _need_native()
    sequences, heads_q, _ = query.shape
    out = torch.empty(sequences, heads_q, _width(value_pages), dtype=query.dtype, device=query.device)
    lse = torch.empty(sequences, heads_q, dtype=torch.float32, device=query.device) if return_lse else None
    if sequences == 0:
        return out, lse
    query = _rows(query)
    buckets, borders = 0, None
    if bias_table is not None:
        bias_table = bias_table.contiguous()
        buckets = bias_table.size(0)
        borders = border_array(buckets, int(max_distance), bool(bidirectional))
    cache = _cache_struct(key_pages, value_pages, page_ptr, page_idx, key_exponents, value_exponents)
    bound = -1 if max_length is None else int(max_length)
    group = heads_q // key_pages.size(1)
    seen = 0 if window is None else int(window)
    ws_bytes = lib.as_paged_attention_workspace_bytes(ctypes.byref(cache), group, seen, bound)
    ws = _native._workspace(ws_bytes, query.device) if ws_bytes else None
    with _native._on(query.device):
        status = lib.as_paged_attention(
            ctypes.byref(cache), query.data_ptr(), _TwoStrides(query.stride(0), query.stride(1)),
            out.data_ptr(), _native._ptr(lse), lengths.data_ptr(), group, float(scale),
            seen, None if bias_table is None else bias_table.data_ptr(), buckets,
            borders, int(bool(bidirectional)), bound, _DTYPES[query.dtype], _native._ptr(ws), ws_bytes,
            _native._stream(query.device))
    _native._raise(status, "autosage::paged_attention")
    return out, lse


def paged_attention_impl(*args, **kwargs):
    """(out, lse) of the registered operator; lse is empty unless ``return_lse``."""
    out, lse = _attention(*args, **kwargs)
    return out, out.new_empty(0, dtype=torch.float32) if lse is None else lse


def paged_attention(query, key_pages, value_pages, page_ptr, page_idx, lengths, *, scale: float = 1.0,
                    window: Optional[int] = None, bias_table=None, max_distance: Optional[int] = None,
                    bidirectional: bool = True, max_length: Optional[int] = None, key_exponents=None,
                    value_exponents=None, return_lse: bool = False):
    """softmax(scale * query . keys) . values of every sequence's last token,
    whose own key and value the cache already holds.

    ``query`` is ``[sequences, query heads, key width]``; each of the cache's
    heads serves ``query heads / heads`` consecutive query heads.  ``lengths``
    counts the tokens of every sequence, the new one included; ``window`` limits
    the attention to the last ones.  ``bias_table`` ``[buckets, query heads]``
    adds the learned bias of the distance to the new token, with the buckets of
    ``csr_position_bias`` for the same ``max_distance`` and ``bidirectional``.
    ``max_length``, an upper bound of ``lengths`` known to the host, lets short
    sequences be answered in one launch.

    Scores, softmax and sums are float32 and the result is rounded once to the
    dtype of ``query``.  (Over 8-bit pages a query is multiplied with the codes,
    so that finite numbers beyond 2^111 may give infinite scores.  On the GPU
    numbers of 4-bit pages below 2^-126 count as zeros, as weights below it do, and a value
    that is held as 2^128 makes NaN of its column where the CPU makes an infinity.)  A sequence without
    tokens, or with scores of -inf alone, gives zeros; a length beyond ``max_length`` or the sequence's pages, or a
    page id outside the cache, gives NaN.  ``return_lse`` adds the logarithm of
    the sum of the exponentials, float32 ``[sequences, query heads]``, with which
    results over parts of a sequence can be joined."""
    out, lse = _attention(query, key_pages, value_pages, page_ptr, page_idx, lengths, scale, window, bias_table,
                          max_distance, bidirectional, max_length, key_exponents, value_exponents, return_lse)
    return (out, lse) if return_lse else out


SCHEMAS = {
    "paged_cache_write": (
        "paged_cache_write(Tensor key, Tensor value, Tensor(a!) key_pages, Tensor(b!) value_pages, Tensor page_ptr, "
        "Tensor page_idx, Tensor token_ptr, Tensor start, Tensor(c!)? key_exponents=None, "
        "Tensor(d!)? value_exponents=None) -> ()",
        paged_cache_write_impl,
    ),
    "paged_cache_read": (
        "paged_cache_read(Tensor key_pages, Tensor value_pages, Tensor page_ptr, Tensor page_idx, Tensor token_ptr, "
        "Tensor start, int tokens, ScalarType? dtype=None, Tensor? key_exponents=None, Tensor? value_exponents=None) "
        "-> (Tensor, Tensor)",
        paged_cache_read_impl,
    ),
    "paged_attention": (
        "paged_attention(Tensor query, Tensor key_pages, Tensor value_pages, Tensor page_ptr, Tensor page_idx, "
        "Tensor lengths, float scale=1.0, int? window=None, Tensor? bias_table=None, int? max_distance=None, "
        "bool bidirectional=True, int? max_length=None, Tensor? key_exponents=None, Tensor? value_exponents=None, "
        "bool return_lse=False) -> (Tensor, Tensor)",
        paged_attention_impl,
    ),
}

__all__ = ["paged_attention", "paged_cache_read", "paged_cache_write"]
