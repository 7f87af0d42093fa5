"""The paged cache of 4-bit numbers on the CPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import autosage_amd
from autosage_amd import _native
from autosage_amd.paged import _cache_struct, _CacheStruct
from tests.paged4_common import E2M1, E8M0, Cache4, quantised_pairs
from tests.paged_common import assert_attention, plain_attention

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def empty(pages, heads, page, width, fill=255):
    codes = torch.full((pages, heads, page, width // 2), fill, dtype=torch.uint8).view(E2M1)
    return codes, torch.full((pages, heads, page, -(-width // 32)), fill, dtype=torch.uint8).view(E8M0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window, biased", [(None, False), (5, False), (None, True), (7, True)])
def test_attention(dtype, window, biased):
    lengths = [0, 1, 9, 40]
    cache = Cache4(lengths, 2, 40, 34, 4, dtype, seed=1)
    gen = torch.Generator().manual_seed(2)
    query = torch.randn(4, 6, 40, generator=gen).to(dtype)
    plain, own = {}, {}
    if biased:
        table = torch.randn(8, 6, generator=gen).to(dtype)
        plain = {"table": table, "max_distance": 20, "bidirectional": False}
        own = {"bias_table": table, "max_distance": 20, "bidirectional": False}
    args, exponents = cache.args("cpu")
    out, lse = autosage_amd.paged_attention(query, *args, torch.tensor(lengths), scale=0.2, window=window,
                                            return_lse=True, **own, **exponents)
    assert_attention(out, lse, plain_attention(cache, query, 0.2, window=window, **plain), dtype=dtype, quantised=True,
                     lse_bound=2e-4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width, value_width", [(2, 30), (32, 64), (72, 34), (256, 254)])
def test_write_then_read(dtype, width, value_width):
    gen = torch.Generator().manual_seed(width)
    (k, ke), (v, ve) = empty(9, 3, 4, width), empty(9, 3, 4, value_width)
    page_ptr, page_idx = torch.tensor([0, 3, 5]), torch.tensor([8, 1, 4, 0, 7])
    key, value = (torch.randn(9, 3, w, generator=gen).to(dtype) for w in (width, value_width))
    token_ptr, start = torch.tensor([0, 6, 8]), torch.tensor([3, 5])
    span = (page_ptr, page_idx, token_ptr, start)
    autosage_amd.paged_cache_write(key, value, k, v, *span, key_exponents=ke, value_exponents=ve)
    back = autosage_amd.paged_cache_read(k, v, *span, 9, dtype=torch.float32, key_exponents=ke, value_exponents=ve)
    for rows, got, codes, exponents in ((key, back[0], k, ke), (value, back[1], v, ve)):
        held, packed, e = quantised_pairs(rows)
        assert torch.equal(got[:8].double(), held[:8]) and not got[8:].any()
        for t, (b, position) in enumerate([(0, 3 + i) for i in range(6)] + [(1, 5), (1, 6)]):
            page = page_idx[page_ptr[b] + position // 4]
            assert torch.equal(codes.view(torch.uint8)[page, :, position % 4], packed[t])
            assert torch.equal(exponents.view(torch.uint8)[page, :, position % 4], e[t])
        # nothing else was written
        assert int((codes.view(torch.uint8) == 255).all(-1).sum()) >= 3 * (36 - 8)


def test_numbers_at_the_edges():
    """Ties, signs, groups of zeros, the smallest and largest numbers, groups with a number that is not finite."""
    rows = torch.zeros(8, 1, 64)
    rows[0, 0, :16] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -6.0, -0.25, -0.75, -1.25, -1.75, -2.5,
                                    -3.5, -5.0])
    rows[1, 0, 0], rows[1, 0, 33] = 6.0001, 3.0
    rows[2, 0, 0], rows[2, 0, 40] = 3.4e38, 2.0**-149
    rows[3, 0, 0], rows[3, 0, 63] = float("inf"), 1.0
    rows[4, 0, 5], rows[4, 0, 32] = float("nan"), -float("inf")
    rows[5, 0, :3] = torch.tensor([2.0**-126, 1.5 * 2.0**-126, 3.0 * 2.0**-126])
    rows[6, 0, 0], rows[6, 0, 1] = 6.0, -0.0
    (k, ke), (v, ve) = empty(2, 1, 4, 64), empty(2, 1, 4, 64)
    span = (torch.tensor([0, 2]), torch.tensor([1, 0]), torch.tensor([0, 8]), torch.tensor([0]))
    autosage_amd.paged_cache_write(rows, rows, k, v, *span, key_exponents=ke, value_exponents=ve)
    key, value = autosage_amd.paged_cache_read(k, v, *span, 8, dtype=torch.float32, key_exponents=ke, value_exponents=ve)
    assert torch.equal(key.nan_to_num(99.0), value.nan_to_num(99.0))
    finite = rows.unflatten(-1, (2, 32)).isfinite().all(-1).repeat_interleave(32, -1)
    assert torch.equal(key.isnan(), ~finite)
    held = quantised_pairs(rows.nan_to_num(0.0, 0.0, 0.0))[0]
    # 3.4e38 / 2^126 is 3.997 (6 * 2^125 = 2.6e38 is less, so 2^126 it is) and held as 4 * 2^126 = 2^128, which float32
    # gives as infinity
    assert held[2, 0, 0] == 2.0**128
    assert torch.equal(key[finite], held[finite].float())
    ties = [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]
    assert key[0, 0, :16].tolist() == ties + [-t for t in ties]
    assert key[6, 0, 1].signbit()
    assert (ke.view(torch.uint8)[0, 0, 3] == 0).all()  # a row of zeros


def test_lengths_pages_and_lists_that_do_not_fit():
    cache = Cache4([4, 9, 9], 1, 8, 6, 4, torch.float32, seed=3)
    (k, v, ptr, idx), e = cache.args("cpu")
    query = torch.randn(3, 2, 8)
    idx[4] = 10**6
    out, lse = autosage_amd.paged_attention(query, k, v, ptr, idx, torch.tensor([5, 9, 9]), return_lse=True, **e)
    assert out[0].isnan().all() and lse[0].isnan().all()
    bad = 1 if int(ptr[1]) <= 4 < int(ptr[2]) else 2
    assert out[bad].isnan().all() and out[3 - bad].isfinite().all()
    # places without a token are NaN: a length into them shows
    out = autosage_amd.paged_attention(query[:1], k, v, ptr[:2], idx, torch.tensor([0]), **e)
    assert not out.any()


def test_refusals():
    cache = Cache4([4, 9], 2, 8, 6, 4, torch.float32, seed=7)
    (k, v, ptr, idx), e = cache.args("cpu")
    query, lengths = torch.randn(2, 4, 8), torch.tensor([4, 9])
    attention, write, read = autosage_amd.paged_attention, autosage_amd.paged_cache_write, autosage_amd.paged_cache_read
    key, value = torch.randn(2, 2, 8), torch.randn(2, 2, 6)
    span = (torch.tensor([0, 1, 2]), torch.tensor([3, 8]))
    ke, ve = e["key_exponents"], e["value_exponents"]
    wide = torch.zeros(4, 2, 4, 129, dtype=torch.uint8).view(E2M1)
    for error, call in [
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths)),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths, key_exponents=ke)),
        (TypeError, lambda: attention(query, k, v, ptr, idx, lengths, key_exponents=ke.view(torch.int8),
                                      value_exponents=ve.view(torch.int8))),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths, key_exponents=ke[..., 0], value_exponents=ve)),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths, key_exponents=ke[:1], value_exponents=ve)),
        (TypeError, lambda: attention(query, k, v.view(torch.uint8), ptr, idx, lengths, **e)),
        (TypeError, lambda: attention(query, k.view(torch.uint8), v.view(torch.uint8), ptr, idx, lengths, **e)),
        (ValueError, lambda: attention(query[..., :4], k, v, ptr, idx, lengths, **e)),
        (TypeError, lambda: attention(query.double(), k, v, ptr, idx, lengths, **e)),
        (ValueError, lambda: attention(torch.randn(2, 4, 258), wide, wide, ptr, idx, lengths, **e)),
        (ValueError, lambda: attention(query, k[..., ::2], v, ptr, idx, lengths, **e)),
        (RuntimeError, lambda: attention(query.clone().requires_grad_(), k, v, ptr, idx, lengths, **e)),
        (ValueError, lambda: write(key, value, k, v, ptr, idx, *span)),
        (ValueError, lambda: write(key[..., :4], value, k, v, ptr, idx, *span, **e)),
        (TypeError, lambda: write(key.half(), value, k, v, ptr, idx, *span, **e)),
        (TypeError, lambda: write(key.double(), value.double(), k, v, ptr, idx, *span, **e)),
        (ValueError, lambda: write(key, value, k[:1].expand(4, 2, 4, 4), v[:4], ptr, idx, *span, key_exponents=ke[:4],
                                   value_exponents=ve[:4])),
        (TypeError, lambda: read(k, v, ptr, idx, *span, 2, dtype=torch.float64, **e)),
        (TypeError, lambda: read(k, v, ptr, idx, *span, 2, dtype=E2M1, **e)),
        (ValueError, lambda: write(k, v, k, v, ptr, idx, *span, **e)),
    ]:
        with pytest.raises(error):
            call()
    # exponents of a token that do not follow one another
    long, far = Cache4([4], 1, 64, 64, 4, torch.float32).args("cpu")
    far = {n: t.view(torch.uint8).repeat_interleave(2, -1)[..., ::2].view(E8M0) for n, t in far.items()}
    with pytest.raises(ValueError, match="contiguous"):
        attention(torch.randn(1, 1, 64), *long, torch.tensor([4]), **far)


def test_native_argument_checks_come_before_any_launch():
    path = _native.package_library_path()
    if not path.exists():
        pytest.skip("HIP library not built")
    lib = _native.open_library(path)
    cache = Cache4([4, 9], 2, 8, 6, 4, torch.float32, seed=9)
    (k, v, ptr, idx), e = cache.args("cpu")

    def struct(**changes):
        c = _CacheStruct.from_buffer(_cache_struct(k, v, ptr, idx, *e.values()))
        assert (c.key_width, c.value_width, c.dtype) == (8, 6, 5)
        for name, what in changes.items():
            setattr(c, name, what)
        return ctypes.byref(c)

    two, fake = (ctypes.c_int64 * 2)(8, 4), 256

    def attention(c, dtype=0, ws=fake, ws_bytes=1 << 30):
        return lib.as_paged_attention(c, fake, two, fake, None, fake, 2, 1.0, 0, None, 0, None, 0, -1, dtype, ws,
                                      ws_bytes, None)

    for status, call, message in [
        (3, lambda: attention(struct(key_width=7)), b"an e2m1 cache holds rows of an even width"),
        (3, lambda: attention(struct(value_width=5)), b"an e2m1 cache holds rows of an even width"),
        (1, lambda: attention(struct(key_exponents=None)), b"an e4m3 cache has exponents"),
        (1, lambda: attention(struct(), dtype=5), b"dtype must be"),
        (0, lambda: attention(struct(sequences=0)), b""),
        (1, lambda: lib.as_paged_cache_write(struct(), fake, two, fake, two, fake, fake, 2, 5, None), b"dtype must be"),
        (0, lambda: lib.as_paged_cache_read(struct(), fake, fake, fake, fake, 0, 0, None), b""),
    ]:
        assert call() == status, message
        assert lib.as_last_error().startswith(message), lib.as_last_error()


@pytest.mark.parametrize("bad", [-1, 10**6, 2**40, -(2**40)])
def test_tokens_whose_page_is_outside_the_cache(bad):
    (k, ke), (v, ve) = empty(4, 1, 4, 8, 17), empty(4, 1, 4, 8, 17)
    before = k.view(torch.uint8).clone()
    span = (torch.tensor([0, 1, 2]), torch.tensor([bad, 2]), torch.tensor([0, 3, 5]), torch.tensor([0, 1]))
    rows = torch.randn(5, 1, 8)
    autosage_amd.paged_cache_write(rows, rows, k, v, *span, key_exponents=ke, value_exponents=ve)
    key, _ = autosage_amd.paged_cache_read(k, v, *span, 5, dtype=torch.float32, key_exponents=ke, value_exponents=ve)
    assert not key[:3].any() and torch.equal(key[3:].double(), quantised_pairs(rows)[0][3:])
    assert int((k.view(torch.uint8) != before).any(-1).sum()) <= 2


def test_numbers_in_every_type():
    """What a type cannot hold is rounded once, or infinite."""
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 16, 16).view(E2M1)
    e = torch.full((1, 1, 16, 1), 127 + 14, dtype=torch.uint8).view(E8M0)
    span = (torch.tensor([0, 1]), torch.tensor([0]), torch.tensor([0, 16]), torch.tensor([0]))
    for dtype in DTYPES:
        key, value = autosage_amd.paged_cache_read(codes, codes, *span, 16, dtype=dtype, key_exponents=e,
                                                   value_exponents=e)
        assert key.dtype == dtype and torch.equal(key, value)
        assert bool(key.isinf().any()) == (dtype == torch.float16)
    assert autosage_amd.paged_cache_read(codes, codes, *span, 16, key_exponents=e, value_exponents=e)[0].dtype == torch.bfloat16
