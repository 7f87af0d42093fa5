"""The paged cache and its attention on the CPU: results, refusals, and the native library's argument checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

import autosage_amd
from autosage_amd import _native
from autosage_amd.paged import _cache_struct, _CacheStruct
from tests.paged_common import E4M3, Cache, assert_attention, plain_attention, quantised_rows

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("window, biased", [(None, False), (5, False), (None, True), (7, True)])
def test_attention(dtype, quantised, window, biased):
    cache = Cache([0, 1, 9, 16, 37], 2, 6, 5, 8, dtype, quantised=quantised, seed=1)
    gen = torch.Generator().manual_seed(2)
    query = torch.randn(5, 6, 6, generator=gen).to(dtype)
    bias = {}
    if biased:
        bias = {"table": torch.randn(8, 6, generator=gen).to(dtype), "max_distance": 20, "bidirectional": False}
    want = plain_attention(cache, query, 0.3, window=window, **bias)
    args, exponents = cache.args("cpu")
    bias = {"bias_table" if k == "table" else k: v for k, v in bias.items()}
    out, lse = autosage_amd.paged_attention(query, *args, torch.tensor(cache.lengths), scale=0.3, window=window,
                                            return_lse=True, **bias, **exponents)
    assert out.dtype == dtype
    assert_attention(out, lse, want, dtype=dtype, quantised=quantised, lse_bound=1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
def test_write_then_read(dtype, quantised):
    cache = Cache([3, 0, 20], 2, 6, 5, 8, dtype, quantised=quantised, seed=3, room=1)
    (key_pages, value_pages, page_ptr, page_idx), exponents = cache.args("cpu")
    before = (key_pages.clone(), value_pages.clone())
    gen = torch.Generator().manual_seed(4)
    key, value = torch.randn(9, 2, 6, generator=gen).to(dtype), torch.randn(9, 2, 5, generator=gen).to(dtype)
    token_ptr, start = torch.tensor([0, 5, 5, 7]), torch.tensor([3, 0, 20])
    autosage_amd.paged_cache_write(key, value, key_pages, value_pages, page_ptr, page_idx, token_ptr, start, **exponents)
    got = autosage_amd.paged_cache_read(key_pages, value_pages, page_ptr, page_idx, token_ptr, start, 9,
                                        dtype=dtype, **exponents)
    for rows, back in zip((key, value), got):
        want = quantised_rows(rows)[0].to(dtype) if quantised else rows
        assert torch.equal(back[:7], want[:7]) and not back[7:].any()
    everything = autosage_amd.paged_cache_read(key_pages, value_pages, page_ptr, page_idx, torch.tensor([0, 3, 3, 23]),
                                               torch.tensor([0, 0, 0]), 23, dtype=dtype, **exponents)
    for kind, back in zip(("key", "value"), everything):
        assert torch.equal(back.double(), torch.cat(cache.rows[kind]).to(dtype).double())
    # nothing but the written places changed
    touched = torch.zeros(key_pages.shape[0], 8, dtype=torch.bool)
    for b, first, count in ((0, 3, 5), (2, 20, 2)):
        t = first + torch.arange(count)
        touched[page_idx[page_ptr[b] + t // 8], t % 8] = True
    for old, new in zip(before, (key_pages, value_pages)):
        a, b = (x.view(torch.uint8).transpose(1, 2)[~touched] for x in (old, new))
        assert torch.equal(a, b)


def test_quantised_numbers_at_the_edges():
    """Rows of zeros, of the largest and smallest numbers, of 448 exactly and just above, and what is not finite."""
    tiny = 2.0**-149
    rows = torch.tensor([[0.0, -0.0, 0.0], [448.0, 1.0, -3.3], [448.0001, 1.0, 2.0**-9], [3.4e38, -1e38, 1.0],
                         [tiny, -tiny, 0.0], [2.0**-126, 2.0**-130, 2.0**-140], [17.0, 19.0, 1.0625]])
    key_pages = torch.zeros(1, 1, 8, 3, dtype=E4M3)
    value_pages = torch.zeros(1, 1, 8, 3, dtype=E4M3)
    key_e, value_e = torch.zeros(1, 1, 8, dtype=torch.int8), torch.zeros(1, 1, 8, dtype=torch.int8)
    lists = (torch.tensor([0, 1]), torch.tensor([0]))
    span = (torch.tensor([0, 7]), torch.tensor([0]))
    x = rows[:, None]
    autosage_amd.paged_cache_write(x, x, key_pages, value_pages, *lists, *span, key_exponents=key_e,
                                   value_exponents=value_e)
    back, _ = autosage_amd.paged_cache_read(key_pages, value_pages, *lists, *span, 7, dtype=torch.float32,
                                            key_exponents=key_e, value_exponents=value_e)
    values, e = quantised_rows(rows)
    assert torch.equal(key_e[0, 0, :7].long(), e) and torch.equal(back[:, 0], values.float())
    assert back[3, 0, 0] == float("inf")  # 3.4e38 is held as 2^128
    odd = torch.tensor([[float("inf"), 1.0, 300.0], [float("nan"), -float("inf"), 2.0]])[:, None]
    autosage_amd.paged_cache_write(odd, odd, key_pages, value_pages, *lists, torch.tensor([0, 2]), span[1],
                                   key_exponents=key_e, value_exponents=value_e)
    back, _ = autosage_amd.paged_cache_read(key_pages, value_pages, *lists, torch.tensor([0, 2]), span[1], 2,
                                            dtype=torch.float32, key_exponents=key_e, value_exponents=value_e)
    assert back[0, 0].isnan().tolist() == [True, False, False] and back[0, 0, 1:].tolist() == [1.0, 288.0]  # steps of 32 from 256 on
    assert back[1, 0].isnan().tolist() == [True, True, False] and back[1, 0, 2] == 2.0


def test_lengths_and_pages_that_do_not_fit():
    cache = Cache([4, 9, 12], 1, 4, 4, 4, torch.float32, seed=5)
    (k, v, ptr, idx), _ = cache.args("cpu")
    query = torch.randn(3, 1, 4)
    call = autosage_amd.paged_attention
    good = call(query, k, v, ptr, idx, torch.tensor([4, 9, 12]))
    out, lse = call(query, k, v, ptr, idx, torch.tensor([5, 9, 12]), return_lse=True)  # one token more than its page holds
    assert out[0].isnan().all() and lse[0].isnan().all() and torch.equal(out[1:], good[1:])
    assert call(query, k, v, ptr, idx, torch.tensor([4, 9, 12]), max_length=9)[2].isnan().all()
    idx = idx.clone()
    idx[1] = k.size(0)
    out = call(query, k, v, ptr, idx, torch.tensor([4, 9, 12]))
    assert out[1].isnan().all() and torch.equal(out[[0, 2]], good[[0, 2]])
    assert not call(query, k, v, ptr, idx, torch.tensor([0, -3, 0])).any()


def test_validation(monkeypatch):
    cache = Cache([4, 9], 1, 4, 4, 4, torch.float32, seed=6)
    (k, v, ptr, idx), _ = cache.args("cpu")
    query, rows = torch.randn(2, 1, 4), torch.randn(2, 1, 4)
    one = torch.tensor([0, 1, 2])
    monkeypatch.setenv("AUTOSAGE_VALIDATE", "1")
    good = torch.tensor([4, 9])
    autosage_amd.paged_attention(query, k, v, ptr, idx, good)
    autosage_amd.paged_cache_write(rows, rows, k, v, ptr, idx, one, torch.tensor([3, 9]))
    bad_idx = idx.clone()
    bad_idx[0] = -1
    for args, message in [((ptr + 1, idx, good), "page_ptr"), ((ptr, bad_idx, good), "page ids"),
                          ((ptr, idx, good + 4), "more tokens"), ((ptr, idx, -good), "negative")]:
        with pytest.raises(ValueError, match=message):
            autosage_amd.paged_attention(query, k, v, *args)
    with pytest.raises(ValueError, match="max_length"):
        autosage_amd.paged_attention(query, k, v, ptr, idx, good, max_length=8)
    twice = torch.tensor([0, 0, 1, 2])  # the first page of both lists
    for token_ptr, start, lists, message in [
            (torch.tensor([0, 1, 3]), good - 1, (ptr, idx), "token_ptr"), (one, good + 4, (ptr, idx), "more tokens"),
            (one, torch.tensor([-1, 0]), (ptr, idx), "token_ptr"),
            (one, torch.tensor([2, 2]), (torch.tensor([0, 1, 4]), twice), "same place")]:
        with pytest.raises(ValueError, match=message):
            autosage_amd.paged_cache_write(rows, rows, k, v, *lists, token_ptr, start)


def test_refusals():
    cache = Cache([4, 9], 2, 4, 3, 4, torch.float32, seed=7)
    (k, v, ptr, idx), _ = cache.args("cpu")
    coded = Cache([4, 9], 2, 4, 3, 4, torch.float32, quantised=True, seed=7)
    (ck, cv, _, _), e = coded.args("cpu")
    query, lengths = torch.randn(2, 4, 4), torch.tensor([4, 9])
    attention, write, read = autosage_amd.paged_attention, autosage_amd.paged_cache_write, autosage_amd.paged_cache_read
    key, value = torch.randn(2, 2, 4), torch.randn(2, 2, 3)
    span = (torch.tensor([0, 1, 2]), torch.tensor([3, 8]))
    table = torch.randn(8, 4)
    for error, call in [
        (ValueError, lambda: attention(query, k[0], v, ptr, idx, lengths)),
        (ValueError, lambda: attention(query, k, v[:, :1], ptr, idx, lengths)),
        (TypeError, lambda: attention(query, k, v.half(), ptr, idx, lengths)),
        (TypeError, lambda: attention(query, k.double(), v.double(), ptr, idx, lengths)),
        (TypeError, lambda: attention(query.half(), k, v, ptr, idx, lengths)),
        (ValueError, lambda: attention(query[:, :3], k, v, ptr, idx, lengths)),
        (ValueError, lambda: attention(query[:, :, :3], k, v, ptr, idx, lengths)),
        (ValueError, lambda: attention(query[:1], k, v, ptr, idx, lengths)),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths[:1])),
        (TypeError, lambda: attention(query, k, v, ptr, idx, lengths.float())),
        (TypeError, lambda: attention(query, k, v, ptr.float(), idx, lengths)),
        (ValueError, lambda: attention(query, k, v, ptr, idx[None], lengths)),
        (ValueError, lambda: attention(query, k, v, ptr[:0], idx, lengths)),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths, window=0)),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths, max_length=-1)),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths, max_distance=9)),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths, bias_table=table)),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths, bias_table=table[:, :2], max_distance=9)),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths, bias_table=table[:7], max_distance=9)),
        (TypeError, lambda: attention(query, k, v, ptr, idx, lengths, bias_table=table.half(), max_distance=9)),
        (ValueError, lambda: attention(query, k, v, ptr, idx, lengths, **e)),
        (ValueError, lambda: attention(query, ck, cv, ptr, idx, lengths)),
        (ValueError, lambda: attention(query, ck, cv, ptr, idx, lengths, key_exponents=e["key_exponents"])),
        (TypeError, lambda: attention(query, ck, cv, ptr, idx, lengths, key_exponents=e["key_exponents"].int(),
                                      value_exponents=e["value_exponents"])),
        (ValueError, lambda: attention(query, ck, cv, ptr, idx, lengths, key_exponents=e["key_exponents"][:1],
                                       value_exponents=e["value_exponents"])),
        (ValueError, lambda: attention(query, k.transpose(2, 3), v, ptr, idx, lengths)),
        (ValueError, lambda: attention(torch.randn(2, 2, 257), torch.randn(4, 2, 4, 257), torch.randn(4, 2, 4, 3), ptr,
                                       idx, lengths)),
        (ValueError, lambda: attention(query, k[:0], v[:0], ptr, idx, lengths)),
        (RuntimeError, lambda: attention(query.clone().requires_grad_(), k, v, ptr, idx, lengths)),
        (ValueError, lambda: write(key[:1], value, k, v, ptr, idx, *span)),
        (ValueError, lambda: write(key[:, :1], value, k, v, ptr, idx, *span)),
        (ValueError, lambda: write(value, key, k, v, ptr, idx, *span)),
        (TypeError, lambda: write(key.half(), value.half(), k, v, ptr, idx, *span)),
        (TypeError, lambda: write(key.half(), value, ck, cv, ptr, idx, *span, **e)),
        (ValueError, lambda: write(key, value, k, v, ptr, idx, span[0][:2], span[1])),
        (ValueError, lambda: write(key, value, k, v, ptr, idx, span[0], span[1][:1])),
        (TypeError, lambda: write(key, value, k, v, ptr, idx, span[0].float(), span[1])),
        (ValueError, lambda: write(key, value, k[:1].expand(4, 2, 4, 4), v[:4], ptr, idx, *span)),
        (RuntimeError, lambda: write(key.clone().requires_grad_(), value, k, v, ptr, idx, *span)),
        (ValueError, lambda: read(k, v, ptr, idx, *span, -1)),
        (RuntimeError, lambda: read(k.clone().requires_grad_(), v, ptr, idx, *span, 2)),
        (TypeError, lambda: read(k, v, ptr, idx, *span, 2, dtype=torch.float16)),
        (TypeError, lambda: read(ck, cv, ptr, idx, *span, 2, dtype=torch.float64, **e)),
    ]:
        with pytest.raises(error):
            call()
    with torch.no_grad():
        attention(query.clone().requires_grad_(), k, v, ptr, idx, lengths)


def test_no_sequences_and_no_tokens():
    cache = Cache([4], 2, 4, 3, 4, torch.float32, seed=8)
    (k, v, _, idx), _ = cache.args("cpu")
    none = torch.zeros(0, dtype=torch.long)
    ptr = torch.zeros(1, dtype=torch.long)
    assert autosage_amd.paged_attention(torch.zeros(0, 4, 4), k, v, ptr, idx, none).shape == (0, 4, 3)
    key, value = autosage_amd.paged_cache_read(k, v, ptr, idx, ptr, none, 3)
    assert key.shape == (3, 2, 4) and value.shape == (3, 2, 3) and not key.any() and not value.any()
    autosage_amd.paged_cache_write(torch.zeros(0, 2, 4), torch.zeros(0, 2, 3), k, v, ptr, idx, ptr, none)


def test_native_argument_checks_come_before_any_launch():
    path = _native.package_library_path()
    if not path.exists():
        pytest.skip("HIP library not built")
    lib = _native.open_library(path)
    cache = Cache([4, 9], 2, 4, 3, 4, torch.float32, seed=9)
    (k, v, ptr, idx), _ = cache.args("cpu")

    def struct(**changes):
        c = _CacheStruct.from_buffer(_cache_struct(k, v, ptr, idx, None, None))
        for name, what in changes.items():
            setattr(c, name, what)
        return ctypes.byref(c)

    two = (ctypes.c_int64 * 2)(8, 4)
    fake = 256

    def attention(c, group=2, dtype=0, window=0, bound=-1, table=None, buckets=0, borders=None, sides=0, ws=fake,
                  ws_bytes=1 << 30, query=fake):
        return lib.as_paged_attention(c, query, two, fake, None, fake, group, 1.0, window, table, buckets, borders,
                                      sides, bound, dtype, ws, ws_bytes, None)

    for status, call, message in [
        (1, lambda: attention(None), b"null cache pointer"),
        (1, lambda: attention(struct(dtype=4)), b"the cache's dtype"),
        (1, lambda: attention(struct(dtype=3)), b"an e4m3 cache has exponents"),
        (1, lambda: attention(struct(pages=0)), b"a cache has 1 to"),
        (1, lambda: attention(struct(page_size=0)), b"a cache has 1 to"),
        (1, lambda: attention(struct(heads=0)), b"heads must lie"),
        (3, lambda: attention(struct(key_width=257)), b"key and value widths"),
        (1, lambda: attention(struct(key_pages=None)), b"null pointer argument"),
        (1, lambda: attention(struct(key_pages=k.data_ptr() + 2)), b"the pages must be aligned"),
        (1, lambda: attention(struct(), dtype=1), b"a cache that is not quantised"),
        (1, lambda: attention(struct(), dtype=3), b"dtype must be"),
        (1, lambda: attention(struct(), group=0), b"query heads must lie"),
        (1, lambda: attention(struct(), group=40000), b"query heads must lie"),
        (1, lambda: attention(struct(), window=-1), b"window and max_length"),
        (1, lambda: attention(struct(), table=fake, buckets=257), b"the number of buckets"),
        (1, lambda: attention(struct(), table=fake, buckets=3, sides=1), b"two sides need"),
        (1, lambda: attention(struct(), table=fake, buckets=3), b"null borders"),
        (1, lambda: attention(struct(), table=fake, buckets=3, borders=(ctypes.c_int32 * 3)(0, 2, 1)), b"borders must"),
        (4, lambda: attention(struct(page_idx_len=1 << 20), ws=None), b"paged attention needs"),
        (4, lambda: attention(struct(page_idx_len=1 << 20), ws_bytes=1000), b"paged attention needs"),
        (1, lambda: attention(struct(), query=None), b"null pointer argument"),
        (0, lambda: attention(struct(sequences=0)), b""),
        (1, lambda: lib.as_paged_cache_write(struct(), fake, two, fake, two, fake, fake, 2, 2, None), b"a cache that"),
        (3, lambda: lib.as_paged_cache_write(struct(), fake, two, fake, two, fake, fake, 1 << 50, 0, None), b"at most 2^26"),
        (1, lambda: lib.as_paged_cache_write(struct(), fake, two, None, two, fake, fake, 2, 0, None), b"null pointer"),
        (1, lambda: lib.as_paged_cache_write(struct(), fake, None, fake, two, fake, fake, 2, 0, None), b"null strides"),
        (0, lambda: lib.as_paged_cache_write(struct(), fake, two, fake, two, fake, fake, 0, 0, None), b""),
        (1, lambda: lib.as_paged_cache_read(struct(), fake + 1, fake, fake, fake, 2, 0, None), b"key and value must"),
        (1, lambda: lib.as_paged_cache_read(struct(sequences=0), fake, fake, fake, fake, 2, 0, None), b"tokens without"),
        (1, lambda: lib.as_csr_position_bias(fake, fake, None, fake, fake, None, 4, 4, 2, 8, None, 0, 0, fake, 8, None),
         b"null borders"),
        (1, lambda: lib.as_csr_position_bias(fake, fake, None, fake, fake, None, 4, 4, 2, 8, None, 0, 3, fake, 8, None),
         b"dtype must"),
        (1, lambda: lib.as_csr_position_bias(fake, fake, None, fake, fake, None, 0, 4, 2, 8, None, 0, 0, fake, 8, None),
         b"edges without"),
        (1, lambda: lib.as_csr_position_bias(fake, None, None, fake, fake, None, 4, 4, 2, 8, None, 0, 0, fake, 8, None),
         b"null pointer"),
        (1, lambda: lib.as_csr_position_bias(fake, fake, None, fake, fake, fake + 1, 4, 4, 2, 8, None, 0, 0, fake, 8, None),
         b"found must be"),
        (3, lambda: lib.as_csr_position_bias(fake, fake, None, fake, fake, None, 4, 1 << 31, 2, 8, None, 0, 0, fake, 8, None),
         b"at most 2^30"),
        (1, lambda: lib.as_csr_position_bias_backward(None, fake, fake, 4, 2, 2, 0, fake, 1 << 20, None), b"null pointer"),
        (1, lambda: lib.as_csr_position_bias_backward(fake, fake, fake, 4, 2, 257, 0, fake, 1 << 20, None),
         b"the number of buckets"),
        (4, lambda: lib.as_csr_position_bias_backward(fake, fake, fake, 4, 2, 2, 0, fake, 8, None),
         b"the position bias gradient needs"),
        (0, lambda: lib.as_csr_position_bias(None, None, None, fake, None, None, 0, 0, 2, 2, (ctypes.c_int32 * 2)(0, 1), 0,
                                             0, fake, 8, None), b""),
    ]:
        assert call() == status, message
        assert lib.as_last_error().startswith(message), lib.as_last_error()


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("bad", [-1, 10**6, 2**40, -(2**40)])
def test_tokens_whose_page_is_outside_the_cache(quantised, bad):
    """They are not written and read as zeros; the others are."""
    cache = Cache([4, 9], 1, 8, 8, 4, torch.float32, quantised=quantised, seed=10)
    (k, v, ptr, idx), e = cache.args("cpu")
    idx = idx.clone()
    idx[2] = bad  # tokens 4 to 7 of the second sequence
    rows = torch.randn(9, 1, 8)
    before = k.view(torch.uint8).clone()
    span = (torch.tensor([0, 0, 9]), torch.tensor([0, 0]))
    autosage_amd.paged_cache_write(rows, rows, k, v, ptr, idx, *span, **e)
    key, value = autosage_amd.paged_cache_read(k, v, ptr, idx, *span, 9, dtype=torch.float32, **e)
    want = quantised_rows(rows)[0].float() if quantised else rows
    for back in (key, value):
        assert not back[4:8].any() and torch.equal(back[:4], want[:4]) and torch.equal(back[8], want[8])
    others = [p for p in range(k.size(0)) if p not in (idx[1], idx[3])]
    assert torch.equal(k.view(torch.uint8)[others], before[others])


def test_lists_outside_the_page_ids():
    """What a list names outside ``page_idx`` is no page: nothing written, zeros, NaN; a list inside is as it was."""
    cache = Cache([4, 9], 1, 8, 8, 4, torch.float32, seed=11)
    (k, v, ptr, idx), _ = cache.args("cpu")
    query, rows = torch.randn(2, 1, 8), torch.randn(8, 1, 8)
    lengths, span = torch.tensor([4, 9]), (torch.tensor([0, 4, 8]), torch.tensor([0, 0]))
    good = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths)
    before = k.clone()
    for lists in (ptr + 10**6, ptr - 5, ptr - 10**6, ptr.flip(0), torch.tensor([-4, -3, -1])):
        assert autosage_amd.paged_attention(query, k, v, lists, idx, lengths).isnan().all()
        autosage_amd.paged_cache_write(rows, rows, k, v, lists, idx, *span)
        assert not autosage_amd.paged_cache_read(k, v, lists, idx, *span, 8)[0].any()
    assert torch.equal(k.nan_to_num(7.0), before.nan_to_num(7.0))
    one = torch.tensor([-1, 1, 10**6])  # cut to [0, 1) and [1, 4)
    assert torch.equal(autosage_amd.paged_attention(query, k, v, one, idx, lengths), good)


@pytest.mark.parametrize("quantised", [False, True])
def test_rows_in_front_of_the_first_token(quantised):
    """``token_ptr`` need not begin at 0: rows in front of it are padding, as those behind its end are."""
    cache = Cache([4, 9], 1, 8, 8, 4, torch.float32, quantised=quantised, seed=12)
    (k, v, ptr, idx), e = cache.args("cpu")
    rows = torch.randn(9, 1, 8)
    span = (torch.tensor([2, 3, 7]), torch.tensor([3, 4]))
    autosage_amd.paged_cache_write(rows, rows, k, v, ptr, idx, *span, **e)
    key, value = autosage_amd.paged_cache_read(k, v, ptr, idx, *span, 9, dtype=torch.float32, **e)
    want = quantised_rows(rows)[0].float() if quantised else rows
    for back in (key, value):
        assert torch.equal(back[2:7], want[2:7]) and not back[:2].any() and not back[7:].any()
    # the tokens in front of those
    old = autosage_amd.paged_cache_read(k, v, ptr, idx, torch.tensor([0, 3, 7]), torch.tensor([0, 0]), 7,
                                        dtype=torch.float32, **e)[0].double()
    assert torch.equal(old, torch.cat([cache.rows["key"][0][:3], cache.rows["key"][1][:4]]).float().double())


def test_token_lists_that_begin_anywhere():
    """Where a position passes 64 bits there is no place, and the other sequence's tokens keep theirs."""
    cache = Cache([4, 9], 1, 8, 8, 4, torch.float32, seed=19)
    rows = torch.randn(6, 1, 8)
    for own, begin in [(-(2**62) - 10, 2**62 - 1), (-(2**63), 2**62 - 1), (-(2**63), 0), (-(2**62), 2**62),
                       (-(2**62), 2**63 - 1), (-(2**63), -(2**63)), (-5, -(2**63))]:
        (k, v, ptr, idx), _ = cache.args("cpu")
        k, v = k.clone(), v.clone()
        token_ptr, start = torch.tensor([own, 3, 6]), torch.tensor([begin, 5])
        autosage_amd.paged_cache_write(rows, rows, k, v, ptr, idx, token_ptr, start)
        key, value = autosage_amd.paged_cache_read(k, v, ptr, idx, token_ptr, start, 6)
        for back in (key, value):
            assert not back[:3].any() and torch.equal(back[3:], rows[3:])


def test_validation_of_lists_with_room(monkeypatch):
    """Only the entries that a call reaches have to be pages: a table padded with -1, windows that are past the first
    pages (given back, or never kept), some of a batch's sequences and rows."""
    monkeypatch.setenv("AUTOSAGE_VALIDATE", "1")
    cache = Cache([9, 22], 1, 8, 8, 4, torch.float32, seed=13)
    (k, v, ptr, idx), _ = cache.args("cpu")
    query, rows, lengths = torch.randn(2, 1, 8), torch.randn(6, 1, 8), torch.tensor([9, 22])
    table = torch.full((2, 8), -1)
    table[0, :3], table[1, :6] = idx[:3], idx[3:]
    wide = torch.arange(3) * 8
    attention, write, read = autosage_amd.paged_attention, autosage_amd.paged_cache_write, autosage_amd.paged_cache_read
    want = attention(query, k, v, ptr, idx, lengths)
    assert torch.equal(attention(query, k, v, wide, table.flatten(), lengths), want)
    assert torch.equal(attention(query[1:], k, v, wide[1:], table.flatten(), lengths[1:]), want[1:])
    write(rows, rows, k, v, wide, table.flatten(), torch.tensor([1, 3, 5]), lengths)
    back, _ = read(k, v, wide, table.flatten(), torch.tensor([1, 3, 5]), lengths, 6)
    assert torch.equal(back[1:5], rows[1:5])
    want = attention(query, k, v, ptr, idx, lengths, window=5)
    table[0, 0], table[1, :4] = 10**9, -1  # in front of tokens 4 and 17
    assert torch.equal(attention(query, k, v, wide, table.flatten(), lengths, window=5), want)
    for bad in (lambda: attention(query, k, v, wide, table.flatten(), lengths, window=6),
                lambda: attention(query, k, v, wide, table.flatten(), lengths + 4),
                lambda: read(k, v, wide, table.flatten(), torch.tensor([0, 1, 2]), torch.tensor([3, 17]), 2),
                lambda: write(rows, rows, k, v, wide, table.flatten(), torch.tensor([0, 2, 4]), torch.tensor([11, 17]))):
        with pytest.raises(ValueError, match="page ids"):
            bad()
    with pytest.raises(ValueError, match="page_ptr"):
        attention(query, k, v, wide - 1, table.flatten(), lengths)
    with pytest.raises(ValueError, match="token_ptr"):
        read(k, v, wide, table.flatten(), torch.tensor([-1, 1, 2]), torch.tensor([4, 17]), 2)
    with pytest.raises(ValueError, match="more tokens"):
        attention(query, k, v, wide, table.flatten(), torch.tensor([9, 33]), window=1)


def test_forward_mode_is_refused():
    cache = Cache([4, 9], 1, 8, 8, 4, torch.float32, seed=14)
    (k, v, ptr, idx), _ = cache.args("cpu")
    query, rows, span = torch.randn(2, 1, 8), torch.randn(2, 1, 8), (torch.tensor([0, 1, 2]), torch.tensor([3, 8]))
    lengths = torch.tensor([4, 9])
    with torch.autograd.forward_ad.dual_level():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: autosage_amd.paged_attention(dual(query), k, v, ptr, idx, lengths),
                     lambda: autosage_amd.paged_attention(query, k, dual(v), ptr, idx, lengths),
                     lambda: autosage_amd.paged_attention(query, k, v, ptr, idx, lengths, max_distance=9,
                                                          bias_table=dual(torch.randn(8, 1))),
                     lambda: autosage_amd.paged_cache_write(rows, dual(rows), k, v, ptr, idx, *span),
                     lambda: autosage_amd.paged_cache_read(dual(k), v, ptr, idx, *span, 2)):
            with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                call()
        autosage_amd.paged_attention(query, k, v, ptr, idx, lengths)


def test_8_bit_numbers_beyond_the_largest_of_a_type():
    """As documented: held as 65,536, which float16 has not; the largest number that stays below is off by 1/16."""
    k, v = torch.zeros(1, 1, 4, 2, dtype=E4M3), torch.zeros(1, 1, 4, 2, dtype=E4M3)
    names = {f"{n}_exponents": torch.zeros(1, 1, 4, dtype=torch.int8) for n in ("key", "value")}
    lists = (torch.tensor([0, 1]), torch.tensor([0]), torch.tensor([0, 3]), torch.tensor([0]))
    rows = torch.tensor([[65504.0, 1.0], [63488.0, -63456.0], [-63456.0, 57344.0]], dtype=torch.float16)[:, None]
    autosage_amd.paged_cache_write(rows, rows, k, v, *lists, **names)
    for dtype, want in ((torch.float16, [[torch.inf, 1.0], [torch.inf, -61440.0], [-61440.0, 57344.0]]),
                        (torch.bfloat16, [[65536.0, 1.0], [65536.0, -61440.0], [-61440.0, 57344.0]])):
        back, _ = autosage_amd.paged_cache_read(k, v, *lists, 3, dtype=dtype, **names)
        assert back[:, 0].tolist() == want


def test_native_groups_whose_product_passes_64_bits():
    path = _native.package_library_path()
    if not path.exists():
        pytest.skip("HIP library not built")
    lib = _native.open_library(path)
    cache = Cache([4, 9], 4, 4, 3, 4, torch.float32, seed=9)
    (k, v, ptr, idx), _ = cache.args("cpu")
    c = _CacheStruct.from_buffer(_cache_struct(k, v, ptr, idx, None, None))
    c.sequences = 0  # nothing is launched
    two = (ctypes.c_int64 * 2)(8, 4)
    for group, status in ((2**62, 1), (2**62 + 1, 1), (16384, 1), (16383, 0)):
        assert lib.as_paged_attention(ctypes.byref(c), 256, two, 256, None, 256, group, 1.0, 0, None, 0, None, 0, -1, 0,
                                      256, 1 << 50, None) == status
        if status:
            assert lib.as_last_error().startswith(b"query heads must lie")
            assert lib.as_paged_attention_workspace_bytes(ctypes.byref(c), group, 0, -1) == 0


def test_validation_of_starts_whose_sum_passes_64_bits(monkeypatch):
    monkeypatch.setenv("AUTOSAGE_VALIDATE", "1")
    cache = Cache([4, 9], 1, 4, 4, 4, torch.float32, seed=15)
    (k, v, ptr, idx), _ = cache.args("cpu")
    rows, one = torch.randn(2, 1, 4), torch.tensor([0, 1, 2])
    for start in (2**63 - 1, 2**62, 2**40):
        with pytest.raises(ValueError, match="more tokens"):
            autosage_amd.paged_cache_write(rows, rows, k, v, ptr, idx, one, torch.tensor([start, 3]))
