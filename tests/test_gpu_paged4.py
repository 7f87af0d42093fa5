"""The paged cache of 4-bit numbers and its attention on the GPU against 64-bit results: every place outside the
sequences holds NaN."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu
from tests.paged4_common import E2M1, E8M0, Cache4, quantised_pairs
from tests.paged_common import assert_attention, plain_attention

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LENGTHS = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 300]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _attend(lengths, heads, group, width, value_width, page, dtype, *, window=None, bias=None, seed=0,
            max_length="given", scale=None, query=None, **layout):
    cache = Cache4(lengths, heads, width, value_width, page, dtype, seed=seed, **layout)
    gen = torch.Generator().manual_seed(seed + 1)
    if query is None:
        query = torch.randn(len(lengths), heads * group, width, generator=gen).to(dtype)
    scale = width**-0.5 if scale is None else scale
    plain, own = {}, {}
    if bias is not None:
        buckets, distance, both = bias
        table = torch.randn(buckets, heads * group, generator=gen).to(dtype)
        plain = {"table": table, "max_distance": distance, "bidirectional": both}
        own = {"bias_table": table.cuda(), "max_distance": distance, "bidirectional": both}
    want = plain_attention(cache, query, scale, window=window, **plain)
    # A weight below 2^-126 (float32's smallest normal number) may be zero, as the hardware's exp2 has it: n of them, each
    # times a value, over a sum of at least 1.  Where one token takes all of the weight and its value is 0, that is
    # all that the result is (scale 4, float32: 1.6e-39 in 64 bits, 0 in 32).
    for b, n in enumerate(lengths):
        if n > 0:
            want[2][b] += n * 2.0**-126 * cache.rows["value"][b].abs().max()
    args, exponents = cache.args()
    bound = max(lengths) if max_length == "given" else max_length
    out, lse = autosage_amd.paged_attention(query.cuda(), *args, torch.tensor(lengths).cuda(), scale=scale,
                                            window=window, max_length=bound, return_lse=True, **own, **exponents)
    # scores are at most a few hundred here: fp32 keeps them to 1e-4
    worst = assert_attention(out, lse, want, dtype=dtype, quantised=True, lse_bound=2e-4)
    print(f"worst error over bound {worst:.3f}")
    return cache, query, out, lse


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width, value_width", [(2, 30), (32, 64), (72, 34), (128, 128), (256, 254), (6, 6)])
@pytest.mark.parametrize("page", [1, 7, 16])
def test_write_then_read(dtype, width, value_width, page):
    lengths, new, heads = [13, 0, 40, 5], [9, 1, 100, 0], 3
    counts = [-(-(n + m) // page) for n, m in zip(lengths, new)]
    pages = sum(counts) + 2
    page_ptr = torch.tensor([0] + counts).cumsum(0).cuda()
    page_idx = torch.randperm(pages, generator=torch.Generator().manual_seed(page))[:sum(counts)].cuda()
    token_ptr, start = torch.tensor([0] + new).cumsum(0).cuda(), torch.tensor(lengths).cuda()
    gen = torch.Generator().manual_seed(width + page)
    tokens = sum(new) + 3  # padding behind the last sequence
    rows = [(torch.randn(tokens, heads, w, generator=gen) * torch.exp(torch.randn(tokens, heads, w, generator=gen))).to(
        dtype) for w in (width, value_width)]
    held, names = [], {}
    for kind, w in (("key", width), ("value", value_width)):
        held.append(torch.full((pages, heads, page, w // 2), 0xA5, dtype=torch.uint8, device="cuda").view(E2M1))
        names[kind + "_exponents"] = torch.full((pages, heads, page, -(-w // 32)), 77, dtype=torch.uint8,
                                                device="cuda").view(E8M0)
    span = (page_ptr, page_idx, token_ptr, start)
    autosage_amd.paged_cache_write(rows[0].cuda(), rows[1].cuda(), *held, *span, **names)
    back = autosage_amd.paged_cache_read(*held, *span, tokens, dtype=dtype, **names)
    sequence = torch.repeat_interleave(torch.arange(4), torch.tensor(new))
    at = start.cpu()[sequence] + torch.arange(sum(new)) - token_ptr.cpu()[sequence]
    where, place = page_idx.cpu()[page_ptr.cpu()[sequence] + at // page], at % page
    for x, got, codes, exponents in zip(rows, back, held, names.values()):
        values, packed, e = quantised_pairs(x[:sum(new)])
        assert torch.equal(got[:sum(new)].cpu(), values.to(dtype)) and not got[sum(new):].any()
        want = torch.full(codes.shape, 0xA5, dtype=torch.uint8)
        want[where, :, place] = packed
        assert torch.equal(codes.view(torch.uint8).cpu(), want)
        want = torch.full(exponents.shape, 77, dtype=torch.uint8)
        want[where, :, place] = e
        assert torch.equal(exponents.view(torch.uint8).cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("tokens, heads, width, value_width", [(3, 300, 34, 34), (40, 129, 2, 66), (1030, 1, 6, 96),
                                                               (2051, 3, 40, 40), (8200, 2, 64, 192), (16390, 5, 32, 10)])
def test_many_tokens_and_heads(dtype, tokens, heads, width, value_width):
    """From one token a workgroup to all that it takes: pages and rows as on the CPU."""
    gen = torch.Generator().manual_seed(tokens)
    rows = [torch.randn(tokens + 2, heads, w, generator=gen).to(dtype) for w in (width, value_width)]
    lengths = [tokens // 3, tokens - tokens // 3 - 1, 1]
    counts = [-(-(n + 1) // 5) for n in lengths]
    order = torch.randperm(sum(counts), generator=gen)
    results = []
    for device in ("cpu", "cuda"):
        pages = [torch.zeros(sum(counts), heads, 5, w // 2, dtype=torch.uint8, device=device).view(E2M1)
                 for w in (width, value_width)]
        e = [torch.zeros(sum(counts), heads, 5, -(-w // 32), dtype=torch.uint8, device=device).view(E8M0)
             for w in (width, value_width)]
        names = dict(zip(("key_exponents", "value_exponents"), e))
        span = [torch.tensor([0] + counts).cumsum(0), order, torch.tensor([1] + lengths).cumsum(0), torch.tensor([1, 1, 1])]
        span = [t.to(device) for t in span]
        autosage_amd.paged_cache_write(*(r.to(device) for r in rows), *pages, *span, **names)
        back = autosage_amd.paged_cache_read(*pages, *span, tokens + 2, dtype=dtype, **names)
        results.append([t.view(torch.uint8).cpu() for t in (*pages, *e)] + [t.cpu() for t in back])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_the_gpu_holds_what_the_cpu_holds():
    """Random bits of float32 and all numbers of the 16-bit types, those that are not finite among them."""
    gen = torch.Generator().manual_seed(3)
    bits = torch.randint(-2**31, 2**31, (2048, 2, 64), generator=gen, dtype=torch.int64).to(torch.int32)
    near = torch.randint(0, 256, (2048, 2, 64), generator=gen).float() / 32 * 2.0 ** torch.randint(-130, 120, (2048, 2, 1), generator=gen)
    all16 = torch.arange(-32768, 32768).to(torch.int16).view(512, 2, 64)
    for rows in (bits.view(torch.float32), near, all16.view(torch.bfloat16), all16.view(torch.float16),
                 all16.view(torch.bfloat16)[torch.randperm(512, generator=gen)].flatten()[torch.randperm(65536, generator=gen)].view(512, 2, 64)):
        tokens = rows.size(0)
        results = []
        for device in ("cpu", "cuda"):
            k, v = (torch.zeros(tokens // 16, 2, 16, 32, dtype=torch.uint8, device=device).view(E2M1) for _ in range(2))
            e = [torch.zeros(tokens // 16, 2, 16, 2, dtype=torch.uint8, device=device).view(E8M0) for _ in range(2)]
            names = dict(zip(("key_exponents", "value_exponents"), e))
            span = [torch.tensor(x, device=device) for x in ([0, tokens // 16], list(range(tokens // 16)), [0, tokens], [0])]
            autosage_amd.paged_cache_write(rows.to(device), rows.to(device), k, v, *span, **names)
            back = autosage_amd.paged_cache_read(k, v, *span, tokens, dtype=rows.dtype, **names)
            results.append([t.view(torch.uint8).cpu() for t in (k, v, *e)] + [t.cpu() for t in back])
        nan = results[0][2] == 255  # codes of groups of NaN say nothing
        for i, (a, b) in enumerate(zip(*results)):
            if i < 2:
                a, b = (t.unflatten(-1, (2, 16)).masked_fill(nan[..., None], 0) for t in (a, b))
            assert torch.equal(a, b) if i < 4 else torch.equal(a.nan_to_num(7.5), b.nan_to_num(7.5)) and torch.equal(
                a.isnan(), b.isnan()), i


def test_numbers_in_every_type():
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 16, 16)
    e = torch.arange(256, dtype=torch.uint8).view(256, 1, 1, 1).expand(256, 1, 16, 1).contiguous()
    every = codes.expand(256, 1, 16, 16).contiguous()
    span = [torch.tensor(x) for x in ([0, 256], list(range(256)), [0, 4096], [0])]
    for dtype in DTYPES:
        results = []
        for device in ("cpu", "cuda"):
            k, exponents = every.to(device).view(E2M1), e.to(device).view(E8M0)
            results.append(autosage_amd.paged_cache_read(k, k, *(t.to(device) for t in span), 4096, dtype=dtype,
                                                         key_exponents=exponents, value_exponents=exponents)[0].cpu())
        assert torch.equal(results[0].isnan(), results[1].isnan())
        assert torch.equal(results[0].nan_to_num(7.5), results[1].nan_to_num(7.5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 7, 8, 12, 16, 64])
def test_lengths_and_pages(dtype, page):
    _attend(LENGTHS, 2, 3, 64, 64, page, dtype, seed=page)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("width, value_width", [(2, 2), (4, 6), (16, 16), (40, 24), (34, 66), (72, 72), (96, 32),
                                                (128, 128), (130, 64), (64, 200), (192, 128), (256, 256), (254, 250),
                                                (8, 256), (160, 10)])
def test_widths(dtype, page, width, value_width):
    _attend([1, 50, 140], 2, 2, width, value_width, page, dtype, seed=width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, group", [(1, 1), (3, 4), (2, 7), (1, 16), (2, 17), (1, 40)])
def test_heads(dtype, heads, group):
    _attend([5, 40, 200], heads, group, 64, 64, 16, dtype, seed=heads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 15, 64, 1000])
@pytest.mark.parametrize("page", [16, 12])
def test_window(dtype, window, page):
    _attend([0, 1, 15, 16, 64, 65, 130, 1500], 2, 2, 64, 64, page, dtype, window=window, seed=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [(32, 128, True), (32, 128, False), (2, 4, False), (256, 700, False)])
@pytest.mark.parametrize("window", [None, 50])
def test_bias(dtype, bias, window):
    _attend([0, 1, 40, 200, 900], 2, 3, 64, 64, 16, dtype, bias=bias, window=window, seed=bias[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("max_length", ["given", None, 9000])
def test_long_and_short_sequences_together(dtype, page, max_length):
    _attend([0, 1, 3000, 17, 513, 64, 512, 2049], 2, 4, 64, 96, page, dtype, max_length=max_length, seed=11)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width, value_width", [(128, 128), (40, 24), (256, 256), (100, 160)])
@pytest.mark.parametrize("window, bias", [(None, None), (1501, None), (None, (32, 128, False)), (1003, (32, 4000, True))])
def test_sequences_in_shares(dtype, width, value_width, window, bias):
    _attend([4000, 30, 0, 1700, 1], 2, 5, width, value_width, 16, dtype, window=window, bias=bias, max_length=None, seed=12)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [64, 3])
def test_one_long_sequence(dtype, page):
    _attend([9001], 1, 8, 128, 128, page, dtype, max_length=None, seed=13)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("layout", [{"interleaved": True}, {"offset": 1}, {"offset": 6}, {"room": 3}])
@pytest.mark.parametrize("width", [64, 40])
def test_layouts(dtype, page, layout, width):
    _attend([1, 40, 130, 600], 3, 2, width, width, page, dtype, seed=14, **layout)
    _attend([1, 40, 130, 600], 3, 2, width, width, page, dtype, seed=14, max_length=None, **layout)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_and_pages(dtype):
    """Queries, keys and values inside a projection; the cache interleaved."""
    cache = Cache4([20, 33], 2, 32, 32, 8, dtype, seed=15, interleaved=True, room=1)
    args, e = cache.args()
    rows = torch.randn(2, 8, 32, generator=torch.Generator().manual_seed(16)).to(dtype)
    wide = rows.cuda()
    lengths = torch.tensor(cache.lengths)
    autosage_amd.paged_cache_write(wide[:, 4:6], wide[:, 6:], *args, torch.arange(3).cuda(), lengths.cuda(), **e)
    for kind, at in (("key", 4), ("value", 6)):
        fresh = quantised_pairs(rows[:, at:at + 2])[0]
        cache.rows[kind] = [torch.cat((x, fresh[b:b + 1])) for b, x in enumerate(cache.rows[kind])]
    cache.lengths = (lengths + 1).tolist()
    out, lse = autosage_amd.paged_attention(wide[:, :4], *args, (lengths + 1).cuda(), scale=0.2, return_lse=True, **e)
    assert_attention(out, lse, plain_attention(cache, rows[:, :4], 0.2), dtype=dtype, quantised=True, lse_bound=2e-4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype):
    _attend([1, 40, 700], 2, 2, 64, 64, 16, dtype, scale=4.0, seed=17)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [64, 40])
def test_queries_of_many_magnitudes(dtype, width):
    """Numbers of one query from 2^-16 to 2^4, and one query of zeros."""
    gen = torch.Generator().manual_seed(18)
    query = torch.randn(3, 4, width, generator=gen) * 2.0 ** torch.randint(-16, 5, (3, 4, width), generator=gen)
    query[1, 2] = 0.0
    _attend([5, 40, 700], 2, 2, width, 64, 16, dtype, query=query.to(dtype), seed=18)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_length", [None, 60])
def test_rows_that_the_bias_masks(dtype, max_length):
    """A bias of -inf leaves nothing of a head, one of the lowest number leaves all of it."""
    lengths = [60, 3, 60]
    cache = Cache4(lengths, 1, 32, 32, 16, dtype, seed=19)
    args, e = cache.args()
    query = torch.randn(3, 3, 32, generator=torch.Generator().manual_seed(20)).to(dtype)
    table = torch.zeros(4, 3, dtype=dtype)
    table[:, 1] = -float("inf")
    table[:, 2] = torch.finfo(dtype).min
    out, lse = autosage_amd.paged_attention(query.cuda(), *args, torch.tensor(lengths).cuda(), scale=0.2,
                                            bias_table=table.cuda(), max_distance=8, bidirectional=False,
                                            max_length=max_length, return_lse=True, **e)
    assert not out[:, 1].any() and (lse[:, 1] == -float("inf")).all()
    want = plain_attention(cache, query, 0.2, table=table.double().clamp_min(-1e30).to(torch.float64), max_distance=8,
                           bidirectional=False)
    assert_attention(out[:, :1], lse[:, :1], tuple(t[:, :1] for t in want), dtype=dtype, quantised=True, lse_bound=2e-4)
    if dtype is torch.float16:  # the others' lowest number swallows every score: the mean of the values
        assert_attention(out[:, 2:], None, tuple(t[:, 2:] for t in want), dtype=dtype, quantised=True)
    else:
        for b, n in enumerate(lengths):
            mean = cache.rows["value"][b][:, 0].mean(0)
            assert torch.allclose(out[b, 2].double().cpu(), mean, rtol=2.0**-7, atol=1e-4 + 2.0**-8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [64, 40])
def test_groups_of_nan(dtype, width):
    """A NaN in a key or a value that is seen shows in its sequence (and, of a value, its columns) alone."""
    cache = Cache4([40, 40, 40, 40], 2, width, width, 16, dtype, seed=21)
    args, e = cache.args()
    query = torch.randn(4, 2, width, device="cuda").to(dtype)
    lengths = torch.tensor(cache.lengths).cuda()
    want = autosage_amd.paged_attention(query, *args, lengths, **e)
    assert want.isfinite().all()
    ptr, idx = cache.page_ptr, cache.page_idx
    e["key_exponents"].view(torch.uint8)[idx[ptr[1] + 1], 1, 3, 0] = 255
    e["value_exponents"].view(torch.uint8)[idx[ptr[2] + 2], 0, 5, 1] = 255
    for max_length in (None, 40):
        out = autosage_amd.paged_attention(query, *args, lengths, max_length=max_length, **e)
        assert out[1, 1].isnan().all() and out[2, 0, 32:].isnan().all()
        same = torch.ones_like(out, dtype=torch.bool)
        same[1, 1], same[2, 0, 32:] = False, False
        assert torch.allclose(out[same].float(), want[same].float(), rtol=2.0**-7, atol=2.0**-9)
    # not seen: a window in front of them
    out = autosage_amd.paged_attention(query, *args, lengths, window=2, **e)
    assert out.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 12])
def test_infinite_queries(dtype, page):
    """Finite heads stay as they are; an infinite number makes its head what the formula says (NaN or infinite scores)."""
    cache = Cache4([40, 700], 1, 64, 64, page, dtype, seed=22)
    args, e = cache.args()
    query = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(23)).to(dtype)
    want = plain_attention(cache, query, 0.125)
    bad = query.clone()
    bad[0, 1, 5], bad[1, 2, 63] = float("inf"), float("nan")
    out, lse = autosage_amd.paged_attention(bad.cuda(), *args, torch.tensor([40, 700]).cuda(), scale=0.125,
                                            return_lse=True, **e)
    assert out[1, 2].isnan().all() and out[0, 1].isnan().any()
    keep = torch.ones(2, 4, dtype=torch.bool)
    keep[0, 1], keep[1, 2] = False, False
    assert_attention(out.cpu()[keep], lse.cpu()[keep], tuple(t[keep] for t in want), dtype=dtype, quantised=True,
                     lse_bound=2e-4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("count", [65, 257, 1100])
@pytest.mark.parametrize("page", [8, 5])
def test_many_sequences(dtype, count, page):
    gen = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 90, (count,), generator=gen).tolist()
    lengths[count // 2] = 1300
    _attend(lengths, 1, 2, 32, 32, page, dtype, max_length=None, seed=24)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [64, 40])
def test_lengths_and_pages_that_do_not_fit(dtype, width):
    cache = Cache4([100, 30, 700, 5, 90], 2, width, width, 16, dtype, seed=25)
    (k, v, ptr, idx), e = cache.args()
    query = torch.randn(5, 4, width, device="cuda").to(dtype)
    good = autosage_amd.paged_attention(query, k, v, ptr, idx, torch.tensor(cache.lengths).cuda(), **e)
    idx = idx.clone()
    idx[ptr[2] + 40] = 2**40
    idx[ptr[4]] = -1
    lengths = torch.tensor([113, 30, 700, 6, 90]).cuda()
    for max_length in (None, 700):
        out, lse = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths, max_length=max_length, return_lse=True,
                                                **e)
        for b, bad in enumerate([True, False, True, False, True]):
            if bad:
                assert out[b].isnan().all() and lse[b].isnan().all(), b
        assert torch.allclose(out[1].float(), good[1].float(), rtol=2.0**-7, atol=2.0**-9)
    out = autosage_amd.paged_attention(query, k, v, ptr, idx, torch.tensor([20, 30, 10, 5, 0]).cuda(), max_length=20, **e)
    assert out[1].isnan().all() and out[0].isfinite().all() and not out[4].any()
    # lists outside the page ids, lengths below zero
    wild = torch.tensor([0, 5, 2**50, -3, 2, 2**62]).cuda()
    out = autosage_amd.paged_attention(query, k, v, wild, idx, torch.tensor([10, -5, 10, 10, 0]).cuda(), **e)
    assert not out[1].any() and not out[4].any()


def test_parts_joined_by_their_lse():
    dtype = torch.bfloat16
    cache, query, whole, _ = _attend([900], 2, 4, 128, 128, 16, dtype, seed=26)
    (k, v, ptr, idx), e = cache.args()
    parts = []
    for first, last in ((0, 512), (512, 900)):
        mine = idx[first // 16:-(-last // 16)].contiguous()
        parts.append(autosage_amd.paged_attention(
            query.cuda(), k, v, torch.tensor([0, mine.numel()]).cuda(), mine, torch.tensor([last - first]).cuda(),
            scale=128**-0.5, return_lse=True, **e))
    lse = torch.stack([p[1] for p in parts])
    share = torch.softmax(lse, 0)[..., None]
    joined = (share * torch.stack([p[0].float() for p in parts])).sum(0)
    assert torch.allclose(joined, whole.float(), rtol=2.0**-7, atol=2.0**-8)


def test_the_registered_operators_and_32_bit_lists(monkeypatch):
    monkeypatch.setenv("AUTOSAGE_VALIDATE", "1")
    cache = Cache4([20, 33], 2, 64, 32, 8, torch.bfloat16, seed=27, room=1)
    (k, v, ptr, idx), e = cache.args()
    query = torch.randn(2, 4, 64, device="cuda").bfloat16()
    rows = torch.randn(2, 2, 64, device="cuda").bfloat16(), torch.randn(2, 2, 32, device="cuda").bfloat16()
    lengths, one = torch.tensor([20, 33]).cuda(), torch.arange(3).cuda()
    lists = ptr.int(), idx.int()
    before = [t._version for t in (k, v, *e.values())]
    torch.ops.autosage.paged_cache_write(*rows, k, v, *lists, one.int(), lengths.int(), *e.values())
    assert all(t._version > old for t, old in zip((k, v, *e.values()), before))
    key, value = torch.ops.autosage.paged_cache_read(k, v, ptr, idx, one, lengths, 2, torch.bfloat16, *e.values())
    for x, got in zip(rows, (key, value)):
        assert torch.equal(got.double().cpu(), quantised_pairs(x.cpu())[0])
    out, lse = torch.ops.autosage.paged_attention(query, k, v, *lists, (lengths + 1).int(), 0.125,
                                                  key_exponents=e["key_exponents"],
                                                  value_exponents=e["value_exponents"], return_lse=True)
    again = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths + 1, scale=0.125, **e)
    assert torch.equal(out, again)
    with pytest.raises(ValueError, match="invalid page lists"):
        autosage_amd.paged_attention(query, k, v, ptr, idx + 1000, lengths, **e)


def test_capture_and_replay_of_steps():
    """Write, attend and advance in one graph: two graphs and eager calls in turn, each replay against eager results."""
    cache = Cache4([300, 0, 45], 2, 64, 64, 16, torch.bfloat16, seed=28, room=8)
    (k, v, ptr, idx), e = cache.args()
    mine = [t.view(torch.uint8).clone() for t in (k, v, *e.values())]
    mine = [mine[0].view(E2M1), mine[1].view(E2M1), mine[2].view(E8M0), mine[3].view(E8M0)]
    own = dict(zip(e, mine[2:]))
    lengths = torch.tensor(cache.lengths).cuda()
    own_lengths = lengths.clone()
    rows = torch.randn(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    query = torch.randn(3, 8, 64, device="cuda", dtype=torch.bfloat16)
    token_ptr = torch.arange(4, device="cuda")

    def step(k, v, lengths, **e):
        autosage_amd.paged_cache_write(rows, rows * 2, k, v, ptr, idx, token_ptr, lengths, **e)
        lengths += 1
        return autosage_amd.paged_attention(query, k, v, ptr, idx, lengths, scale=0.125, return_lse=True, **e)

    step(*mine[:2], own_lengths, **own)
    step(k, v, lengths, **e)
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step(k, v, lengths, **e))
        graphs.append(graph)
    torch.cuda.synchronize()
    for turn in range(6):
        rows.normal_()
        query.normal_()
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        want = step(*mine[:2], own_lengths, **own)
        assert torch.equal(own_lengths, lengths)
        assert all(torch.equal(a, b) for a, b in zip(results[turn % 2], want))
    assert torch.equal(k.view(torch.uint8), mine[0].view(torch.uint8))


def test_another_stream_and_two_calls_at_once():
    calls = []
    for seed in (29, 30):
        cache = Cache4([4000, 10, 900], 2, 64, 64, 16, torch.bfloat16, seed=seed)
        args, e = cache.args()
        query = torch.randn(3, 4, 64, device="cuda", dtype=torch.bfloat16)
        calls.append(((query, *args, torch.tensor(cache.lengths).cuda()), e))
    want = [autosage_amd.paged_attention(*c, scale=0.125, **e) for c, e in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        got = []
        for stream, (c, e) in zip(streams, calls):
            with torch.cuda.stream(stream):
                got.append(autosage_amd.paged_attention(*c, scale=0.125, **e))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_places_beyond_32_bits():
    """A cache of more than 2^32 bytes, against the pages themselves: the sequence has the pages at the end and those
    whose offsets are the same in 32 bits."""
    heads, page, width = 8, 64, 128
    wrap = (1 << 32) // (heads * page * width // 2)
    k, v = (torch.empty(wrap + 40, heads, page, width // 2, dtype=torch.uint8, device="cuda").view(E2M1) for _ in range(2))
    names = {kind: torch.empty(wrap + 40, heads, page, 4, dtype=torch.uint8, device="cuda").view(E8M0)
             for kind in ("key_exponents", "value_exponents")}
    idx = torch.tensor([wrap + 39, 39, wrap + 37, 37, wrap // 2 + 37]).cuda()
    ptr, lengths = torch.tensor([0, 5]).cuda(), torch.tensor([320]).cuda()
    gen = torch.Generator().manual_seed(31)
    rows = torch.randn(320, heads, width, generator=gen).bfloat16()
    span = (torch.tensor([0, 320]).cuda(), torch.tensor([0]).cuda())
    autosage_amd.paged_cache_write(rows.cuda(), -rows.cuda(), k, v, ptr, idx, *span, **names)
    held, packed, e = quantised_pairs(rows)
    assert torch.equal(k.view(torch.uint8)[idx].transpose(1, 2).reshape(320, heads, -1).cpu(), packed)
    assert torch.equal(names["value_exponents"].view(torch.uint8)[idx].transpose(1, 2).reshape(320, heads, -1).cpu(), e)
    key, value = autosage_amd.paged_cache_read(k, v, ptr, idx, *span, 320, dtype=torch.bfloat16, **names)
    assert torch.equal(key.double().cpu(), held) and torch.equal(value.double().cpu(), -held)
    cache = Cache4([1], heads, width, width, page, torch.bfloat16)
    cache.lengths, cache.rows = [320], {"key": [held], "value": [-held]}
    query = torch.randn(1, heads, width, generator=gen).bfloat16()
    out, lse = autosage_amd.paged_attention(query.cuda(), k, v, ptr, idx, lengths, scale=0.1, return_lse=True, **names)
    assert_attention(out, lse, plain_attention(cache, query, 0.1), dtype=torch.bfloat16, quantised=True, lse_bound=2e-4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("scale", [0.0, -0.3])
@pytest.mark.parametrize("bias", [None, (8, 20, False)])
def test_scales_of_zero_and_below(dtype, page, scale, bias):
    """A scale of zero gives all tokens the same weight (or the bias's), one below zero prefers small products."""
    _attend([1, 40, 0, 700], 2, 3, 64, 64, page, dtype, scale=scale, bias=bias, seed=32)
    _attend([1, 40, 0, 700], 2, 3, 64, 64, page, dtype, scale=scale, bias=bias, max_length=None, window=33, seed=33)
