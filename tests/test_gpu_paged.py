"""The paged cache and its attention on the GPU against 64-bit results: every place outside the sequences holds NaN."""

from __future__ import annotations

import pytest
import torch

import autosage_amd
from tests.gpu_common import require_gpu
from tests.paged_common import E4M3, Cache, assert_attention, plain_attention, quantised_rows

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _attend(lengths, heads, group, width, value_width, page, dtype, *, quantised=False, window=None, bias=None, seed=0,
            max_length="given", scale=None, **layout):
    cache = Cache(lengths, heads, width, value_width, page, dtype, quantised=quantised, seed=seed, **layout)
    gen = torch.Generator().manual_seed(seed + 1)
    query = torch.randn(len(lengths), heads * group, width, generator=gen).to(dtype)
    scale = width**-0.5 if scale is None else scale
    plain, own = {}, {}
    if bias is not None:
        buckets, distance, both = bias
        table = torch.randn(buckets, heads * group, generator=gen).to(dtype)
        plain = {"table": table, "max_distance": distance, "bidirectional": both}
        own = {"bias_table": table.cuda(), "max_distance": distance, "bidirectional": both}
    want = plain_attention(cache, query, scale, window=window, **plain)
    args, exponents = cache.args()
    bound = max(lengths) if max_length == "given" else max_length
    out, lse = autosage_amd.paged_attention(query.cuda(), *args, torch.tensor(lengths).cuda(), scale=scale,
                                            window=window, max_length=bound, return_lse=True, **own, **exponents)
    # scores are at most a few hundred here: fp32 keeps them to 1e-4
    worst = assert_attention(out, lse, want, dtype=dtype, quantised=quantised, lse_bound=2e-4)
    print(f"worst error over bound {worst:.3f}")
    return cache, query, out, lse


LENGTHS = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 300]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("page", [1, 7, 8, 12, 16, 64])
def test_lengths_and_pages(dtype, quantised, page):
    _attend(LENGTHS, 2, 3, 64, 64, page, dtype, quantised=quantised, seed=page)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("width, value_width", [(1, 1), (3, 5), (16, 16), (40, 24), (33, 65), (72, 72), (128, 128),
                                                (129, 64), (64, 200), (192, 128), (256, 256), (255, 250)])
def test_widths(dtype, quantised, width, value_width):
    _attend([1, 50, 140], 2, 2, width, value_width, 16, dtype, quantised=quantised, seed=width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads, group", [(1, 1), (3, 4), (2, 7), (1, 16), (2, 17), (1, 40)])
def test_heads(dtype, quantised, heads, group):
    _attend([5, 77, 0, 33], heads, group, 64, 64, 16, dtype, quantised=quantised, seed=group)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("window", [1, 15, 64, 1000])
def test_window(dtype, quantised, window):
    _attend([0, 1, 14, 15, 16, 200, 333], 2, 2, 64, 32, 16, dtype, quantised=quantised, window=window, seed=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("bias", [(32, 128, True), (32, 128, False), (2, 4, False), (256, 700, False)])
@pytest.mark.parametrize("window", [None, 50])
def test_bias(dtype, quantised, bias, window):
    _attend([1, 33, 130, 400], 2, 3, 32, 32, 8, dtype, quantised=quantised, bias=bias, window=window, seed=1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("max_length", ["given", None, 4000])
def test_long_and_short_sequences_together(dtype, quantised, max_length):
    _attend([3000, 1, 0, 1700, 64, 2999], 1, 4, 64, 64, 16, dtype, quantised=quantised, max_length=max_length, seed=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_length", ["given", None])
def test_one_long_sequence(dtype, max_length):
    _attend([20011], 2, 2, 32, 32, 16, dtype, max_length=max_length, seed=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("layout", [{"interleaved": True}, {"offset": 1}, {"offset": 8}, {"room": 3}])
def test_layouts(dtype, quantised, layout):
    _attend([5, 40, 90], 2, 2, 64, 64, 16, dtype, quantised=quantised, seed=4, **layout)


@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_inside_a_larger_tensor(dtype):
    cache, query, out, _ = _attend([5, 40, 90], 2, 2, 40, 40, 16, dtype, seed=5)
    args, _ = cache.args()
    lengths = torch.tensor(cache.lengths).cuda()
    wide = torch.full((3, 5, 91), float("nan"), dtype=dtype, device="cuda")
    for at in (0, 1, 8):
        view = wide[:, 1:, at:at + 40]
        view.copy_(query.cuda())
        assert torch.equal(autosage_amd.paged_attention(view, *args, lengths, scale=40**-0.5, max_length=90), out)
    turned = query.cuda().permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(autosage_amd.paged_attention(turned, *args, lengths, scale=40**-0.5, max_length=90), out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
def test_large_scores(dtype, quantised):
    """Scores of a few hundred: one token takes all of the weight, the others underflow."""
    _attend([10, 100, 600], 1, 2, 64, 64, 16, dtype, quantised=quantised, scale=3.0, seed=6)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_the_bias_masks(dtype):
    """-inf in the table masks the buckets of the near tokens: short sequences see nothing, zeros and -inf."""
    cache = Cache([1, 4, 9, 200], 1, 32, 32, 8, dtype, seed=7)
    gen = torch.Generator().manual_seed(8)
    query, table = torch.randn(4, 2, 32, generator=gen).to(dtype), torch.randn(8, 2, generator=gen).to(dtype)
    table[:4] = -torch.inf  # distances 0 to 3
    table[7, 1] = torch.finfo(dtype).min
    want = plain_attention(cache, query, 1.0, table=table, max_distance=50, bidirectional=False)
    args, _ = cache.args()
    out, lse = autosage_amd.paged_attention(query.cuda(), *args, torch.tensor(cache.lengths).cuda(), return_lse=True,
                                            bias_table=table.cuda(), max_distance=50, bidirectional=False)
    assert not out[:2].any() and bool((lse[:2] == -torch.inf).all())
    assert out.isfinite().all()
    plain = (want[0], want[1], torch.where(want[2] > 1e3, 0.0, want[2]))  # the lowest number is no size of a score
    sizes = plain_attention(cache, query, 1.0)[2]
    assert_attention(out, None, (plain[0], plain[1], plain[2] + 4 * sizes.amax()), dtype=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_length", [None, 60])
def test_masks_of_the_lowest_number(dtype, max_length):
    """Scores that are all the type's lowest number have equal weights; beside others they have none."""
    cache = Cache([7, 60], 1, 32, 32, 8, dtype, seed=23)
    query = torch.randn(2, 1, 32, dtype=dtype, device="cuda")
    table = torch.zeros(8, 1, dtype=dtype, device="cuda")
    table[:7] = torch.finfo(dtype).min  # distances below 14: all of the short one, the last 14 of the long one
    args, _ = cache.args()
    out = autosage_amd.paged_attention(query, *args, torch.tensor(cache.lengths).cuda(), scale=0.0, bias_table=table,
                                       max_distance=20, bidirectional=False, max_length=max_length).double().cpu()
    rows = [cache.rows["value"][0][:, 0].mean(0), cache.rows["value"][1][:46, 0].mean(0)]
    eps = torch.finfo(dtype).eps
    for got, want in zip(out[:, 0], rows):
        assert torch.allclose(got, want, rtol=eps, atol=1e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("count", [65, 257, 600, 1100])
@pytest.mark.parametrize("page", [8, 5])
def test_many_sequences(dtype, count, page):
    """More sequences than lanes, threads and shares, some without tokens, with and without a bound of their lengths."""
    gen = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 45, (count,), generator=gen).tolist()
    lengths[count // 2], lengths[0], lengths[-1] = 700, 0, 0
    cache, query, out, lse = _attend(lengths, 1, 2, 16, 16, page, dtype, seed=count, max_length=None)
    args, _ = cache.args()
    again = autosage_amd.paged_attention(query.cuda(), *args, torch.tensor(lengths).cuda(), scale=0.25, max_length=700)
    assert torch.equal(again, out)
    short = [min(n, 45) for n in lengths]
    single = autosage_amd.paged_attention(query.cuda(), *args, torch.tensor(short).cuda(), scale=0.25, max_length=45)
    keep = [i for i, n in enumerate(lengths) if n <= 45]
    assert torch.allclose(single[keep].float(), out[keep].float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_and_nan_rows_that_are_seen(dtype):
    cache = Cache([40, 40, 40], 1, 32, 32, 8, dtype, seed=9)
    (k, v, ptr, idx), _ = cache.args()
    query = torch.ones(3, 1, 32, dtype=dtype, device="cuda")
    lengths = torch.tensor(cache.lengths).cuda()
    want = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths)
    place = idx[ptr[:3] + 2]
    k[place[0], 0, 3, 5] = float("nan")
    v[place[1], 0, 3, 7] = float("inf")
    k[place[2], 0, 3, 9] = -float("inf")  # a score of -inf: as if the token were not there
    got = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths)
    assert got[0].isnan().all()
    assert got[1, 0, 7] == float("inf") and torch.equal(got[1, 0, :7], want[1, 0, :7])
    keep = [t for t in range(40) if t != 19]
    rows_k, rows_v = cache.rows["key"][2][keep, 0], cache.rows["value"][2][keep, 0]
    p = torch.softmax(rows_k @ query[2, 0].double().cpu(), 0)
    assert torch.allclose(got[2, 0].double().cpu(), p @ rows_v, rtol=torch.finfo(dtype).eps, atol=2e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths_and_pages_that_do_not_fit(dtype):
    cache = Cache([4, 90, 12], 2, 64, 64, 4, dtype, seed=10)
    (k, v, ptr, idx), _ = cache.args()
    query = torch.randn(3, 4, 64, device="cuda", dtype=dtype)
    call = autosage_amd.paged_attention
    lengths = torch.tensor([4, 90, 12]).cuda()
    for bound in (None, 200):
        good = call(query, k, v, ptr, idx, lengths, max_length=bound)
        out, lse = call(query, k, v, ptr, idx, lengths + torch.tensor([1, 0, 0]).cuda(), return_lse=True, max_length=bound)
        assert out[0].isnan().all() and lse[0].isnan().all() and torch.equal(out[1:], good[1:])
        for bad in (-1, k.size(0), 2**40, -(2**40)):
            other = idx.clone()
            other[1 + 20] = bad
            out = call(query, k, v, ptr, other, lengths, max_length=bound)
            assert out[1].isnan().all() and torch.equal(out[[0, 2]], good[[0, 2]])
        assert not call(query, k, v, ptr, idx, torch.tensor([0, -3, 0]).cuda(), max_length=bound).any()
        # lists that descend, or end behind page_idx: nothing outside is read
        for other in (ptr.flip(0), ptr + 10**6, ptr - 10**6, ptr * 2**40):
            call(query, k, v, other.contiguous(), idx, lengths, max_length=bound)
    out = call(query, k, v, ptr, idx, lengths, max_length=50)
    assert out[1].isnan().all() and torch.equal(out[[0, 2]], good[[0, 2]])


def test_shared_pages_and_lists_with_room():
    """Two sequences share their first pages; page_idx is a table with room for more pages than are in use."""
    cache = Cache([64, 100], 2, 64, 64, 16, torch.bfloat16, seed=11)
    (k, v, ptr, idx), _ = cache.args()
    table = torch.full((3, 9), 2**50, device="cuda")
    table[0, :4] = idx[:4]
    table[1, :7] = idx[4:11]
    table[2, :4], table[2, 4:7] = idx[:4], idx[8:11]
    query = torch.randn(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    query[2] = query[0]
    lengths = torch.tensor([64, 100, 64]).cuda()
    rows = torch.arange(4, device="cuda") * 9
    for bound in (None, 100, 5000):
        out = autosage_amd.paged_attention(query, k, v, rows, table.flatten(), lengths, max_length=bound)
        assert torch.equal(out[0], out[2])
        want = autosage_amd.paged_attention(query[:2], k, v, ptr, idx, lengths[:2], max_length=100)
        assert torch.allclose(out[:2].float(), want.float(), rtol=2.0**-7, atol=2.0**-9)


@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_joined_by_their_lse(dtype):
    cache, query, out, lse = _attend([160], 1, 3, 64, 64, 16, dtype, seed=12)
    (k, v, _, idx), _ = cache.args()
    parts = [autosage_amd.paged_attention(query.cuda(), k, v, torch.tensor([0, n]).cuda(), idx[a:a + n].contiguous(),
                                          torch.tensor([16 * n]).cuda(), scale=0.125, return_lse=True)
             for a, n in ((0, 3), (3, 7))]
    weights = torch.softmax(torch.stack([p[1] for p in parts]), 0)[..., None]
    joined = (weights * torch.stack([p[0].float() for p in parts])).sum(0)
    assert torch.allclose(joined, out.float(), rtol=2 * torch.finfo(dtype).eps, atol=2 * torch.finfo(dtype).eps)
    assert torch.allclose(torch.logsumexp(torch.stack([p[1] for p in parts]), 0), lse, atol=1e-4)


# ---- write and read ------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("width, value_width", [(1, 3), (8, 16), (40, 24), (64, 64), (72, 33), (128, 128), (256, 255)])
@pytest.mark.parametrize("page", [1, 7, 16])
def test_write_then_read(dtype, quantised, width, value_width, page):
    lengths, new = [3, 0, 40, 0, 17], [5, 0, 1, 33, 12]
    cache = Cache([a + b for a, b in zip(lengths, new)], 3, width, value_width, page, dtype, quantised=quantised, seed=13)
    (k, v, ptr, idx), exponents = cache.args()
    before = [t.view(torch.uint8).clone() for t in (k, v)]
    gen = torch.Generator().manual_seed(14)
    total = sum(new) + 4  # four rows of padding
    key = (torch.randn(total, 3, width, generator=gen) * 3).to(dtype)
    value = (torch.randn(total, 3, value_width, generator=gen) / 100).to(dtype)
    token_ptr, start = torch.tensor([0] + new).cumsum(0).cuda(), torch.tensor(lengths).cuda()
    key[-4:] = float("nan")
    autosage_amd.paged_cache_write(key.cuda(), value.cuda(), k, v, ptr, idx, token_ptr, start, **exponents)
    got = autosage_amd.paged_cache_read(k, v, ptr, idx, token_ptr, start, total, dtype=dtype, **exponents)
    for rows, back in zip((key, value), got):
        want = quantised_rows(rows[:-4])[0].to(dtype) if quantised else rows[:-4]
        assert torch.equal(back[:-4].cpu(), want) and not back[-4:].any()
    # the tokens that were there, and every place of no new token
    after = [a + b for a, b in zip(lengths, new)]
    all_ptr = torch.tensor([0] + after).cumsum(0).cuda()
    old = autosage_amd.paged_cache_read(k, v, ptr, idx, all_ptr, torch.zeros_like(start), sum(after), dtype=dtype,
                                        **exponents)
    for kind, back in zip(("key", "value"), old):
        for b, n in enumerate(lengths):
            a = int(all_ptr[b])
            assert torch.equal(back[a:a + n].double().cpu(), cache.rows[kind][b][:n].to(dtype).double())
    touched = torch.zeros(k.shape[0], page, dtype=torch.bool)
    for b, (a, n) in enumerate(zip(lengths, new)):
        t = a + torch.arange(n)
        touched[cache.page_idx[cache.page_ptr[b] + t // page], t % page] = True
    for a, b in zip(before, (k, v)):
        a, b = a.transpose(1, 2).cpu(), b.view(torch.uint8).transpose(1, 2).cpu()
        assert torch.equal(a[~touched], b[~touched])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out", DTYPES)
def test_8_bit_numbers_in_every_type(dtype, out):
    gen = torch.Generator().manual_seed(15)
    x = (torch.randn(300, 2, 48, generator=gen) * torch.exp(6 * torch.randn(300, 2, 1, generator=gen))).to(dtype)
    x = torch.where(x.isfinite(), x, 1.0)
    k, v = (torch.zeros(20, 2, 16, 48, dtype=E4M3, device="cuda") for _ in range(2))
    e = [torch.zeros(20, 2, 16, dtype=torch.int8, device="cuda") for _ in range(2)]
    lists = (torch.tensor([0, 20]).cuda(), torch.randperm(20, generator=gen).cuda())
    span = (torch.tensor([0, 300]).cuda(), torch.tensor([0]).cuda())
    names = {"key_exponents": e[0], "value_exponents": e[1]}
    autosage_amd.paged_cache_write(x.cuda(), -x.cuda(), k, v, *lists, *span, **names)
    key, value = autosage_amd.paged_cache_read(k, v, *lists, *span, 300, dtype=out, **names)
    want = quantised_rows(x)[0].to(out)
    assert torch.equal(key.cpu(), want) and torch.equal(value.cpu(), -want)


def test_8_bit_numbers_at_the_edges():
    """The rows of the CPU test, in a width that fills and one that leaves lanes idle, against the CPU."""
    tiny = 2.0**-149
    rows = torch.tensor([[0.0, -0.0, 0.0], [448.0, 1.0, -3.3], [448.0001, 1.0, 2.0**-9], [3.4e38, -1e38, 1.0],
                         [tiny, -tiny, 0.0], [2.0**-126, 2.0**-130, 2.0**-140], [17.0, 19.0, 1.0625],
                         [float("inf"), 1.0, 300.0], [float("nan"), -float("inf"), 2.0]])
    for width in (3, 96):
        x = rows.repeat(1, width // 3)[:, None]
        results = []
        for device in ("cpu", "cuda"):
            k, v = (torch.zeros(1, 1, 9, width, dtype=E4M3, device=device) for _ in range(2))
            e = [torch.zeros(1, 1, 9, dtype=torch.int8, device=device) for _ in range(2)]
            lists = (torch.tensor([0, 1], device=device), torch.tensor([0], device=device))
            span = (torch.tensor([0, 9], device=device), torch.tensor([0], device=device))
            names = {"key_exponents": e[0], "value_exponents": e[1]}
            autosage_amd.paged_cache_write(x.to(device), x.to(device), k, v, *lists, *span, **names)
            back = autosage_amd.paged_cache_read(k, v, *lists, *span, 9, dtype=torch.float32, **names)
            results.append((e[0].cpu(), *(t.cpu() for t in back)))
        for a, b in zip(*results):
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("quantised", [False, True])
def test_strided_rows_and_pages(quantised):
    """Keys and values inside one projection's output, pages of both inside one tensor, at odd offsets."""
    dtype = torch.bfloat16
    for width, at in ((40, 1), (64, 0), (64, 8), (64, 3)):
        cache = Cache([9, 30], 2, width, width, 8, dtype, quantised=quantised, seed=16, interleaved=True)
        (k, v, ptr, idx), exponents = cache.args()
        gen = torch.Generator().manual_seed(17)
        fused = torch.randn(39, 7, width + 9, generator=gen).to(dtype).cuda()
        key, value = fused[:, 2:4, at:at + width], fused[:, 4:6, at:at + width]
        token_ptr, start = torch.tensor([0, 9, 39]).cuda(), torch.zeros(2, dtype=torch.long, device="cuda")
        autosage_amd.paged_cache_write(key, value, k, v, ptr, idx, token_ptr, start, **exponents)
        back = autosage_amd.paged_cache_read(k, v, ptr, idx, token_ptr, start, 39, dtype=dtype, **exponents)
        for rows, got in zip((key, value), back):
            want = quantised_rows(rows.cpu())[0].to(dtype) if quantised else rows.cpu()
            assert torch.equal(got.cpu(), want)


def test_tokens_without_a_place():
    cache = Cache([4, 9], 1, 8, 8, 4, torch.float32, seed=18)
    (k, v, ptr, idx), _ = cache.args()
    bad = idx.clone()
    bad[2] = k.size(0)
    rows = torch.ones(6, 1, 8, device="cuda")
    before = k.clone()
    token_ptr = torch.tensor([0, 3, 6]).cuda()
    for lists, start in [((ptr, idx), [4, 12]), ((ptr, idx), [-3, -3]), ((ptr, idx), [2**40, 2**62]),
                         ((ptr, bad), [8, 4]), ((ptr + 10**6, idx), [0, 0]), ((ptr * 0, idx), [0, 0])]:
        start = torch.tensor(start).cuda()
        autosage_amd.paged_cache_write(rows, rows, k, v, *lists, token_ptr, start)
        key, value = autosage_amd.paged_cache_read(k, v, *lists, token_ptr, start, 6)
        assert not key.any() and not value.any()
    assert torch.equal(k.nan_to_num(7.0), before.nan_to_num(7.0))


@pytest.mark.parametrize("quantised", [False, True])
def test_the_registered_operators(quantised):
    ops = torch.ops.autosage
    cache = Cache([9, 30], 2, 24, 16, 8, torch.float16, quantised=quantised, seed=24, room=1)
    (k, v, ptr, idx), e = cache.args()
    e = tuple(e.values())
    rows = [torch.randn(4, 2, w, device="cuda", dtype=torch.float16) for w in (24, 16)]
    span = (torch.tensor([0, 1, 4]).cuda(), torch.tensor([9, 30]).cuda())
    query, lengths = torch.randn(2, 4, 24, device="cuda", dtype=torch.float16), torch.tensor([10, 33]).cuda()
    table = torch.randn(8, 4, device="cuda", dtype=torch.float16)
    names = dict(zip(("key_exponents", "value_exponents"), e))
    assert ops.paged_cache_write(*rows, k, v, ptr, idx, *span, *e) is None
    for a, b in zip(ops.paged_cache_read(k, v, ptr, idx, *span, 4, torch.float16, *e),
                    autosage_amd.paged_cache_read(k, v, ptr, idx, *span, 4, dtype=torch.float16, **names)):
        assert torch.equal(a, b) and a.any()
    out, lse = ops.paged_attention(query, k, v, ptr, idx, lengths, 0.2, 20, table, 15, False, 40, *e, True)
    want = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths, scale=0.2, window=20, bias_table=table,
                                        max_distance=15, bidirectional=False, max_length=40, return_lse=True, **names)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    out, lse = ops.paged_attention(query, k, v, ptr, idx, lengths, **names)
    assert torch.equal(out, autosage_amd.paged_attention(query, k, v, ptr, idx, lengths, **names)) and lse.numel() == 0


def test_32_bit_lists_and_validation(monkeypatch):
    cache = Cache([9, 30], 2, 24, 16, 8, torch.float16, seed=25)
    (k, v, ptr, idx), _ = cache.args()
    query, lengths = torch.randn(2, 4, 24, device="cuda", dtype=torch.float16), torch.tensor([9, 30]).cuda()
    want = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths)
    assert torch.equal(autosage_amd.paged_attention(query, k, v, ptr.int(), idx.int(), lengths.int()), want)
    monkeypatch.setenv("AUTOSAGE_VALIDATE", "1")
    assert torch.equal(autosage_amd.paged_attention(query, k, v, ptr, idx, lengths), want)
    with pytest.raises(ValueError, match="page ids"):
        autosage_amd.paged_attention(query, k, v, ptr, idx + k.size(0), lengths)
    with pytest.raises(ValueError, match="more tokens"):
        autosage_amd.paged_attention(query, k, v, ptr, idx, lengths + 30)


# ---- together ---------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_one_at_a_time_equal_the_attention_over_edges(dtype):
    """The whole of it: causal attention of a text over the edges of a CSR graph with a learned position bias, head by
    head; then the same tokens one at a time through the cache."""
    n, heads, width, buckets, distance = 70, 2, 32, 16, 40
    gen = torch.Generator().manual_seed(19)
    q, k, v = (torch.randn(n, heads, width, generator=gen).to(dtype).cuda() for _ in range(3))
    table = torch.randn(buckets, heads, generator=gen).to(dtype).cuda()
    crow = torch.arange(n + 1).cumsum(0).cuda()
    col = torch.cat([torch.arange(i + 1) for i in range(n)]).cuda()
    bias = autosage_amd.csr_position_bias(crow, col, table, max_distance=distance, bidirectional=False)
    scale = width**-0.5
    ops = torch.ops.autosage
    rows = []
    for h in range(heads):
        scores = ops.sddmm_csr(crow, col, q[:, h].float().contiguous(), k[:, h].float().contiguous()) * scale
        p = ops.csr_row_softmax(crow, scores + bias[h].float())
        rows.append(ops.spmm_csr(crow, col, p, v[:, h].float().contiguous()))
    whole = torch.stack(rows, 1)
    page = 8
    pages = [torch.full((12, heads, page, width), float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
    table_of_pages = torch.randperm(12, generator=gen).cuda()[:10]
    ptr = torch.tensor([0, 10]).cuda()
    one = torch.tensor([0, 1]).cuda()
    for t in range(n):
        start = torch.tensor([t]).cuda()
        autosage_amd.paged_cache_write(k[t:t + 1], v[t:t + 1], *pages, ptr, table_of_pages, one, start)
        out = autosage_amd.paged_attention(q[t:t + 1], *pages, ptr, table_of_pages, start + 1, scale=scale,
                                           bias_table=table, max_distance=distance, bidirectional=False)
        # both are within a few fp32 roundings of the exact result; 16 bits round once more
        assert torch.allclose(out[0].float(), whole[t], rtol=torch.finfo(dtype).eps, atol=2e-5)


@pytest.mark.parametrize("quantised", [False, True])
def test_capture_and_replay_of_steps(quantised):
    """Write, attend and advance in one graph: two graphs and eager calls in turn, each replay against eager results."""
    dtype = torch.bfloat16
    cache = Cache([300, 0, 45], 2, 64, 64, 16, dtype, quantised=quantised, seed=20, room=8)
    (k, v, ptr, idx), exponents = cache.args()
    for t in (k, v):  # places that no token has been written to are not seen; give eager and captured runs the same
        t.view(torch.uint8).copy_(torch.where(t.float().isnan(), torch.zeros((), device="cuda"), t.float()).to(t.dtype).view(
            torch.uint8))
    mine = [k.clone(), v.clone(), *(None if e is None else e.clone() for e in exponents.values())]
    lengths = torch.tensor(cache.lengths).cuda()
    rows = torch.randn(3, 2, 64, device="cuda", dtype=dtype)
    query = torch.randn(3, 8, 64, device="cuda", dtype=dtype)
    token_ptr = torch.arange(4, device="cuda")

    def step(k, v, lengths, **e):
        autosage_amd.paged_cache_write(rows, rows * 2, k, v, ptr, idx, token_ptr, lengths, **e)
        lengths += 1
        return autosage_amd.paged_attention(query, k, v, ptr, idx, lengths, scale=0.125, return_lse=True, **e)

    own = {"key_exponents": mine[2], "value_exponents": mine[3]}
    own_lengths = lengths.clone()
    step(mine[0], mine[1], own_lengths, **own)
    step(k, v, lengths, **exponents)
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step(k, v, lengths, **exponents))
        graphs.append(graph)
    torch.cuda.synchronize()
    for turn in range(6):
        rows.normal_()
        query.normal_()
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        want = step(mine[0], mine[1], own_lengths, **own)
        assert torch.equal(own_lengths, lengths)
        for a, b in zip(results[turn % 2], want):
            assert torch.equal(a, b)
    assert torch.equal(k.view(torch.uint8), mine[0].view(torch.uint8))


def test_another_stream_and_two_calls_at_once():
    calls = []
    for seed in (21, 22):
        cache = Cache([4000, 10, 900], 2, 64, 64, 16, torch.bfloat16, seed=seed)
        args, _ = cache.args()
        query = torch.randn(3, 4, 64, device="cuda", dtype=torch.bfloat16)
        calls.append((query, *args, torch.tensor(cache.lengths).cuda()))
    want = [autosage_amd.paged_attention(*c, scale=0.125) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        got = []
        for stream, c in zip(streams, calls):
            with torch.cuda.stream(stream):
                got.append(autosage_amd.paged_attention(*c, scale=0.125))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("quantised", [False, True])
def test_offsets_beyond_32_bits(quantised):
    """A cache of more than 2^32 elements, the sequence's pages at its end and its start."""
    dtype = E4M3 if quantised else torch.bfloat16
    heads, page, width = 8, 64, 128
    pages = (1 << 32) // (heads * page * width) + 40
    k, v = (torch.empty(pages, heads, page, width, dtype=dtype, device="cuda") for _ in range(2))
    e = [torch.zeros(pages, heads, page, dtype=torch.int8, device="cuda") for _ in range(2)] if quantised else [None, None]
    names = {"key_exponents": e[0], "value_exponents": e[1]}
    idx = torch.tensor([pages - 1, 0, pages - 3, 1, pages // 2 + 1]).cuda()
    ptr = torch.tensor([0, 5]).cuda()
    rows = torch.randn(300, heads, width, device="cuda", dtype=torch.bfloat16)
    span = (torch.tensor([0, 300]).cuda(), torch.tensor([0]).cuda())
    autosage_amd.paged_cache_write(rows, -rows, k, v, ptr, idx, *span, **names)
    key, value = autosage_amd.paged_cache_read(k, v, ptr, idx, *span, 300, dtype=torch.bfloat16, **names)
    if not quantised:
        assert torch.equal(key, rows) and torch.equal(value, -rows)
    query = torch.randn(1, heads, width, device="cuda", dtype=torch.bfloat16)
    got = autosage_amd.paged_attention(query, k, v, ptr, idx, torch.tensor([300]).cuda(), scale=width**-0.5, **names)
    s = (key.double() * query[0].double()).sum(-1) * width**-0.5
    want = (torch.softmax(s, 0)[..., None] * value.double()).sum(0)
    assert torch.allclose(got[0].double(), want, rtol=2.0**-8, atol=1e-4)


def test_token_lists_that_begin_anywhere():
    """Where a position passes 64 bits there is no place, and the other sequence's tokens keep theirs."""
    cache = Cache([4, 9], 1, 8, 8, 4, torch.float32, seed=19)
    rows = torch.randn(6, 1, 8, device="cuda")
    for own, begin in [(-(2**62) - 10, 2**62 - 1), (-(2**63), 2**62 - 1), (-(2**63), 0), (-(2**62), 2**62),
                       (-(2**62), 2**63 - 1), (-(2**63), -(2**63)), (-5, -(2**63))]:
        (k, v, ptr, idx), _ = cache.args()
        before = k.clone()
        token_ptr, start = torch.tensor([own, 3, 6]).cuda(), torch.tensor([begin, 5]).cuda()
        autosage_amd.paged_cache_write(rows, rows, k, v, ptr, idx, token_ptr, start)
        key, value = autosage_amd.paged_cache_read(k, v, ptr, idx, token_ptr, start, 6)
        for back in (key, value):
            assert not back[:3].any() and torch.equal(back[3:], rows[3:])
        for t in range(5, 8):
            before[idx[ptr[1] + t // 4], 0, t % 4] = rows[t - 2, 0]
        assert torch.equal(k.nan_to_num(7.0), before.nan_to_num(7.0))


@pytest.mark.parametrize("registered", [False, True])
@pytest.mark.parametrize("quantised", [False, True])
def test_a_write_is_seen_by_autograd(quantised, registered):
    """What a graph saved of the pages is no longer what it was: backward refuses, as after any write in place."""
    cache = Cache([4, 9], 1, 8, 8, 4, torch.float32, quantised=quantised, seed=26)
    (k, v, ptr, idx), e = cache.args()
    rows = torch.randn(2, 1, 8, device="cuda")
    span = (torch.tensor([0, 1, 2]).cuda(), torch.tensor([3, 8]).cuda())
    written = [k, v, *(t for t in e.values() if t is not None)]
    before = [t._version for t in written]
    if registered:
        torch.ops.autosage.paged_cache_write(rows, rows, k, v, ptr, idx, *span, *e.values())
    else:
        autosage_amd.paged_cache_write(rows, rows, k, v, ptr, idx, *span, **e)
    assert all(t._version > old for t, old in zip(written, before))
    if not quantised:
        query = torch.ones(8, device="cuda", requires_grad=True)
        scores = k[0, 0] * query
        autosage_amd.paged_cache_write(rows, rows, k, v, ptr, idx, *span)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            scores.sum().backward()


def test_forward_mode_is_refused():
    """By the public functions and the registered operators, whose results would have no tangent."""
    cache = Cache([4, 9], 1, 8, 8, 4, torch.float32, seed=29)
    (k, v, ptr, idx), _ = cache.args()
    coded, e = Cache([4, 9], 1, 8, 8, 4, torch.float32, quantised=True, seed=29).args()
    query, rows = torch.randn(2, 1, 8, device="cuda"), torch.randn(2, 1, 8, device="cuda")
    span, lengths = (torch.tensor([0, 1, 2]).cuda(), torch.tensor([3, 8]).cuda()), torch.tensor([4, 9]).cuda()
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))

        for of in (autosage_amd, torch.ops.autosage):
            for call in (lambda: of.paged_attention(dual(query), k, v, ptr, idx, lengths),
                         lambda: of.paged_attention(dual(query), *coded, lengths, **e),
                         lambda: of.paged_cache_write(rows, dual(rows), k, v, ptr, idx, *span),
                         lambda: of.paged_cache_read(k, dual(v), ptr, idx, *span, 2)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
            of.paged_attention(query, *coded, lengths, **e)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [8, 5])
@pytest.mark.parametrize("width, value_width", [(3, 5), (5, 3), (1, 200), (40, 40), (33, 65), (129, 130), (200, 136),
                                                (255, 250)])
@pytest.mark.parametrize("from_end", [1, 3])
def test_infinite_numbers_at_the_ends_of_rows(dtype, page, width, value_width, from_end):
    """Rows shorter than a run, rows whose last run is moved back over the one before, and wide ones: a score of -inf is
    no token, an infinite value makes its own column infinite and no other."""
    at, value_at = max(width - from_end, 0), max(value_width - from_end, 0)
    cache = Cache([40, 40, 700], 1, width, value_width, page, dtype, seed=30)
    (k, v, ptr, idx), _ = cache.args()
    query = torch.full((3, 1, width), 0.25, dtype=dtype, device="cuda")
    lengths = torch.tensor(cache.lengths).cuda()
    want = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths)
    for b, pages, column, what in ((0, k, at, -torch.inf), (1, v, value_at, torch.inf), (2, k, at, -torch.inf)):
        pages[idx[ptr[b] + 19 // page], 0, 19 % page, column] = what
    got = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths)
    others = [d for d in range(value_width) if d != value_at]
    assert got[1, 0, value_at] == torch.inf and torch.equal(got[1, 0, others], want[1, 0, others])
    for b in (0, 2):
        keep = [t for t in range(cache.lengths[b]) if t != 19]
        for rows in cache.rows.values():
            rows[b] = rows[b][keep]
        cache.lengths[b] -= 1
    plain = plain_attention(cache, query.cpu(), 1.0)
    assert_attention(got[[0, 2]], None, [t[[0, 2]] for t in plain], dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_length", [None, 700])
@pytest.mark.parametrize("quantised", [False, True])
def test_two_masks_and_their_lse(dtype, max_length, quantised):
    """-3e38 beside the type's lowest number: tokens of the former have all of the weight, and the logarithm of the sum
    is the mask's number.  A score times log2(e) would be infinite for either."""
    cache = Cache([7, 2, 700], 1, 32, 32, 8, dtype, quantised=quantised, seed=27)
    query = torch.randn(3, 1, 32, dtype=dtype, device="cuda")
    table = torch.full((8, 1), torch.finfo(dtype).min, dtype=dtype)
    table[:3] = -3e38  # distances 0 to 2
    args, e = cache.args()
    out, lse = autosage_amd.paged_attention(query, *args, torch.tensor(cache.lengths).cuda(), scale=0.0, return_lse=True,
                                            bias_table=table.cuda(), max_distance=20, bidirectional=False,
                                            max_length=max_length, **e)
    for b, n in enumerate(cache.lengths):
        rows = cache.rows["value"][b][max(n - 3, 0):, 0]
        # equal weights: three fp32 terms and a quotient, bf16 parts of a weight of 1 are exact; one rounding to the type
        allowed = rows.abs().mean(0) * 2.0**-21 + rows.mean(0).abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0**-10)
        assert bool(((out[b, 0].double().cpu() - rows.mean(0)).abs() <= allowed).all())
        # log(3) is nothing beside 3e38
        assert lse[b, 0].item() == table[0, 0].item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_near_the_largest_number(dtype):
    """Finite scores of up to 3e38 in both signs: the largest takes all of the weight."""
    for page, most in ((8, 5), (8, 690), (5, 300)):
        cache = Cache([700], 1, 8, 8, page, dtype, seed=31)
        (k, v, ptr, idx), _ = cache.args()
        rows = torch.zeros(700, 1, 8, dtype=dtype, device="cuda")
        rows[:, 0, 0] = torch.linspace(-3e19, 2.9e19, 700, device="cuda").to(dtype)
        rows[most, 0, 0] = 3e19
        values = torch.randn(700, 1, 8, device="cuda").to(dtype)
        span, lengths = (torch.tensor([0, 700]).cuda(), torch.tensor([0]).cuda()), torch.tensor([700]).cuda()
        autosage_amd.paged_cache_write(rows, values, k, v, ptr, idx, *span)
        query = torch.full((1, 1, 8), 1e19, dtype=dtype, device="cuda")
        out, lse = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths, return_lse=True)
        assert torch.equal(out[0], values[most])
        # one product, exact in fp32 for bf16, rounded once for float32 (and once by the scale of 1)
        want = float(rows[most, 0, 0].double() * query[0, 0, 0].double())
        assert abs(lse[0, 0].item() / want - 1) <= 2.0**-23


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("width, page", [(32, 8), (5, 8), (200, 8), (64, 5)])
def test_infinite_queries(dtype, quantised, width, page):
    """Scores of -inf alone are no token at all: zeros.  A score of +inf makes its head NaN, and no other."""
    cache = Cache([40, 700], 1, width, width, page, dtype, quantised=quantised, seed=32)
    (k, v, ptr, idx), e = cache.args()
    rows = torch.randn(740, 1, width, device="cuda").to(dtype)
    rows[:, :, 2] = rows[:, :, 2].abs() + 1
    span, lengths = (torch.tensor([0, 40, 740]).cuda(), torch.tensor([0, 0]).cuda()), torch.tensor([40, 700]).cuda()
    autosage_amd.paged_cache_write(rows, rows, k, v, ptr, idx, *span, **e)
    query = torch.randn(2, 3, width, device="cuda").to(dtype)
    want = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths, scale=0.1, **e)
    query[:, 0, 2], query[:, 2, 2] = -torch.inf, torch.inf
    out, lse = autosage_amd.paged_attention(query, k, v, ptr, idx, lengths, scale=0.1, return_lse=True, **e)
    assert not out[:, 0].any() and bool((lse[:, 0] == -torch.inf).all())
    assert torch.equal(out[:, 1], want[:, 1]) and out[:, 2].isnan().all()


# ---- paths between the others ------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("page", [16, 12])
@pytest.mark.parametrize("window, bias", [(1501, None), (None, (32, 128, False)), (1003, (32, 4000, True))])
def test_windows_and_biases_of_sequences_in_shares(dtype, quantised, page, window, bias):
    """Parts begin inside a sequence at any token, near to the query and far."""
    _attend([3000, 1, 0, 1700, 64, 2999], 2, 2, 32, 32, page, dtype, quantised=quantised, window=window, bias=bias,
            max_length=None, seed=33)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("page", [12, 1])
@pytest.mark.parametrize("width, value_width", [(128, 128), (200, 136), (256, 255), (5, 200), (100, 3), (250, 1)])
def test_tokens_looked_up_one_by_one(dtype, quantised, page, width, value_width):
    _attend([1, 50, 140, 700], 2, 2, width, value_width, page, dtype, quantised=quantised, max_length=None, seed=width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width, value_width", [(64, 64), (200, 136), (5, 3)])
def test_exponents_that_are_not_neighbours(dtype, width, value_width):
    """Exponents with the tokens of a page outermost: written, read and attended to as those with them innermost."""
    lengths = [5, 40, 90]
    cache = Cache(lengths, 2, width, value_width, 16, dtype, quantised=True, seed=34)
    (k, v, ptr, idx), e = cache.args()
    turned = {name: t.permute(2, 0, 1).contiguous().permute(1, 2, 0) for name, t in e.items()}
    gen = torch.Generator().manual_seed(35)
    rows = [torch.randn(135, 2, w, generator=gen).to(dtype).cuda() for w in (width, value_width)]
    span = (torch.tensor([0, 5, 45, 135]).cuda(), torch.zeros(3, dtype=torch.long, device="cuda"))
    results = []
    for names in (e, turned):
        pages = [torch.zeros_like(k.view(torch.uint8)).view(E4M3), torch.zeros_like(v.view(torch.uint8)).view(E4M3)]
        autosage_amd.paged_cache_write(*rows, *pages, ptr, idx, *span, **names)
        results.append([*(p.view(torch.uint8) for p in pages), *names.values(),
                        *autosage_amd.paged_cache_read(*pages, ptr, idx, *span, 135, dtype=dtype, **names)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    # the attention over them, looked up one by one
    cache.rows = {kind: [t.double().cpu() for t in results[1][at].split(lengths)] for kind, at in (("key", 4), ("value", 5))}
    query = torch.randn(3, 4, width, generator=gen).to(dtype)
    for bound in (90, None):
        out, lse = autosage_amd.paged_attention(query.cuda(), *pages, ptr, idx, torch.tensor(lengths).cuda(), scale=0.1,
                                                return_lse=True, max_length=bound, **turned)
        assert_attention(out, lse, plain_attention(cache, query, 0.1), dtype=dtype, quantised=True, lse_bound=2e-4)


@pytest.mark.parametrize("quantised", [False, True])
def test_places_beyond_32_bits(quantised):
    """A cache of more than 2^32 elements, against the pages themselves: the sequence has the pages at the end and those
    whose offsets are the same in 32 bits."""
    dtype = E4M3 if quantised else torch.bfloat16
    heads, page, width = 8, 64, 128
    wrap = (1 << 32) // (heads * page * width)
    k, v = (torch.empty(wrap + 40, heads, page, width, dtype=dtype, device="cuda") for _ in range(2))
    e = [torch.zeros(wrap + 40, heads, page, dtype=torch.int8, device="cuda") for _ in range(2)] if quantised else []
    names = dict(zip(("key_exponents", "value_exponents"), e))
    idx = torch.tensor([wrap + 39, 39, wrap + 37, 37, wrap // 2 + 37]).cuda()
    ptr, lengths = torch.tensor([0, 5]).cuda(), torch.tensor([320]).cuda()
    gen = torch.Generator().manual_seed(36)
    rows = torch.randn(320, heads, width, generator=gen).bfloat16()
    span = (torch.tensor([0, 320]).cuda(), torch.tensor([0]).cuda())
    autosage_amd.paged_cache_write(rows.cuda(), -rows.cuda(), k, v, ptr, idx, *span, **names)
    held, exponents = quantised_rows(rows) if quantised else (rows.double(), None)
    for pages, sign, of in ((k, 1, 0), (v, -1, 1)):
        there = pages[idx].transpose(1, 2).reshape(320, heads, width).double().cpu()
        if quantised:
            assert torch.equal(e[of][idx].transpose(1, 2).reshape(320, heads).long().cpu(), exponents)
            there = torch.ldexp(there, exponents[..., None])
        assert torch.equal(there, sign * held)
    key, value = autosage_amd.paged_cache_read(k, v, ptr, idx, *span, 320, dtype=torch.bfloat16, **names)
    assert torch.equal(key.double().cpu(), held) and torch.equal(value.double().cpu(), -held)
    cache = Cache([1], heads, width, width, page, torch.bfloat16)
    cache.lengths, cache.rows = [320], {"key": [held], "value": [-held]}
    query = torch.randn(1, heads, width, generator=gen).bfloat16()
    out, lse = autosage_amd.paged_attention(query.cuda(), k, v, ptr, idx, lengths, scale=0.1, return_lse=True, **names)
    assert_attention(out, lse, plain_attention(cache, query, 0.1), dtype=torch.bfloat16, quantised=quantised, lse_bound=2e-4)
